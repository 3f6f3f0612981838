"""The 8-bit rows, norms and linear against float64 on the CPU (GPU).

Every case prints its name before it launches.  Integers are compared exactly
where the quotient they round is exact in the kernel's inputs (fp16 rows of the
plain and the RMS kind, fp32 rows of the plain kind); elsewhere an integer may
differ from the oracle's only where the oracle's quotient lies within the fp32
rounding error of a half.  u = 2^-24 is fp32's rounding, fp16's is 2^-11.
"""
import math

import pytest
import torch

from dollama_amd import ops
from oracle import quant_ref as Q
from oracle import ref_ops as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
WIDTHS = [1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 511, 512, 513, 640, 1003, 1024, 1031, 1280, 1536, 1537, 2048, 2500,
          4096, 4101, 8192, 8200, 16384, 16385, 20000]


def announce(msg):
    print(f"[case] {msg}", flush=True)


def cpu(shape, seed, dtype=torch.float16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def spread(rows, K, seed, dtype=torch.float16):
    """Rows with channels of unequal spread, as activations have them."""
    g = torch.Generator().manual_seed(seed)
    ch = torch.exp(0.7 * torch.randn(K, generator=g))
    return (torch.randn(rows, K, generator=g) * ch).to(dtype)


def gpu_rows(rows, K, dtype):
    """[rows, K] filled with a sentinel, inside a wider tensor that has to keep it."""
    whole = torch.full((rows + 2, K + 24), 77, dtype=dtype, device="cuda")
    return whole, whole[1:rows + 1, 8:8 + K]


def untouched(whole, rows, K):
    w = whole.clone()
    w[1:rows + 1, 8:8 + K] = 77
    return bool((w == 77).all())


def sum_steps(K):
    """Most fp32 additions a value of a row passes through: 32 in a thread's
    registers (or every K / 1024th value of long rows), 6 in a wave, 16 waves."""
    return max(32, K // 1024 + 1) + 6 + 16


# --------------------------------------------------------------- quantise ---
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K", WIDTHS)
def test_quantize_rows_is_the_nearest_integer(gpu, K, dtype):
    rows = 7
    announce(f"quantize {rows}x{K} {dtype}")
    x = spread(rows, K, K, dtype)
    # exact halves: values that are odd multiples of max / 254
    x[1] = (torch.arange(K) % 255 - 127).to(dtype)
    x[2] = ((torch.arange(K) * 2 + 1) % 255).to(dtype)
    x[2, 0] = 254
    x[3] = 0
    x[4] = torch.tensor([2.0 ** -24, -2.0 ** -23])[torch.arange(K) % 2].to(dtype)
    _, q, s = Q.rows(x.double())
    wq, out = gpu_rows(rows, K, torch.int8)
    got, scale = ops.quantize_rows(x.cuda(), out=out)
    assert got is out and untouched(wq, rows, K)
    assert torch.equal(out.cpu().double(), q)
    # max / 127 is one fp32 division
    assert torch.equal(scale.cpu(), x.abs().amax(1).float() / 127.0)
    assert float((scale.cpu().double() - s).abs().max()) <= U * float(s.max())


def test_quantize_rows_of_tiny_and_huge_fp32(gpu):
    announce("quantize fp32 rows near the ends of the range")
    x = spread(8, 333, 5, torch.float32)
    f = torch.tensor([1e-44, 1e-38, 1e-37, 2.0 ** -101, 2.0 ** -99, 1e30, 1e38, 1.0])
    x = x / x.abs().amax(1, keepdim=True) * f[:, None]
    t, q, _ = Q.rows(x.double())
    got, scale = ops.quantize_rows(x.cuda())
    assert torch.equal(got.cpu().double(), q)
    assert torch.equal(scale.cpu(), x.abs().amax(1) / 127.0)


@pytest.mark.parametrize("K", [5, 320, 1500, 3000, 9000, 17000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_with_infinity_or_nan_come_out_as_nan_alone(gpu, K, dtype):
    announce(f"non-finite rows K={K} {dtype}")
    x = spread(6, K, 3, dtype)
    x[1, K - 1] = float("inf")
    x[2, 0] = -float("inf")
    x[4, K // 2] = float("nan")
    clean = torch.tensor([0, 3, 5])
    ok = [r for r in clean.tolist()]
    g = cpu((K,), 4) * 0.3 + 1
    for name, call in (("quantize", lambda v: ops.quantize_rows(v)),
                       ("rms", lambda v: ops.rms_norm_q8(v, g.cuda())),
                       ("layer", lambda v: ops.layer_norm_q8(v, g.cuda(), g.cuda()))):
        q, s = call(x.cuda())
        q0, s0 = call(x[clean].cuda())
        assert torch.isnan(s[[1, 2, 4]]).all(), name
        assert (q[[1, 2, 4]] == 0).all(), name
        assert torch.equal(q[ok], q0) and torch.equal(s[ok], s0), f"{name}: a row depends on its neighbours"
        y = ops.dequantize_rows(q, s)
        assert torch.isnan(y[[1, 2, 4]]).all() and torch.isfinite(y[ok]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 15), (5, 16), (4, 17), (33, 640), (7, 1003), (2, 20000)])
def test_dequantize_rows(gpu, rows, K, dtype):
    announce(f"dequantize {rows}x{K} {dtype}")
    g = torch.Generator().manual_seed(K)
    q = torch.randint(-128, 128, (rows, K), generator=g, dtype=torch.int8)
    s = torch.rand(rows, generator=g) * 0.3
    wide = torch.zeros(rows, K + 11, dtype=torch.int8, device="cuda")
    wide[:, 3:3 + K] = q.cuda()
    wy, out = gpu_rows(rows, K, dtype)
    ops.dequantize_rows(wide[:, 3:3 + K], s.cuda(), out=out)
    assert untouched(wy, rows, K)
    assert torch.equal(out.cpu(), (q.float() * s[:, None]).to(dtype))
    assert torch.equal(ops.dequantize_rows(q.cuda(), s.cuda(), dtype=dtype).cpu(), out.cpu())


# ------------------------------------------------------------------ norms ---
def check_rows(q, scale, v, err, what):
    """q and scale of the oracle's rows v, whose values the kernel has within
    err (absolute, per row)."""
    t, ref, s = Q.rows(v)
    top = v.abs().amax(1)
    slack = 127.0 * 2.0 * err / top.clamp_min(1e-300)  # v and its maximum
    off = (t - q.double()).abs()
    assert bool((off <= 0.5 + slack[:, None]).all()), f"{what}: off by {float(off.max())}"
    far = ((t - torch.floor(t) - 0.5).abs() > slack[:, None])
    assert torch.equal(q.double()[far], ref[far]), f"{what}: an integer away from a half differs"
    bound = err / 127.0 + 2 * U * s
    assert bool(((scale.double() - s).abs() <= bound).all()), f"{what}: scale"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("residual,gamma", [(False, False), (False, True), (True, True)])
@pytest.mark.parametrize("K", WIDTHS)
def test_rms_norm_q8(gpu, K, residual, gamma, dtype):
    rows, eps = 5, 1e-5
    announce(f"rms_norm_q8 {rows}x{K} residual={residual} gamma={gamma} {dtype}")
    x = spread(rows, K, K + 1, dtype)
    x[3] = 0
    r = cpu((rows, K), 2, dtype) if residual else None
    if residual:
        r[3] = 0
    g = cpu((K,), 3) * 0.3 + 1 if gamma else None
    h = (x.float() + r.float()).to(dtype) if residual else x
    wq, out = gpu_rows(rows, K, torch.int8)
    wh, ho = gpu_rows(rows, K, dtype) if residual else (None, None)
    res = ops.rms_norm_q8(x.cuda(), None if g is None else g.cuda(), None if r is None else r.cuda(), eps=eps,
                          sum_out=ho, out=out)
    assert untouched(wq, rows, K)
    if residual:
        assert untouched(wh, rows, K) and torch.equal(res[2].cpu(), h)
    hd = h.double()
    gd = None if g is None else g.double()
    prod = hd if g is None else hd * gd
    if dtype == torch.float32:
        prod = (h if g is None else h * g.float()).double()  # one fp32 rounding
    # the integers come from the products alone, exact to the last half
    _, q, _ = Q.rows(prod)
    assert torch.equal(out.cpu().double(), q)
    v = Q.rms_norm(hd, gd, eps)
    top = v.abs().amax(1)
    # a square, its sum's roundings (halved by the root), mean, root, quotient, product of scale
    rel = U * (0.5 * (sum_steps(K) + 2) + 5)
    s = top / 127.0
    assert bool(((res[1].cpu().double() - s).abs() <= rel * s).all())
    assert float(res[1][3]) == 0.0


@pytest.mark.parametrize("K", [5, 77, 640, 1283, 5000, 20000])
def test_rms_norm_q8_of_tiny_and_huge_fp32_without_eps(gpu, K):
    """The squares of these pass fp32's range in either direction."""
    announce(f"rms_norm_q8 of fp32 rows near the ends of the range, K={K}")
    f = torch.tensor([1e-41, 1e-36, 1e-30, 1e-23, 1e-20, 1.0, 1e18, 1e25, 1e35])
    x = spread(9, K, K, torch.float32).clamp(-99, 99) * f[:, None]
    g = cpu((K,), 3) * 0.3 + 1
    for gamma in (None, g, g * 1000, g / 1000):
        q, s = ops.rms_norm_q8(x.cuda(), None if gamma is None else gamma.cuda(), eps=0.0)
        prod = x.double() if gamma is None else x.double() * gamma.double()
        _, ref, top = Q.rows(prod)
        ref_s = top / x.double().square().mean(1).sqrt()
        assert torch.equal(q.cpu().double(), ref)
        # one rounding from fp64
        assert bool(((s.cpu().double() - ref_s).abs() <= U * (1 + 2.0 ** -20) * ref_s).all())


@pytest.mark.parametrize("rows,K", [(300000, 5), (30000, 60), (20000, 77), (10000, 200), (8000, 320), (8192, 640),
                                    (4099, 701), (8192, 1280), (5000, 1283), (4096, 1800), (1024, 2500), (512, 5000),
                                    (300, 8192), (256, 12000), (150, 16384), (150, 20000)])
def test_rms_norm_q8_integers_of_fp32_rows_are_those_of_64_bits(gpu, rows, K):
    """Millions of products with gamma, some of whose quotients lie as close to a
    half as the products' fp32 rounding is to them."""
    announce(f"rms_norm_q8 {rows}x{K} against float64, fp32")
    x = spread(rows, K, K, torch.float32).cuda()
    r = cpu((rows, K), 2, torch.float32).cuda()
    g = (cpu((K,), 3) * 0.3 + 1).cuda()
    eps = torch.tensor(1e-5).double().cuda()
    q, s, h = ops.rms_norm_q8(x, g, residual=r, eps=1e-5)
    hd = h.double()
    _, ref, top = Q.rows(hd * g.double())  # exact: 24 and 11 bits
    assert int((q.double() != ref).sum()) == 0
    ref = top / torch.sqrt(hd.square().mean(1) + eps)
    assert bool(((s.double() - ref).abs() <= U * (1 + 2.0 ** -20) * ref).all())


@pytest.mark.parametrize("K", [5, 77, 640, 1283, 5000, 20000])
def test_norms_round_exact_halves_to_the_even_integer(gpu, K):
    """Rows of small integers whose maximum makes many quotients half an integer
    exactly: 254 v = (2k + 1) a for v = a / 2 and where 127 divides a."""
    announce(f"norms of rows with exact halves, K={K}")
    gen = torch.Generator().manual_seed(K)
    top = torch.tensor([254, 2, 127 * 6, 127 * 16, 2046, 10, 127 * 14, 508])
    x = torch.round((torch.rand(8, K, generator=gen) * 2 - 1).double() * top[:, None])
    x[:, 0], x[:, 1] = top.double(), -(top // 2).double()
    halves = (x * 254).remainder(top[:, None]) == 0
    assert bool(((halves & ((x * 254 / top[:, None]).remainder(2) == 1)).sum(1) >= 1).all())
    for dtype in (torch.float16, torch.float32):
        for scale in (1.0, 2.0 ** -9):
            h = (x * scale).to(dtype)
            assert torch.equal(h.double(), x * scale)
            _, ref, _ = Q.rows(x)
            for gamma in (None, 1.0, 1.2998046875, -0.0625):
                g = None if gamma is None else torch.full((K,), gamma, dtype=torch.float16, device="cuda")
                q, _ = ops.rms_norm_q8(h.cuda(), g)
                sign = -1.0 if gamma is not None and gamma < 0 else 1.0
                assert torch.equal(q.cpu().double(), sign * ref), f"rms {dtype} {scale} {gamma}"
            # beta alone: rows of equal values
            for row in range(8):
                q, _ = ops.layer_norm_q8(torch.ones(2, K, dtype=dtype, device="cuda"), None, h[row].half().cuda())
                assert torch.equal(q.cpu().double(), ref[row].expand(2, K)), f"layer {dtype} {scale} {row}"


def test_norms_of_zero_rows_without_eps(gpu):
    """0 / 0 is not formed: a row of zeros has scale 0 whatever eps is (RMS); of
    equal values, a LayerNorm with eps > 0 has beta alone."""
    announce("norms of rows without spread")
    for K in (3, 64, 640, 1300, 5000, 17000):
        z = torch.zeros(3, K, dtype=torch.float16, device="cuda")
        q, s = ops.rms_norm_q8(z, eps=0.0)
        assert (q == 0).all() and (s == 0).all()
        b = cpu((K,), 3).cuda()
        q, s = ops.layer_norm_q8(z + 5, None, b)
        ref, rs = ops.quantize_rows(b[None].expand(3, K).contiguous())
        assert torch.equal(q, ref) and torch.equal(s, rs)


@pytest.mark.parametrize("rows,K", [(4099, 513), (4096, 640), (4103, 701), (5001, 768), (4096, 1100), (4098, 1283),
                                    (4096, 1536), (4097, 1800), (5000, 2048)])
def test_layer_norm_q8_of_many_rows(gpu, rows, K):
    """The kernels that many fp16 rows of 513 to 768 and of 1025 to 2048 values take."""
    announce(f"layer_norm_q8 {rows}x{K}")
    x, g, b = spread(rows, K, K), cpu((K,), 3) * 0.3 + 1, cpu((K,), 4) * 0.2
    whole, out = gpu_rows(rows, K, torch.int8)
    q, s = ops.layer_norm_q8(x.cuda(), g.cuda(), b.cuda(), out=out)
    assert untouched(whole, rows, K)
    hd = x.double()
    v = Q.layer_norm(hd, g.double(), b.double(), 1e-5)
    check_rows(q.cpu(), s.cpu(), v, layer_error(hd, v, g, K, 1e-5), f"layer_norm {rows}x{K}")


def layer_error(hd, v, g, K, eps):
    """Per row, how far fp32 arithmetic may leave a LayerNorm's values from v.  The
    mean is off by its sum's roundings of mean |h| at most, and shifts every value
    by as much; the root's relative error as in the RMS norm; difference, product,
    affine and its rounding: 4 more."""
    gmax = 1.0 if g is None else float(g.double().abs().max())
    d = hd - hd.mean(1, keepdim=True)
    rs = 1.0 / torch.sqrt((d * d).mean(1) + eps)
    n = sum_steps(K)
    shift = U * (n + 3) * hd.abs().mean(1)
    rel = U * (0.5 * (n + 5) + 7) + 0.5 * (shift * rs) ** 2
    return gmax * rs * (shift + d.abs().amax(1) * rel + U * hd.abs().amax(1)) + U * v.abs().amax(1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("residual,affine", [(False, False), (False, True), (True, True)])
@pytest.mark.parametrize("K", WIDTHS)
def test_layer_norm_q8(gpu, K, residual, affine, dtype):
    rows, eps = 5, 1e-5
    announce(f"layer_norm_q8 {rows}x{K} residual={residual} affine={affine} {dtype}")
    x = spread(rows, K, K + 1, dtype)
    x[1] += 40  # a mean far from 0
    x[3] = 0
    r = cpu((rows, K), 2, dtype) if residual else None
    g = cpu((K,), 3) * 0.3 + 1 if affine else None
    b = cpu((K,), 4) * 0.2 if affine else None
    h = (x.float() + r.float()).to(dtype) if residual else x
    wq, out = gpu_rows(rows, K, torch.int8)
    wh, ho = gpu_rows(rows, K, dtype) if residual else (None, None)
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    res = ops.layer_norm_q8(x.cuda(), up(g), up(b), up(r), eps=eps, sum_out=ho, out=out)
    assert untouched(wq, rows, K)
    if residual:
        assert untouched(wh, rows, K) and torch.equal(res[2].cpu(), h)
    hd = h.double()
    v = Q.layer_norm(hd, None if g is None else g.double(), None if b is None else b.double(), eps)
    gmax = 1.0 if g is None else float(g.double().abs().max())
    d = hd - hd.mean(1, keepdim=True)
    rs = 1.0 / torch.sqrt((d * d).mean(1) + eps)
    # the mean is off by the sum's roundings of mean |h| at most, and shifts
    # every value by as much; the root's relative error as in the RMS norm;
    # difference, product, affine and its rounding: 4 more
    n = sum_steps(K)
    shift = U * (n + 2) * hd.abs().mean(1)
    dmax = d.abs().amax(1)
    rel = U * (0.5 * (n + 4) + 6) + 0.5 * (shift * rs) ** 2
    err = gmax * rs * (shift + dmax * rel + U * hd.abs().amax(1)) + U * v.abs().amax(1)
    check_rows(out.cpu(), res[1].cpu(), v, err, f"layer_norm {K}")


def same_rows(q, scale, v, tol, what):
    """q and scale of the oracle's rows v (float64), each integer the nearest one
    unless its quotient lies within tol (per row) of a half; the scale rounded once."""
    t, ref, s = Q.rows(v)
    off = q.double() != ref
    near = (t - torch.floor(t) - 0.5).abs() <= tol[:, None]
    assert not bool((off & ~near).any()), f"{what}: {int((off & ~near).sum())} integers differ"
    # from fp64 that is off by 2^-45 or so, to fp32
    assert bool(((scale.double() - s).abs() <= U * (1 + 2.0 ** -20) * s + 2.0 ** -149).all()), f"{what}: scale"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("mean", [0, 40])
@pytest.mark.parametrize("rows,K", [(300000, 5), (30000, 60), (20000, 77), (10000, 200), (8000, 320), (1000, 640),
                                    (8192, 640), (4099, 701), (1500, 1031), (5000, 1283), (4096, 1800), (1024, 2500),
                                    (512, 5000), (256, 12000), (150, 20000)])
def test_layer_norm_q8_integers_are_those_of_64_bits(gpu, rows, K, mean, dtype):
    """Millions of values, some of whose quotients lie as close to a half as fp32
    statistics are to the real ones."""
    announce(f"layer_norm_q8 {rows}x{K} around {mean} against float64, {dtype}")
    x = (spread(rows, K, K).cuda().float() + mean).to(dtype)
    g, b = (cpu((K,), 3) * 0.3 + 1).cuda(), (cpu((K,), 4) * 0.2).cuda()
    eps = torch.tensor(1e-5).double().cuda()  # as the entry points take it
    h = x.double()
    v = Q.layer_norm(h, g.double(), b.double(), eps)
    # sums of K values in fp64, in any order, in kernel and oracle: (K + 8) 2^-53 of the
    # largest |h| each, which shifts v by as much over the spread; 127 / top of it twice
    rs = 1.0 / torch.sqrt((h - h.mean(1, keepdim=True)).square().mean(1) + eps)
    tol = 4 * 127 * (K + 8) * 2.0 ** -53 * h.abs().amax(1) * rs * float(g.abs().max()) / v.abs().amax(1)
    q, s = ops.layer_norm_q8(x, g, b)
    same_rows(q, s, v, tol, f"layer_norm {rows}x{K}")


@pytest.mark.parametrize("K", [5, 77, 640, 1283, 5000, 20000])
def test_layer_norm_q8_of_tiny_and_huge_fp32_without_eps(gpu, K):
    """The squares of these pass fp32's range in either direction."""
    announce(f"layer_norm_q8 of fp32 rows near the ends of the range, K={K}")
    f = torch.tensor([1e-36, 1e-30, 1e-23, 1e-20, 1.0, 1e18, 1e25, 1e34])
    x = spread(8, K, K, torch.float32) * f[:, None]
    g = cpu((K,), 3) * 0.3 + 1
    v = Q.layer_norm(x.double(), g.double(), None, 0.0)
    q, s = ops.layer_norm_q8(x.cuda(), g.cuda(), eps=0.0)
    tol = torch.full((8,), 4 * 127 * (K + 8) * 2.0 ** -53 * math.sqrt(K) * float(g.abs().max()), dtype=torch.float64)
    same_rows(q.cpu(), s.cpu(), v, tol, f"layer_norm {K}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K", [3, 7, 77, 640, 1283, 5000, 20000])
def test_layer_norm_q8_of_equal_values_is_zero(gpu, K, dtype):
    announce(f"layer_norm_q8 of rows of one value, K={K} {dtype}")
    x = torch.tensor([0.3, -1.7, 1234.5, 1e-3]).to(dtype).cuda()[:, None].expand(4, K).contiguous()
    q, s = ops.layer_norm_q8(x)
    assert (q == 0).all() and (s == 0).all()
    q, s = ops.layer_norm_q8(x, eps=0.0)  # 0 / 0
    assert (q == 0).all() and torch.isnan(s).all()


def test_norms_write_the_sum_in_place_and_read_strided_rows(gpu):
    announce("norms: sum over x or over the residual, rows inside wider tensors")
    for K in (40, 640, 2052, 5000, 17000):
        for dtype in (torch.float16, torch.float32):
            x, r, g = spread(9, K, 1, dtype).cuda(), cpu((9, K), 2, dtype).cuda(), (cpu((K,), 3) + 1).cuda()
            for norm in (ops.rms_norm_q8, ops.layer_norm_q8):
                q, s, h = norm(x, g, residual=r)
                for target in ("x", "residual"):
                    xi, ri = x.clone(), r.clone()
                    t = xi if target == "x" else ri
                    qi, si, hi = norm(xi, g, residual=ri, sum_out=t)
                    assert hi is t and torch.equal(hi, h) and torch.equal(qi, q) and torch.equal(si, s)
                wx, xs = gpu_rows(9, K, dtype)
                wr, rs = gpu_rows(9, K, dtype)
                xs.copy_(x)
                rs.copy_(r)
                qi, si, hi = norm(xs, g, residual=rs)
                assert torch.equal(hi, h) and torch.equal(qi, q) and torch.equal(si, s)
                # a row's result does not depend on the others
                q1, s1, h1 = norm(x[4:5], g, residual=r[4:5])
                assert torch.equal(q1, q[4:5]) and torch.equal(s1, s[4:5]) and torch.equal(h1, h[4:5])


@pytest.mark.parametrize("K", [5, 40, 643, 2052, 17000])
def test_norms_between_column_slices_of_one_tensor(gpu, K):
    announce(f"norms: x, residual and sum side by side in the rows of one tensor, K {K}")
    for dtype in (torch.float16, torch.float32):
        x, r = spread(9, K, 1, dtype).cuda(), cpu((9, K), 2, dtype).cuda()
        for norm in (ops.rms_norm_q8, ops.layer_norm_q8):
            q, s, h = norm(x, residual=r)
            for order in ((0, 1, 2), (2, 0, 1), (1, 2, 0)):
                whole = torch.full((9, 3 * K), 77, dtype=dtype, device="cuda")
                xs, rs, hs = (whole[:, c * K:(c + 1) * K] for c in order)
                xs.copy_(x)
                rs.copy_(r)
                qs, ss, _ = norm(xs, residual=rs, sum_out=hs)
                assert torch.equal(hs, h) and torch.equal(qs, q) and torch.equal(ss, s)
                assert torch.equal(xs, x) and torch.equal(rs, r)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K", [5, 60, 77, 200, 640, 1283, 2052, 5000, 9000, 17000])
def test_norms_with_a_non_finite_gamma_or_beta(gpu, K, dtype):
    """v is not finite in any row then, rows of zeros included (0 times infinity)."""
    announce(f"norms with infinities and NaN in gamma and beta, K={K} {dtype}")
    x, g, b = spread(4, K, 1, dtype).cuda(), (cpu((K,), 3) + 1).cuda(), cpu((K,), 4).cuda()
    x[2] = 0
    for value in (float("inf"), float("-inf"), float("nan")):
        for at in (0, K // 2, K - 1):
            h = g.clone()
            h[at] = value
            for q, s in (ops.rms_norm_q8(x, h), ops.layer_norm_q8(x, h, b), ops.layer_norm_q8(x, None, h)):
                assert (q == 0).all() and torch.isnan(s).all(), f"{value} at {at}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K", [5, 40, 640, 643, 1283, 2052, 5000, 17000])
def test_norms_that_do_not_write_their_sum(gpu, K, dtype):
    """A residual with no place for the sum, which the C entries take: the same
    rows as with one, and x and the residual as they were."""
    from dollama_amd import _lib
    announce(f"norms of a sum that is not written, K={K} {dtype}")
    rows, t = 9, "fp16" if dtype == torch.float16 else "f32"
    x, r = spread(rows, K, 1, dtype).cuda(), cpu((rows, K), 2, dtype).cuda()
    g, b = (cpu((K,), 3) + 1).cuda(), (cpu((K,), 4) * 0.2).cuda()
    x0, r0 = x.clone(), r.clone()
    stream = torch.cuda.current_stream().cuda_stream
    for name, norm, extra in (("rms", ops.rms_norm_q8, ()), ("layer", ops.layer_norm_q8, (b,))):
        q, s, _ = norm(x, g, *extra, residual=r, eps=1e-5)
        whole, out = gpu_rows(rows, K, torch.int8)
        scale = torch.full((rows,), 77.0, device="cuda")
        _lib.call(f"dlm_{name}_norm_q8_{t}", x.data_ptr(), K, r.data_ptr(), K, None, 0, g.data_ptr(),
                  *(e.data_ptr() for e in extra), out.data_ptr(), K + 24, scale.data_ptr(), rows, K, 1e-5, stream)
        assert torch.equal(out, q) and torch.equal(scale, s) and untouched(whole, rows, K), name
        assert torch.equal(x, x0) and torch.equal(r, r0), name


# ----------------------------------------------------------------- linear ---
def int8_rows(rows, K, seed, low=-127):
    """Random 8-bit rows at a 16-byte row stride whose padding holds garbage."""
    g = torch.Generator().manual_seed(seed)
    whole = torch.randint(low, 128, (rows, (K + 15) // 16 * 16), generator=g, dtype=torch.int8)
    whole[:, K:] = 113
    return whole.cuda()[:, :K], whole[:, :K]


def check_linear(M, N, K, act="none", bias=True, residual=True, dtype=torch.float16, beta=1.0, seed=1, low=-127):
    announce(f"linear_q8 {M}x{N}x{K} act={act} bias={bias} residual={residual} beta={beta} {dtype}")
    xg, x = int8_rows(M, K, seed, low)
    wg, w = int8_rows(N, K, seed + 1, low)
    g = torch.Generator().manual_seed(seed + 2)
    sx = (torch.rand(M, generator=g) + 0.5) * (1.5 / (64 * math.sqrt(K)))
    sw = (torch.rand(N, generator=g) + 0.5) / 64
    cols = N // 2 if act == "geglu" else N
    b = cpu((N,), seed + 3) if bias else None
    r = cpu((M, cols), seed + 4, dtype) if residual else None
    ref, mag = Q.linear(x, sx, w, sw, b, r, act, beta)
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    wy, out = gpu_rows(M, cols, dtype)
    code = {"none": ops.ACT_NONE, "silu": ops.ACT_SILU, "gelu": ops.ACT_GELU, "geglu": ops.ACT_GEGLU}[act]
    y = ops.linear_q8(xg, sx.cuda(), wg, sw.cuda(), bias=up(b), residual=up(r), act=code, out=out, beta=beta)
    assert y is out and untouched(wy, M, cols), "wrote outside its rows"
    # conversion, two scales, bias, residual: u each of what they act on, times
    # at most 1.13 (the activations' slopes); the activations add 4 u (silu) or
    # the 1.5e-7 of the erf approximation on half the value
    tol = 8 * U * mag + (0 if act == "none" else 4e-7 * mag)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -11 * ref.abs() * 1.001 + 2.0 ** -25
    off = (out.cpu().double() - ref).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.2f} of the bound"
    plain = ops.linear_q8(xg, sx.cuda(), wg, sw.cuda(), bias=up(b), residual=up(r), act=code, dtype=dtype, beta=beta)
    assert torch.equal(plain, out), "the output's layout shows in its values"
    return xg, sx, wg, sw, b, r, out


SHAPES = [(1, 1, 1), (1, 16, 64), (1, 1280, 640), (1, 63, 1003), (2, 17, 15), (3, 40, 16), (5, 333, 17), (7, 128, 4099),
          (13, 320, 2560), (16, 96, 63), (17, 96, 65), (31, 130, 100), (32, 64, 1000), (33, 64, 128), (64, 80, 640),
          (65, 77, 127), (100, 1283, 200), (128, 256, 256), (154, 640, 2048), (200, 1, 513), (257, 300, 1280),
          (300, 161, 1000), (513, 640, 640), (1000, 320, 333), (2100, 200, 130)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_q8(gpu, M, N, K, dtype):
    check_linear(M, N, K, dtype=dtype)
    check_linear(M, N, K, bias=False, residual=False, dtype=dtype, seed=9)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu", "geglu"])
@pytest.mark.parametrize("M,N,K", [(1, 16, 40), (1, 640, 320), (9, 320, 1003), (40, 96, 64), (154, 1280, 640),
                                   (300, 336, 200), (1030, 640, 320)])
def test_linear_q8_activations(gpu, M, N, K, act, dtype):
    check_linear(M, N, K, act=act, dtype=dtype, residual=False)
    check_linear(M, N, K, act=act, dtype=dtype, beta=-0.75, seed=5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tile", range(1, 15))
def test_linear_q8_every_kernel(gpu, tile, dtype):
    """Every kernel and tile the plan chooses among (dlm_q8_force_tile), on shapes
    with ragged last tiles in both directions, K from less than a slice to more
    than the ring, odd N, K tails of 1 to 15 values, and rows of padding."""
    from dollama_amd import _lib
    try:
        _lib.call("dlm_q8_force_tile", tile)
        for M, N, K in ((300, 340, 648), (70, 161, 1003), (200, 16, 5), (1, 35, 127), (129, 129, 128), (260, 272, 1297),
                        (513, 78, 384), (16, 2, 640)):
            check_linear(M, N, K, dtype=dtype)
        check_linear(300, 340, 648, act="silu", dtype=dtype, residual=False, seed=21)
        check_linear(257, 99, 200, act="gelu", dtype=dtype, beta=0.5, seed=23)
        check_linear(300, 336, 648, act="geglu", dtype=dtype, residual=False, seed=25)
        check_linear(131, 144, 333, act="geglu", dtype=dtype, beta=-2.0, seed=27)
    finally:
        _lib.call("dlm_q8_force_tile", 0)


@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_q8_sums_reach_the_ends_of_their_range(gpu, M):
    """K = 131071 products of -128 x -128 stay below 2^31; the sums are exact
    also where fp32 sums would not be (one odd unit among 2^31)."""
    announce(f"largest K, M={M}")
    K, N = 131071, 24
    x = torch.full((M, 131072), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((N, 131072), -128, dtype=torch.int8, device="cuda")[:, :K]
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    y = ops.linear_q8(x, one_m, w, one_n, dtype=torch.float32)
    assert (y == float(128 * 128 * K)).all()  # 2^14 (2^17 - 1): exact in fp32
    check_linear(M, N, 4096, low=-128, dtype=torch.float32)


def test_linear_q8_in_place_residual_and_nan_rows(gpu):
    for M, N, K in ((3, 64, 100), (70, 200, 640), (300, 640, 640)):
        xg, sx, wg, sw, b, r, out = check_linear(M, N, K)
        y = r.cuda()
        ops.linear_q8(xg, sx.cuda(), wg, sw.cuda(), bias=b.cuda(), residual=y, out=y)
        assert torch.equal(y, out)
        sx = sx.clone()
        sx[M // 2] = float("nan")
        y = ops.linear_q8(xg, sx.cuda(), wg, sw.cuda(), bias=b.cuda(), residual=r.cuda())
        assert torch.isnan(y[M // 2]).all()
        rest = [i for i in range(M) if i != M // 2]
        assert torch.equal(y[rest], out[rest])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_linear_q8_between_column_slices_of_one_tensor(gpu, dtype):
    for M, N, K in ((3, 33, 100), (70, 200, 640), (300, 645, 256)):
        xg, sx, wg, sw, b, r, out = check_linear(M, N, K, dtype=dtype)
        for first in (0, 1):
            whole = torch.full((M, 2 * N + 3), 77, dtype=dtype, device="cuda")
            rs = whole[:, first * N:(first + 1) * N]
            y = whole[:, (1 - first) * N:(2 - first) * N]
            rs.copy_(r)
            ops.linear_q8(xg, sx.cuda(), wg, sw.cuda(), bias=b.cuda(), residual=rs, out=y)
            assert torch.equal(y, out) and torch.equal(rs, r.cuda()) and (whole[:, 2 * N:] == 77).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_linear_q8_activations_of_infinities_and_nan(gpu, dtype):
    announce(f"linear_q8 activations of infinities and NaN {dtype}")
    x = torch.ones(5, 64, dtype=torch.int8, device="cuda")
    w = torch.ones(32, 64, dtype=torch.int8, device="cuda")
    sx, sw = torch.ones(5, device="cuda"), torch.full((32,), 2.0 ** -6, device="cuda")  # sums of 1
    b = torch.zeros(32, dtype=torch.float16, device="cuda")
    b[4], b[5], b[6], b[7] = float("inf"), float("-inf"), float("nan"), -60000.0
    for act in (ops.ACT_SILU, ops.ACT_GELU):
        y = ops.linear_q8(x, sx, w, sw, bias=b, act=act, dtype=dtype)
        assert (y[:, 4] == float("inf")).all() and torch.isnan(y[:, 6]).all() and (y[:, 7] == 0).all()
        assert torch.isfinite(y[:, :4]).all() and torch.isfinite(y[:, 8:]).all()
    # GEGLU: columns 4-7 are the gates of outputs 0-3
    y = ops.linear_q8(x, sx, w, sw, bias=b, act=ops.ACT_GEGLU, dtype=dtype)
    assert (y[:, 0] == float("inf")).all() and torch.isnan(y[:, 2]).all() and (y[:, 3] == 0).all()
    assert torch.isfinite(y[:, 4:]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_linear_q8_activations_at_minus_infinity(gpu, dtype):
    """GELU takes its limit, 0, as a gate too; SiLU is the quotient x / (1 + exp(-x)),
    NaN there."""
    announce(f"linear_q8 activations at -infinity {dtype}")
    x = torch.ones(5, 64, dtype=torch.int8, device="cuda")
    w = torch.ones(32, 64, dtype=torch.int8, device="cuda")
    sx, sw = torch.ones(5, device="cuda"), torch.full((32,), 2.0 ** -6, device="cuda")  # sums of 1
    b = torch.zeros(32, dtype=torch.float16, device="cuda")
    b[5] = float("-inf")
    y = ops.linear_q8(x, sx, w, sw, bias=b, act=ops.ACT_GELU, dtype=dtype)
    assert (y[:, 5] == 0).all()
    y = ops.linear_q8(x, sx, w, sw, bias=b, act=ops.ACT_SILU, dtype=dtype)
    assert torch.isnan(y[:, 5]).all() and torch.isfinite(y[:, 6:]).all()
    # columns 4-7 are the gates of outputs 0-3
    y = ops.linear_q8(x, sx, w, sw, bias=b, act=ops.ACT_GEGLU, dtype=dtype)
    assert (y[:, 1] == 0).all() and torch.isfinite(y).all()


def test_linear_q8_activations_over_their_range(gpu):
    """Each activation of 400,000 values of either sign from 1e-6 to 30, one product
    each: GELU within 4e-7 |x| (7.5e-8 of its tail's approximation, 5 roundings and
    the reciprocal's of a tail of at most 1/2), SiLU within |x| 2^-24 relative (the
    exponent's rounding) and 6 roundings."""
    announce("linear_q8 activations against float64")
    g = torch.Generator().manual_seed(3)
    z = torch.exp(torch.rand(400000, generator=g, dtype=torch.float64) * math.log(3e7) + math.log(1e-6)).float()
    z = torch.cat([z, -z, torch.zeros(8)])
    N = z.numel()
    w = torch.zeros(N, 16, dtype=torch.int8, device="cuda")
    w[:, 0] = 1
    x = torch.zeros(1, 16, dtype=torch.int8, device="cuda")
    x[0, 0] = 1
    run = lambda act: ops.linear_q8(x, torch.ones(1, device="cuda"), w, z.cuda(), act=act,  # noqa: E731
                                    dtype=torch.float32)[0].cpu().double()
    zd = z.double()
    ref = zd * torch.special.ndtr(zd)
    assert bool(((run(ops.ACT_GELU) - ref).abs() <= 4e-7 * zd.abs()).all())
    ref = zd * torch.sigmoid(zd)
    assert bool(((run(ops.ACT_SILU) - ref).abs() <= (6 + zd.abs()) * 2.0 ** -24 * ref.abs()).all())


def test_linear_q8_row_results_do_not_depend_on_the_batch(gpu):
    announce("linear_q8: a row alone, in small batches and in a large one")
    M, N, K = 700, 640, 1280
    xg, sx, wg, sw, b, r, out = check_linear(M, N, K, act="gelu")
    for lo, n in ((0, 1), (5, 3), (16, 16), (100, 40), (333, 154), (0, 512)):
        y = ops.linear_q8(xg[lo:lo + n], sx[lo:lo + n].cuda(), wg, sw.cuda(), bias=b.cuda(),
                          residual=r[lo:lo + n].cuda(), act=ops.ACT_GELU)
        assert torch.equal(y, out[lo:lo + n]), f"rows {lo}..{lo + n}"


@pytest.mark.parametrize("act,residual,dtype", [("none", False, torch.float16), ("none", True, torch.float16),
                                                ("geglu", False, torch.float16), ("silu", True, torch.float16),
                                                ("gelu", False, torch.float32), ("none", True, torch.float32)])
def test_linear_q8_is_the_same_on_every_tile(gpu, act, residual, dtype):
    """Four million outputs of each form: among so many, some lie so close to a tie
    that one rounding more or less shows."""
    from dollama_amd import _lib
    announce(f"linear_q8 on every tile: {act} residual={residual} {dtype}")
    M, N, K = 1024, 4096, 48
    xg, _ = int8_rows(M, K, 3)
    wg, _ = int8_rows(N, K, 4)
    torch.manual_seed(5)
    sx, sw = torch.rand(M, device="cuda") * 1e-2, torch.rand(N, device="cuda") * 1e-2
    b = torch.randn(N, device="cuda").half()
    cols = N // 2 if act == "geglu" else N
    r = torch.randn(M, cols, device="cuda").to(dtype) if residual else None
    code = {"none": ops.ACT_NONE, "silu": ops.ACT_SILU, "gelu": ops.ACT_GELU, "geglu": ops.ACT_GEGLU}[act]
    run = lambda: ops.linear_q8(xg, sx, wg, sw, bias=b, residual=r, act=code, beta=0.7, dtype=dtype)  # noqa: E731
    ref = run()
    try:
        for tile in range(1, 15):
            _lib.call("dlm_q8_force_tile", tile)
            assert torch.equal(run(), ref), f"tile {tile}"
    finally:
        _lib.call("dlm_q8_force_tile", 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,K", [(2300, 1100), (2300, 1536), (4200, 1537), (4200, 2048), (1100, 2049), (1500, 2560),
                                    (1024, 2901)])
def test_layer_norm_rows_do_not_depend_on_their_number(gpu, rows, K, dtype):
    announce(f"layer_norm_q8 rows alone and among {rows}, K={K} {dtype}")
    x = (spread(rows, K, K).cuda().float() + 3).to(dtype)
    g, b = (cpu((K,), 3) * 0.3 + 1).cuda(), (cpu((K,), 4) * 0.2).cuda()
    # eps makes the variance count: a sum in another order shows in the scales
    q, s = ops.layer_norm_q8(x, g, b, eps=0.5)
    for lo, n in ((0, 1), (17, 5), (100, 900)):
        q1, s1 = ops.layer_norm_q8(x[lo:lo + n], g, b, eps=0.5)
        assert torch.equal(q1, q[lo:lo + n]) and torch.equal(s1, s[lo:lo + n]), f"rows {lo}..{lo + n}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K", [48, 100, 320, 513, 640, 701, 768, 769, 1031, 1280, 1501, 1536, 1800, 2048, 3000])
def test_row_results_do_not_depend_on_the_number_of_rows(gpu, K, dtype):
    announce(f"rows alone and among 5000, K={K} {dtype}")
    torch.manual_seed(K)
    x = torch.randn(5000, K, device="cuda").to(dtype) + 3
    r = torch.randn(5000, K, device="cuda").to(dtype)
    g, b = torch.randn(K, device="cuda").half(), torch.randn(K, device="cuda").half()
    for call in (lambda v, w: ops.quantize_rows(v), lambda v, w: ops.rms_norm_q8(v, g, residual=w),
                 lambda v, w: ops.layer_norm_q8(v, g, b, residual=w)):
        whole = call(x, r)
        for lo, n in ((0, 1), (17, 5), (1000, 1100), (0, 4095), (0, 4096)):
            for a, c in zip(whole, call(x[lo:lo + n], r[lo:lo + n])):
                assert torch.equal(a[lo:lo + n], c), f"rows {lo}..{lo + n}"


# ------------------------------------------------------------- large sizes ---
def test_rows_past_32_bit_offsets(gpu):
    """Tensors of more than 2^31 elements, and more rows than one launch takes
    (2^21): rows at the ends and at the launches' borders equal the same rows alone."""
    for rows, K, dtype in ((70000, 32768, torch.float16), ((1 << 21) + 77, 24, torch.float32)):
        announce(f"quantize, norms, dequantize {rows}x{K} {dtype}")
        torch.manual_seed(K)
        x = torch.randn(rows, K, device="cuda", dtype=dtype)
        g = torch.rand(K, device="cuda").half() + 0.5
        pick = torch.tensor([0, 1, rows // 2, min(rows - 1, (1 << 21) - 1), min(rows - 1, 1 << 21), rows - 2, rows - 1])
        for name, call in (("quantize", lambda v: ops.quantize_rows(v)), ("rms", lambda v: ops.rms_norm_q8(v, g)),
                           ("layer", lambda v: ops.layer_norm_q8(v, g, g))):
            q, s = call(x)
            q1, s1 = call(x[pick])
            assert torch.equal(q[pick], q1) and torch.equal(s[pick], s1), name
        y = ops.dequantize_rows(q, s)
        assert torch.equal(y[pick], ops.dequantize_rows(q1, s1))
        del x, y, q, s


def test_linear_q8_past_32_bit_offsets(gpu):
    """Operands and outputs of more than 4 GiB, and more rows than one launch takes."""
    for M, N, K in ((40000, 60000, 16), (36000, 16, 131071), ((1 << 24) + 300, 16, 16)):
        announce(f"linear_q8 {M}x{N}x{K}")
        torch.manual_seed(N)
        ld = (K + 15) // 16 * 16
        x = torch.randint(-128, 128, (M, ld), device="cuda", dtype=torch.int8)[:, :K]
        w = torch.randint(-128, 128, (N, ld), device="cuda", dtype=torch.int8)[:, :K]
        sx, sw = torch.rand(M, device="cuda") * 1e-3, torch.rand(N, device="cuda") * 1e-2
        b = torch.randn(N, device="cuda").half()
        y = ops.linear_q8(x, sx, w, sw, bias=b)
        pick = torch.tensor([0, M // 2, min(M - 1, (1 << 24) - 1), min(M - 1, 1 << 24), M - 1], device="cuda")
        rows = x.new_zeros(len(pick), ld)
        rows[:, :K] = x[pick]
        assert torch.equal(y[pick], ops.linear_q8(rows[:, :K], sx[pick], w, sw, bias=b))
        part = slice(max(0, N - 9), N)  # the last columns against float64
        ref = (rows[:, :K].double().cpu() @ w[part].double().cpu().t()) * sx[pick].double().cpu()[:, None]
        ref = ref * sw[part].double().cpu() + b[part].double().cpu()
        mag = ref.abs() + 2 * b[part].double().cpu().abs()
        off = (y[pick][:, part].cpu().double() - ref).abs()
        assert bool((off <= 8 * U * mag + 2.0 ** -11 * ref.abs() * 1.001 + 2.0 ** -25).all())
        del x, w, y


def test_linear_q8_of_most_columns_on_every_tile(gpu):
    """The largest N with more rows than the smallest tile's launch takes."""
    from dollama_amd import _lib
    M, N, K = 130, 1 << 25, 16
    announce(f"linear_q8 {M}x{N}x{K} on every tile")
    torch.manual_seed(1)
    x = torch.randint(-128, 128, (M, K), device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), device="cuda", dtype=torch.int8)
    sx, sw = torch.rand(M, device="cuda") * 1e-2, torch.rand(N, device="cuda") * 1e-2
    ref, y = ops.linear_q8(x, sx, w, sw), torch.empty(M, N, dtype=torch.float16, device="cuda")
    cols = torch.tensor([0, 1, N // 2, N - 33, N - 1], device="cuda")
    z = (x.double().cpu() @ w[cols].double().cpu().t()) * sx.double().cpu()[:, None] * sw[cols].double().cpu()
    assert bool(((ref[:, cols].cpu().double() - z).abs() <= (2.0 ** -11 + 2.0 ** -20) * z.abs() + 2.0 ** -25).all())
    try:
        for tile in range(1, 15):
            print(f"[case] tile {tile}", flush=True)
            _lib.call("dlm_q8_force_tile", tile)
            y.zero_()
            assert torch.equal(ops.linear_q8(x, sx, w, sw, out=y), ref), f"tile {tile}"
    finally:
        _lib.call("dlm_q8_force_tile", 0)


# --------------------------------------------------------------- together ---
class Block:
    """Norm, gated projection, row quantisation, projection back and residual:
    a feed-forward layer in 8 bits."""

    def __init__(self, C, F, seed):
        k = lambda *s, i=0: cpu(s, seed + i)  # noqa: E731
        self.gamma, self.beta = (k(C, i=1) * 0.2 + 1).cuda(), (k(C, i=2) * 0.1).cuda()
        self.w1, self.b1 = (k(2 * F, C, i=3).float() / math.sqrt(C)).half(), k(2 * F, i=4) * 0.1
        self.w2, self.b2 = (k(C, F, i=5).float() / math.sqrt(F)).half(), k(C, i=6) * 0.1
        wp, self.b1p = ops.pack_geglu(self.w1.cuda(), self.b1.cuda())
        self.q1, self.s1 = ops.quantize_rows(wp)
        self.q2, self.s2 = ops.quantize_rows(self.w2.cuda())
        self.b2g = self.b2.cuda()

    def __call__(self, x, attn, rms=False):
        if rms:
            q, s, h = ops.rms_norm_q8(x, self.gamma, residual=attn)
        else:
            q, s, h = ops.layer_norm_q8(x, self.gamma, self.beta, residual=attn)
        f = ops.linear_q8(q, s, self.q1, self.s1, bias=self.b1p, act=ops.ACT_GEGLU)
        q, s = ops.quantize_rows(f)
        return ops.linear_q8(q, s, self.q2, self.s2, bias=self.b2g, residual=h, out=h)

    def exact(self, x, attn, rms=False):
        """The unquantised layer in float64."""
        h = x.double() + attn.double()
        g = self.gamma.cpu().double()
        n = Q.rms_norm(h, g, 1e-6) if rms else Q.layer_norm(h, g, self.beta.cpu().double(), 1e-5)
        z = n @ self.w1.double().t() + self.b1.double()
        v, t = z.chunk(2, 1)
        return h, (v * (t * torch.special.ndtr(t))) @ self.w2.double().t() + self.b2.double()


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("M", [1, 2, 33, 154, 1024])
def test_feed_forward_in_8_bits(gpu, M, rms):
    """Against the unquantised layer.  A rounding to 8 bits is off by a / 254 at
    most and a / 254 / sqrt(3) in the root mean square; with a about 4 times a
    row's root mean square, that is 0.9% of it.  Four such sources (two
    activations, two weights) add up to 2%; the gate's slope and the product of
    two of them leave it below 4%."""
    announce(f"feed-forward block M={M} rms={rms}")
    C, F = 640, 2560
    blk = Block(C, F, 100)
    x, a = cpu((M, C), 1), cpu((M, C), 2)
    h, ff = blk.exact(x, a, rms)
    y = blk(x.cuda(), a.cuda(), rms)
    got = y.cpu().double() - h
    assert float((got - ff).norm() / ff.norm()) <= 0.04


def test_feed_forward_on_other_streams_and_in_graphs(gpu):
    """Eager on the default stream = eager on another = captured and replayed,
    two graphs replayed at the same time on two streams included."""
    announce("feed-forward block: streams and graphs")
    blk = Block(320, 1280, 50)
    xs = [cpu((M, 320), M).cuda() for M in (1, 48, 600)]
    at = [cpu((M, 320), M + 1).cuda() for M in (1, 48, 600)]
    ref = [blk(x, a) for x, a in zip(xs, at)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [blk(x, a) for x, a in zip(xs, at)]
    side.synchronize()
    for r, g in zip(ref, got):
        assert torch.equal(r, g)
    graphs = []
    for x, a in zip(xs, at):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = blk(x, a)
        graphs.append((g, y))
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in range(4):
        for (g, y), s in zip(graphs, streams):
            y.zero_()
        torch.cuda.synchronize()
        for (g, y), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        junk = torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")
        torch.cuda.synchronize()
        for (g, y), r in zip(graphs, ref):
            assert torch.equal(y, r), f"replay {i}"
        del junk
    xs[1].copy_(cpu((48, 320), 999).cuda())  # new values in the captured inputs
    torch.cuda.synchronize()
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[1][1], blk(xs[1], at[1]))


# --------------------------------------------------------------- refusals ---
def test_refusals(gpu):
    announce("refusals (no kernel is launched)")
    x = cpu((4, 64), 1).cuda()
    q, s = ops.quantize_rows(x)
    w, sw = ops.quantize_rows(cpu((32, 64), 2).cuda())
    g = torch.ones(64, dtype=torch.float16, device="cuda")
    no = lambda f, *a, **k: pytest.raises((ValueError, RuntimeError), f, *a, **k)  # noqa: E731
    no(ops.quantize_rows, x.cpu())
    no(ops.quantize_rows, x[0])
    no(ops.quantize_rows, x.t())
    no(ops.quantize_rows, x.to(torch.bfloat16))
    no(ops.quantize_rows, x[:1].expand(4, 64))
    no(ops.quantize_rows, x[:, :0])
    no(ops.quantize_rows, x, out=torch.empty(4, 63, dtype=torch.int8, device="cuda"))
    no(ops.quantize_rows, x, scale=torch.empty(3, device="cuda"))
    no(ops.quantize_rows, x, out=x.view(torch.int8)[:, :64])  # over its own input
    no(ops.dequantize_rows, q, s, dtype=torch.bfloat16)
    no(ops.dequantize_rows, q, s[:3])
    no(ops.rms_norm_q8, x, g[:63])
    no(ops.rms_norm_q8, x, g.float())
    no(ops.rms_norm_q8, x, g, sum_out=x)
    no(ops.rms_norm_q8, x, g, residual=x.float())
    no(ops.rms_norm_q8, x, g, eps=-1.0)
    no(ops.rms_norm_q8, x, g, eps=float("nan"))
    wide = torch.zeros(5, 64, dtype=torch.float16, device="cuda")
    no(ops.rms_norm_q8, wide[:4], g, residual=x, sum_out=wide[1:])  # rows shifted by one
    no(ops.layer_norm_q8, x, g, g[:60])
    no(ops.linear_q8, q, s, w[:, :63], sw)
    no(ops.linear_q8, q, s[:3], w, sw)
    no(ops.linear_q8, q, s, w, sw.half())
    no(ops.linear_q8, q, s, w, sw, act=7)
    no(ops.linear_q8, q, s, w[:24], sw[:24], act=ops.ACT_GEGLU)
    no(ops.linear_q8, q, s, w, sw, dtype=torch.bfloat16)
    no(ops.linear_q8, q, s, w, sw, bias=torch.zeros(31, dtype=torch.float16, device="cuda"))
    no(ops.linear_q8, q, s, w, sw, residual=torch.zeros(4, 32, device="cuda"))  # fp32 with an fp16 output
    no(ops.linear_q8, q, s, w, sw, out=q.view(torch.float16)[:, :32])  # over an input
    ragged = torch.zeros(4 * 50, dtype=torch.int8, device="cuda").view(4, 50)
    no(ops.linear_q8, ragged, s, torch.zeros(8, 64, dtype=torch.int8, device="cuda")[:, :50], sw[:8])
    tight = torch.zeros(3 * 64 + 50, dtype=torch.int8, device="cuda").as_strided((4, 50), (64, 1))
    no(ops.linear_q8, tight, s, torch.zeros(8, 64, dtype=torch.int8, device="cuda")[:, :50], sw[:8])
    # no rows: empty results
    assert ops.linear_q8(q[:0], s[:0], w, sw).shape == (0, 32)
    assert ops.rms_norm_q8(x[:0], g)[0].shape == (0, 64)
    q63, s63 = ops.quantize_rows(x[:, :63])
    w63, sw63 = ops.quantize_rows(cpu((32, 63), 2).cuda())
    assert ops.linear_q8(q63[:0], s63[:0], w63, sw63).shape == (0, 32)
    assert ops.linear_q8(q63, s63, w63[:0], sw63[:0]).shape == (4, 0)
