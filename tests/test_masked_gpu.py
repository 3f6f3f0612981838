"""Rotary positions, query / key norms and masked attention against float64 on the
CPU (GPU).

Every case prints its name before it launches.  u is half a step of the type: 2^-11
for fp16, 2^-8 for bf16; fp32's is 2^-24.
"""
import math

import pytest
import torch

from dollama_amd import _lib, ops
from oracle import masked_ref as M

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
NAMES = {torch.float16: "fp16", torch.bfloat16: "bf16"}


def u(dt):
    return torch.finfo(dt).eps / 2


def announce(msg):
    print(f"[case] {msg}", flush=True)


def rnd(shape, seed, dt=torch.float32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dt)


def inside(shape, dt, fill=77.0):
    """A view of this shape whose surroundings hold `fill` and have to keep it: heads with a
    gap of 8 values between them, tokens with one of a head."""
    B, S, H, Dh = shape
    whole = torch.full((B + 1, S + 2, H + 1, Dh + 8), fill, dtype=dt, device="cuda")
    return whole, whole[:B, 1:S + 1, :H, :Dh]


def untouched(whole, view, fill=77.0):
    w = whole.clone()
    B, S, H, Dh = view.shape
    w[:B, 1:S + 1, :H, :Dh] = fill
    return bool((w == fill).all())


def within(got, want, tol, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: non-finite"
    worst = ((got - want).abs() / tol).max() if got.numel() else torch.zeros(())
    print(f"[parity] {what}: {float(worst):.3f} of the bound", flush=True)
    assert worst <= 1.0, f"{what}: {float(worst)} times the bound"


# ------------------------------------------------------------------ rotary ---
def turn_tol(y, size, dt):
    """One rounding to the type (fp16's smallest step is 2^-24), and in fp32: a turn's
    fraction rounded to 2^-25 of a turn (2e-7 rad), the sine's and cosine's own error below
    2^-18, three products and sums of 2^-24; the norm's sum of squares and root stay below 2^-18
    of the value, on a sum of 256 squares in eight-element chains.  Together under 2^-16 of the pair."""
    return u(dt) * y.abs() * (1 + 2.0 ** -8) + 2.0 ** -16 * size + (2.0 ** -24 if dt == torch.float16 else 0.0)


def positions(B, S, A, kind, far=0):
    n = torch.arange(S)
    p = torch.stack([(n * (3 * a + 1) + 7 * a) % (S + 11 * a + 1) + far * (a == 0) for a in range(A)], 1)
    p = p[None] + torch.arange(B)[:, None, None]
    return p.to(kind)


ROTARY = [
    # Dh, sections, heads, key heads
    (2, [1], 1, 1), (8, [2, 2], 3, 3), (16, [8], 2, 1), (40, [20], 5, 5), (64, [16, 16], 10, 10), (64, [8, 12, 12], 4, 2),
    (72, [36], 7, 7), (80, [8, 16, 16], 13, 13), (96, [48], 6, 3), (128, [8, 28, 28], 32, 8), (128, [64], 5, 1),
    (128, [0, 64, 0], 2, 2), (128, [16, 16], 9, 3), (128, [1, 2], 3, 3), (256, [128], 3, 3), (256, [32, 48, 48], 2, 1),
    (96, [7, 0, 9, 11], 3, 3), (74, [37], 3, 3), (254, [100, 27], 2, 1), (50, [3], 4, 2),
]


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Dh,sections,H,Hkv", ROTARY)
def test_rotary_and_norm(gpu, Dh, sections, H, Hkv, interleaved, dt):
    kinds = [torch.int32, torch.int64, torch.float32]
    for n, (B, S) in enumerate([(1, 1), (2, 5), (1, 67), (3, 33)]):
        announce(f"rotary {B}x{S}x{H}+{Hkv}x{Dh} {sections} interleaved={interleaved} {dt}")
        qkv = rnd((B, S, H + 2 * Hkv, Dh), Dh + n, dt, 2.0)
        dev = qkv.cuda()
        q, k = qkv[:, :, :H], qkv[:, :, H:H + Hkv]
        dq, dk = dev[:, :, :H], dev[:, :, H:H + Hkv]
        gq, gk = rnd((Dh,), 3, dt, 0.3) + 1, rnd((Dh,), 4, dt, 0.3) + 1
        kind = kinds[n % 3]
        pos = positions(B, S, len(sections), kind, far=[0, 1000, 10 ** 6, 0][n])
        if kind == torch.float32:
            pos = pos + 0.25
        f = ops.rotary_freqs(sections, shared=n == 1)
        fc = f.cpu()
        # alone
        y, size = M.rotary(q, pos, fc, sections, interleaved)
        whole, out = inside((B, S, H, Dh), dt)
        got = ops.rotary_axes(dq, pos.cuda(), f, sections, interleaved=interleaved, out=out)
        assert got is out and untouched(whole, out)
        within(out, y, turn_tol(y, size, dt), "rotary")
        assert torch.equal(ops.rotary_axes(dq, pos.cuda(), f, sections, interleaved=interleaved), out.contiguous())
        # with the norms
        a, b = ops.qk_norm_rotary(dq, dk, gq.cuda(), gk.cuda(), pos.cuda(), f, sections, interleaved=interleaved, eps=1e-5)
        for got, x, g, what in ((a, q, gq, "norm q"), (b, k, gk, "norm k")):
            y, size = M.rotary(M.norm(x, g, 1e-5), pos, fc, sections, interleaved)
            within(got, y, turn_tol(y, size, dt), what)
        # in place, inside the fused projection, whose values stay
        v = dev[:, :, H + Hkv:].clone()
        c, d = ops.qk_norm_rotary(dq, dk, gq.cuda(), gk.cuda(), pos.cuda(), f, sections, interleaved=interleaved, eps=1e-5,
                                  q_out=dq, k_out=dk)
        assert torch.equal(c, a) and torch.equal(d, b) and torch.equal(dev[:, :, H + Hkv:], v)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_rotary_of_unaligned_and_head_major_views(gpu, dt):
    B, S, H, Dh = 2, 19, 3, 64
    sections = [12, 20]
    pos = positions(B, S, 2, torch.int32)
    f = ops.rotary_freqs(sections)
    want = None
    for shift in (0, 1, 2, 4):
        announce(f"rotary at {shift} elements past alignment {dt}")
        x = rnd((B, S, H, Dh), 5, dt)
        flat = torch.zeros(x.numel() + 8, dtype=dt, device="cuda")
        d = flat[shift:shift + x.numel()].view(B, S, H, Dh)
        d.copy_(x)
        y, size = M.rotary(x, pos, f.cpu(), sections, False)
        got = ops.rotary_axes(d, pos.cuda(), f, sections)
        within(got, y, turn_tol(y, size, dt), "rotary")
        want = got if want is None else want
        assert torch.equal(got, want)  # no vector width changes a result
    announce("rotary of head-major views, positions of one line for every batch")
    hm = rnd((B, H, S, Dh), 6, dt)
    y, size = M.rotary(hm.transpose(1, 2), pos[:1], f.cpu(), sections, True)
    dev = hm.cuda()
    ops.rotary_axes(dev.transpose(1, 2), pos[0].cuda(), f, sections, interleaved=True, out=dev.transpose(1, 2))
    within(dev.transpose(1, 2), y, turn_tol(y, size, dt), "head-major")


def test_norm_at_the_ends_of_the_range(gpu):
    """Squares past fp32's range on both sides, zeros, infinities and NaN."""
    announce("norm of huge and tiny bf16 heads")
    x = rnd((1, 8, 2, 128), 7)
    f = torch.tensor([1.0, 1e30, 1e38, 1e-20, 1e-30, 1e-38, 3e19, 1e-15])
    x = (x / x.abs().amax(-1, keepdim=True) * f[None, :, None, None]).to(torch.bfloat16)
    for eps in (0.0, 1e-38, 1e-6):
        y = M.norm(x, None, eps)
        got, _ = ops.qk_norm_rotary(x.cuda(), eps=eps)
        # (an output below bf16's normal range may lose its last bits)
        within(got, y, turn_tol(y, y.abs(), torch.bfloat16) + 2.0 ** -126, f"eps={eps}")
    h = (rnd((1, 4, 1, 64), 8) * torch.tensor([1.0, 65504.0, 2.0 ** -24, 6e-8])[None, :, None, None]).clamp(-65504, 65504)
    h = h.half()
    y = M.norm(h, None, 1e-20)
    keep = h.double().square().sum(-1) > 0
    got, _ = ops.qk_norm_rotary(h.cuda(), eps=1e-20)
    within(got[keep], y[keep], turn_tol(y[keep], y[keep].abs(), torch.float16), "fp16")
    announce("norm of heads with zeros, infinities and NaN")
    z = rnd((1, 4, 2, 80), 9, torch.float16)
    z[0, 0] = 0
    z[0, 1, 0, 3] = float("inf")
    z[0, 2, 1, 5] = float("nan")
    got, _ = ops.qk_norm_rotary(z.cuda(), eps=1e-6)
    got = got.cpu()
    assert (got[0, 0] == 0).all()
    assert got[0, 1, 0, 3].isnan() and (got[0, 1, 0, torch.arange(80) != 3] == 0).all()
    assert got[0, 2, 1].isnan().all()
    ok = torch.ones(4, 2, dtype=torch.bool)
    ok[1, 0] = ok[2, 1] = False
    y = M.norm(z, None, 1e-6)
    within(got[0][ok], y[0][ok], turn_tol(y[0][ok], y[0][ok].abs(), torch.float16), "their neighbours")


# --------------------------------------------------------------- attention ---
def att_tol(ref, n, dt, v):
    """u for the weights' rounding, in the product and in their sum; the scores' errors
    (units of 2^-24) likewise; sums of n terms, 16 to a matrix instruction or two to a dot
    product over a quarter of them; the output's rounding.  fp16 weights are at least 2^7 at the
    base, so those below the normal range lose n 2^-25 / 2^7 of the largest value."""
    e = ref["err"] * 2.0 ** -24
    e = torch.expm1(e.clamp_max(5.0))
    chain = (n / 4 + 64) * 2.0 ** -24
    tol = 2 * (u(dt) * (1 + e) + e + 2.0 ** -21 + chain) * ref["A"] + u(dt) * ref["o"].abs()
    small = n * 2.0 ** -31 + 2.0 ** -24 if dt == torch.float16 else 2.0 ** -126
    return tol + small * float(v[torch.isfinite(v)].abs().max() if v.numel() else 1.0)


def attend(q, k, v, what, out=None, **kw):
    """The operator on the GPU against the definition."""
    announce(what)
    ref = M.attention(q, k, v, **kw)
    dev = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    got = ops.attention_masked(q.cuda(), k.cuda(), v.cuda(), out=out, **dev)
    within(got, ref["o"], att_tol(ref, k.shape[1], q.dtype, v), what)
    return got


def qkv(B, Sq, Sk, H, Hkv, Dh, dt, seed=0, std=1.5):
    return rnd((B, Sq, H, Dh), seed, dt, std), rnd((B, Sk, Hkv, Dh), seed + 1, dt, std), rnd((B, Sk, Hkv, Dh), seed + 2, dt)


SIZES = [
    # B, Sq, Sk, H, Hkv, Dh: few rows, their ends, the many-row kernel, both split over the keys
    (1, 1, 1, 1, 1, 8), (2, 1, 33, 4, 1, 64), (1, 3, 31, 2, 2, 40), (2, 1, 700, 8, 2, 128), (1, 5, 1500, 16, 2, 128),
    (1, 33, 65, 1, 1, 64), (1, 64, 130, 2, 2, 72), (1, 65, 64, 1, 1, 80), (2, 77, 77, 3, 3, 64), (1, 129, 257, 2, 1, 96),
    (1, 200, 511, 5, 1, 128), (2, 128, 128, 2, 2, 88), (1, 130, 300, 2, 1, 256), (1, 2, 600, 3, 1, 256), (1, 70, 1300, 2, 2, 104),
    (3, 17, 95, 6, 2, 16), (1, 31, 2100, 1, 1, 128),
]


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_attention_sizes_and_modes(gpu, size, dt):
    B, Sq, Sk, H, Hkv, Dh = size
    q, k, v = qkv(*size, dt, seed=sum(size))
    whole, out = inside((B, Sq, H, Dh), dt)
    name = "x".join(map(str, size)) + " " + NAMES[dt]
    attend(q, k, v, f"{name} plain", out=out)
    assert untouched(whole, out)
    attend(q, k, v, f"{name} causal", causal=True)  # with Sq > Sk the first queries see nothing
    slopes = torch.exp2(-8 * torch.arange(1, H + 1) / H)
    table = rnd((H, 2 * 20 + 1), 5)
    attend(q, k, v, f"{name} cap", cap=20.0)
    attend(q, k, v, f"{name} tight cap", cap=2.0, scale=0.4)
    attend(q, k, v, f"{name} slopes causal cap", causal=True, slopes=slopes, cap=30.0)
    attend(q, k, v, f"{name} table", rel_bias=table)
    attend(q, k, v, f"{name} table of one entry, causal", rel_bias=rnd((H, 1), 6), causal=True)
    attend(q, k, v, f"{name} scale", scale=1.7)
    g = torch.Generator().manual_seed(1)
    a = torch.randint(-3, Sk + 3, (B, Sq, 2), generator=g)
    window = torch.stack([a.amin(-1), a.amax(-1)], -1).to(torch.int32)  # some leave nothing
    attend(q, k, v, f"{name} intervals", key_range=window)
    place = torch.randint(-5, Sk + 5, (B, Sq), generator=g).to(torch.int32)
    attend(q, k, v, f"{name} intervals, places, causal, table", key_range=window, q_pos=place, causal=True, rel_bias=table)
    attend(q, k, v, f"{name} one line of intervals and places", key_range=window[0], q_pos=place[0], slopes=slopes)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_attention_documents_prefix_lengths(gpu, dt):
    lengths = [1, 100, 63, 64, 65, 0, 7, 128, 200]
    r = ops.document_ranges(lengths, tokens=640, device="cpu")
    q, k, v = qkv(1, 640, 640, 4, 2, 64, dt, 11)
    got = attend(q, k, v, "documents with padding behind them", key_range=r)
    assert (got[0, sum(lengths):] == 0).all()
    attend(q, k, v, "documents in order", key_range=r, causal=True, cap=15.0)
    # a document's result is the one it has alone
    at = 0
    for n in lengths:
        if n:
            alone = ops.attention_masked(q[:, at:at + n].cuda(), k[:, at:at + n].cuda(), v[:, at:at + n].cuda())
            ref = M.attention(q[:, at:at + n], k[:, at:at + n], v[:, at:at + n])
            within(alone, ref["o"], att_tol(ref, n, dt, v), f"document of {n} alone")
        at += n
    q, k, v = qkv(3, 150, 150, 6, 2, 80, dt, 12)
    attend(q, k, v, "prefixes", key_range=ops.prefix_ranges([0, 50, 149], 150, device="cpu"))
    q, k, v = qkv(3, 20, 150, 6, 2, 80, dt, 13)
    attend(q, k, v, "prefixes, the last queries", key_range=ops.prefix_ranges([0, 140, 150], 20, 150, device="cpu"))
    n = torch.tensor([1, 77, 900, 513, 64])
    q, k, v = qkv(5, 1, 900, 8, 2, 128, dt, 14)
    attend(q, k, v, "a cache in use up to a length", q_pos=(n - 1)[:, None].to(torch.int32), causal=True, cap=50.0)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_documents_that_share_row_blocks(gpu, dt):
    """Workgroups of 128 rows that hold the end of one document and the start of others, long
    and short, apart and not, with the keys in one part and in several."""
    cases = [(1, 1, 64, [700, 650]), (2, 2, 64, [100, 1300, 90]), (2, 1, 96, [64, 64, 900, 10, 500]),
             (4, 4, 64, [300, 280, 310, 290, 305]), (1, 1, 128, [1000, 1, 1, 1000]), (6, 3, 80, [257, 700, 3, 385]),
             (2, 2, 256, [300, 400]), (8, 1, 64, [150, 200, 170])]
    for H, Hkv, Dh, lengths in cases:
        S = sum(lengths)
        q, k, v = qkv(1, S, S, H, Hkv, Dh, dt, S)
        r = ops.document_ranges(lengths, device="cpu")
        attend(q, k, v, f"documents {lengths} x{H}/{Hkv}x{Dh} {dt}", key_range=r)
        attend(q, k, v, f"documents {lengths}, causal, cap", key_range=r, causal=True, cap=20.0)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("B,S,H,Hkv,Dh", [(1, 129, 3, 3, 64), (2, 700, 5, 5, 40), (3, 400, 7, 7, 64), (1, 1300, 9, 3, 64),
                                          (5, 260, 4, 2, 128)])
def test_row_blocks_of_every_head_in_any_order(gpu, B, S, H, Hkv, Dh, dt):
    """Causal rows of several heads and batches: each row block is taken once."""
    q, k, v = qkv(B, S, S, H, Hkv, Dh, dt, S)
    attend(q, k, v, f"causal {B}x{S}x{H}/{Hkv}x{Dh} {dt}", causal=True)


@pytest.mark.parametrize("Sq,Sk,H,Hkv,Dh", [(1, 20000, 1, 1, 64), (1, 5000, 2, 1, 128), (1, 4100, 3, 3, 256), (3, 16500, 2, 1, 80),
                                            (50, 9000, 1, 1, 64), (70, 6000, 2, 2, 128), (40, 3000, 1, 1, 256)])
def test_keys_in_many_parts(gpu, Sq, Sk, H, Hkv, Dh):
    q, k, v = qkv(1, Sq, Sk, H, Hkv, Dh, torch.bfloat16, Sk)
    name = f"{Sq}x{Sk}x{H}/{Hkv}x{Dh}"
    attend(q, k, v, f"{name} in parts", causal=True)
    few = torch.tensor([[Sk // 2, Sk // 2 + 40]], dtype=torch.int32).expand(Sq, 2).contiguous()
    attend(q, k, v, f"{name}, keys in few of the parts", key_range=few)
    few[::2] = torch.tensor([Sk - 1, 3], dtype=torch.int32)
    attend(q, k, v, f"{name}, every other row without keys", key_range=few, cap=10.0)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_caps_and_tables_of_any_size(gpu, dt):
    for Sq, Sk in ((1, 90), (140, 200)):
        q, k, v = qkv(1, Sq, Sk, 2, 1, 64, dt, Sk)
        for cap, scale in ((1e6, None), (1e-3, None), (5.0, 1e-3), (3e4, 1.0), (0.5, 1.0), (1e5, 8.0)):
            attend(q, k, v, f"cap {cap}, scale {scale}, {Sq}x{Sk}", cap=cap, scale=scale)
        for R in (0, 63, 255, 256, 600):  # in LDS up to 1024 entries of a key head's heads
            t = rnd((2, 2 * R + 1), R)
            attend(q, k, v, f"table of R = {R}, {Sq}x{Sk}", rel_bias=t)
            attend(q, k, v, f"table of R = {R} under a cap, {Sq}x{Sk}", rel_bias=t, cap=6.0, causal=True)


def test_attention_of_nothing(gpu):
    announce("no keys, no queries, no batch, a mask of nothing")
    q, k, v = (t.cuda() for t in qkv(2, 3, 0, 4, 2, 64, torch.float16))
    assert (ops.attention_masked(q, k, v) == 0).all()
    assert (ops.attention_masked(q, k, v, causal=True, cap=3.0) == 0).all()
    assert ops.attention_masked(q[:, :0], k, v).shape == (2, 0, 4, 64)
    assert ops.attention_masked(q[:0], k[:0], v[:0]).shape == (0, 3, 4, 64)
    for Sq in (2, 90):
        q, k, v = (t.cuda() for t in qkv(2, Sq, 700, 4, 4, 64, torch.bfloat16))
        none = torch.tensor([5, 5], dtype=torch.int32, device="cuda").expand(2, Sq, 2).contiguous()
        assert (ops.attention_masked(q, k, v, key_range=none) == 0).all()
        none[:, :, 0], none[:, :, 1] = 2 ** 31 - 1, -2 ** 31
        assert (ops.attention_masked(q, k, v, key_range=none) == 0).all()
        far = torch.full((2, Sq), -2 ** 31, dtype=torch.int32, device="cuda")
        assert (ops.attention_masked(q, k, v, q_pos=far, causal=True) == 0).all()


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("Sq,Sk,H,Hkv,Dh", [(1, 300, 4, 1, 64), (200, 200, 2, 2, 64), (140, 140, 4, 2, 128), (3, 100, 2, 2, 256),
                                            (100, 100, 2, 2, 256), (90, 700, 2, 1, 80)])
def test_what_masked_keys_hold_has_no_effect(gpu, Sq, Sk, H, Hkv, Dh, dt):
    inf, nan = float("inf"), float("nan")
    q, k, v = qkv(2, Sq, Sk, H, Hkv, Dh, dt, 21)
    p = torch.arange(Sk - Sq, Sk)
    bad = Sk - 1 - (Sq - 1) // 2  # half of the causal queries come before it
    n = max(1, Sk // 2)
    cases = {"causal": dict(causal=True), "length": dict(key_range=torch.tensor([3, n], dtype=torch.int32).expand(2, Sq, 2))}
    for name, kw in cases.items():
        kw = {a: b.contiguous() if isinstance(b, torch.Tensor) else b for a, b in kw.items()}
        dev = {a: b.cuda() if isinstance(b, torch.Tensor) else b for a, b in kw.items()}
        at = [bad, min(Sk - 1, bad + 1)] if name == "causal" else [0, 2, n, Sk - 1]
        for what, x in (("NaN", nan), ("infinity", inf), ("-infinity", -inf)):
            announce(f"{what} in masked keys, {name}, {Sq}x{Sk}x{Dh} {dt}")
            k2, v2 = k.clone(), v.clone()
            v2[0, at] = x
            k2[0, at, :, ::3] = x
            v2[1, at, :, 1] = x
            m, _ = M.visible(2, Sq, Sk, kw.get("key_range"), None, kw.get("causal", False))
            sees = m[:, :, at].any(-1)
            ref = M.attention(q, k, v, **kw)
            got = ops.attention_masked(q.cuda(), k2.cuda(), v2.cuda(), **dev).cpu()
            tol = att_tol(ref, Sk, dt, v)
            within(got[~sees], ref["o"][~sees], tol[~sees], f"{name}, {what}: rows that do not see it")
            # and rows that do: batch 1 has it in one dim of V alone
            if sees[1].any():
                s1 = got[1][sees[1]]
                assert (s1[..., 1].isnan() if what == "NaN" else s1[..., 1] == x).all(), what
                rest = [d for d in range(Dh) if d != 1]
                within(s1[..., rest], ref["o"][1][sees[1]][..., rest], tol[1][sees[1]][..., rest], "their other dims")
            if sees[0].any():
                assert not torch.isfinite(got[0][sees[0]]).any()


@pytest.mark.parametrize("mode", ["plain", "cap", "slopes", "table", "cap and table"])
def test_masked_keys_change_no_bit(gpu, mode):
    """The same bits whatever masked keys hold: zeros, large values, infinities, NaN; short rows
    and long ones, an interval that ends inside a tile at both ends."""
    H = 2
    kw = {"plain": {}, "cap": dict(cap=30.0), "slopes": dict(slopes=torch.tensor([0.1, 0.01]).cuda()),
          "table": dict(rel_bias=rnd((H, 41), 1).cuda()), "cap and table": dict(cap=30.0, rel_bias=rnd((H, 41), 1).cuda())}[mode]
    for Sq, Sk in ((3, 200), (150, 300)):
        q, k, v = (t.cuda() for t in qkv(1, Sq, Sk, H, H, 64, torch.float16, 27))
        r = torch.tensor([[37, Sk - 45]], dtype=torch.int32, device="cuda").expand(Sq, 2).contiguous()
        want = None
        for x in (0.0, 60000.0, float("inf"), -float("inf"), float("nan")):
            announce(f"masked keys of {x}, {mode}, {Sq}x{Sk}")
            k2, v2 = k.clone(), v.clone()
            for t in (k2, v2):
                t[:, :37] = x
                t[:, Sk - 45:] = x
            got = ops.attention_masked(q, k2, v2, key_range=r, **kw)
            want = got if want is None else want
            assert torch.isfinite(got).all() and torch.equal(got, want), f"{mode}: {x}"


@pytest.mark.parametrize("Sq", [1, 100])
def test_values_at_the_end_of_bf16s_range(gpu, Sq):
    """Sums of weights times values stay in fp32 while a row's scores grow from tile to tile."""
    announce(f"values of 1e36 under growing scores, {Sq} rows")
    Sk = 500
    q, k, v = qkv(1, Sq, Sk, 1, 1, 64, torch.bfloat16, 28)
    k = (k.float() * torch.linspace(0.2, 3, Sk)[None, :, None, None]).bfloat16()
    small = M.attention(q, k, v)
    got = ops.attention_masked(q.cuda(), k.cuda(), (v.float() * 2.0 ** 116).bfloat16().cuda()).double() * 2.0 ** -116
    within(got, small["o"], att_tol(small, Sk, torch.bfloat16, v), "values of 2^116")


@pytest.mark.parametrize("cap", [0.5, 1e3, 1e4, 1e6, 3e38])
@pytest.mark.parametrize("bias", [False, True], ids=["cap", "cap and slopes"])
def test_small_scores_under_large_caps(gpu, cap, bias):
    """A capped score's error goes by the score, not by the cap (below a half of it, where the cap is a
    polynomial: 8 units of the score, less than the product's own error, so twice that); above,
    units of the cap."""
    for Sq, Sk in ((2, 300), (150, 200)):
        announce(f"cap {cap}, {Sq}x{Sk}, slopes {bias}")
        q, k, v = qkv(1, Sq, Sk, 2, 2, 64, torch.float16, 29)
        kw = dict(slopes=torch.tensor([0.05, 0.01])) if bias else {}
        ref = M.attention(q, k, v, cap=cap, **kw)
        ref["err"] = 2 * M.attention(q, k, v, **kw)["err"] + (16 * cap if cap < 100 else 0.0)
        dev = {n: t.cuda() for n, t in kw.items()}
        got = ops.attention_masked(q.cuda(), k.cuda(), v.cuda(), cap=cap, **dev)
        within(got, ref["o"], att_tol(ref, Sk, torch.float16, v), f"cap {cap}")


@pytest.mark.parametrize("mode", ["slopes", "table"])
def test_places_at_both_ends(gpu, mode):
    """Places of +-2^30 among the rows of one wave."""
    kw = dict(slopes=torch.tensor([1e-9])) if mode == "slopes" else dict(rel_bias=rnd((1, 11), 3))
    for Sq in (4, 140):
        q, k, v = qkv(1, Sq, 90, 1, 1, 64, torch.float16, 30)
        places = torch.tensor([-(1 << 30), 1 << 30, 0, 89], dtype=torch.int32).repeat(35)[:Sq].contiguous()
        attend(q, k, v, f"places at both ends, {Sq} rows, {mode}", q_pos=places, **kw)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("Sq,Sk", [(1, 400), (150, 150)])
def test_tables_of_infinities_and_lowest_values(gpu, Sq, Sk, dt):
    q, k, v = qkv(1, Sq, Sk, 3, 3, 64, dt, 31)
    low = torch.finfo(torch.float32).min
    R = 40
    t = rnd((3, 2 * R + 1), 32)
    t[0, 45:] = -math.inf      # no key five or more behind the query
    t[0, ::3] = low            # weightless beside any other
    t[1, :] = low              # every key alike: the mean of what a query sees
    t[2, :] = -math.inf        # nothing
    v2 = v.clone()
    announce(f"table of -infinity and the lowest value {Sq}x{Sk} {dt}")
    # (scores vanish beside the lowest value, in fp32 as in any other arithmetic of them: bias alone)
    ref = M.attention(q, k, v, rel_bias=t)
    got = ops.attention_masked(q.cuda(), k.cuda(), v2.cuda(), rel_bias=t.cuda()).cpu()
    assert (got[:, :, 2] == 0).all()
    flat = ref["err"].clone()
    ref["err"][:, :, 1] = 0.0
    mean = v.double()[:, :, 1].mean(1, keepdim=True).expand(1, Sq, 64)
    ref["o"][:, :, 1] = mean
    ref["err"][:, :, 0] = M.attention(q, k, v, rel_bias=torch.where(t == low, -math.inf, t))["err"][:, :, 0]
    assert flat.shape == ref["err"].shape
    within(got[:, :, :2], ref["o"][:, :, :2], att_tol(ref, Sk, dt, v)[:, :, :2], "table")
    # keys that a -infinity hides may hold anything
    v2[0, -1, 2] = float("nan")
    v2[0, 0, 2] = float("inf")
    got = ops.attention_masked(q.cuda(), k.cuda(), v2.cuda(), rel_bias=t.cuda()).cpu()
    assert (got[:, :, 2] == 0).all()


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_scores_of_any_size(gpu, dt):
    """Peaked rows: the base moves up and down by thousands between tiles."""
    for Sq, Sk in ((2, 500), (130, 500)):
        q, k, v = qkv(1, Sq, Sk, 2, 2, 64, dt, 41, std=8.0)
        attend(q, k, v, f"large scores {Sq}x{Sk}")
        attend(q, k, v, f"large scores under a large cap {Sq}x{Sk}", cap=500.0)
        k = (k.float() * torch.linspace(-3, 3, Sk)[None, :, None, None]).to(dt)
        attend(q, k, v, f"growing scores {Sq}x{Sk}", scale=0.5, slopes=torch.tensor([0.0, 3.0]))
        attend(q, k * 0, v, f"equal scores {Sq}x{Sk}")
        attend(q, k, v, f"tiny scale {Sq}x{Sk}", scale=1e-30)


def test_flat_rows_keep_their_weights(gpu):
    """One key far above very many: fp16 weights far below the largest still count."""
    announce("one key above 60000 others by 2^13")
    Sk = 60000
    q = torch.zeros(1, 1, 1, 64, dtype=torch.float16)
    q[..., 0] = 8.0
    k = torch.zeros(1, Sk, 1, 64, dtype=torch.float16)
    k[0, 0, 0, 0] = 13 * math.log(2)
    v = torch.ones(1, Sk, 1, 64, dtype=torch.float16)
    v[0, 0] = 0
    for Sq in (1, 70):
        qq = q.expand(1, Sq, 1, 64).contiguous()
        ref = M.attention(qq, k, v, scale=0.125)
        got = ops.attention_masked(qq.cuda(), k.cuda(), v.cuda(), scale=0.125)
        within(got, ref["o"], att_tol(ref, Sk, torch.float16, v), f"{Sq} rows")


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_attention_of_strided_operands(gpu, dt):
    B, S, H, Hkv, Dh = 2, 100, 4, 2, 64
    x = rnd((B, S, H + 2 * Hkv, Dh), 51, dt)
    d = x.cuda()
    ref = M.attention(x[:, :, :H], x[:, :, H:H + Hkv], x[:, :, H + Hkv:], causal=True)
    tol = att_tol(ref, S, dt, x)
    announce("slices of a fused projection")
    got = ops.attention_masked(d[:, :, :H], d[:, :, H:H + Hkv], d[:, :, H + Hkv:], causal=True)
    within(got, ref["o"], tol, "fused")
    announce("head-major operands")
    hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (d[:, :, :H], d[:, :, H:H + Hkv], d[:, :, H + Hkv:])]
    out = torch.empty(B, H, S, Dh, dtype=dt, device="cuda").transpose(1, 2)
    assert torch.equal(ops.attention_masked(*hm, causal=True, out=out), got)
    announce("no batch dimension, masks of one line")
    one = ops.attention_masked(d[1, :, :H], d[1, :, H:H + Hkv], d[1, :, H + Hkv:], causal=True)
    assert torch.equal(one, got[1])  # nor does the batch change a row
    announce("queries and masks shared by the batch")
    qs = d[:1, :, :H].expand(B, S, H, Dh)
    same = ops.attention_masked(qs, d[:, :, H:H + Hkv], d[:, :, H + Hkv:], causal=True)
    assert torch.equal(same[0], got[0])


def test_offsets_past_32_bits(gpu):
    """Keys 4 MiB apart, 2.5 GiB of them, behind a batch of the same: byte offsets past 2^32
    and element offsets past 2^31."""
    announce("keys 2^21 elements apart, two batches of 640")
    Sk, step = 640, 1 << 21
    big = torch.empty(2 * Sk * step, dtype=torch.float16, device="cuda")
    view = big.view(2, Sk, step)[:, :, :128].view(2, Sk, 2, 64)
    kv = rnd((2, Sk, 2, 64), 61, torch.float16)
    view.copy_(kv)
    k, v = view[:, :, :1], view[:, :, 1:]
    for Sq in (1, 80):
        q = rnd((2, Sq, 1, 64), 62, torch.float16, 1.5)
        ref = M.attention(q, kv[:, :, :1], kv[:, :, 1:], causal=True)
        got = ops.attention_masked(q.cuda(), k, v, causal=True)
        within(got, ref["o"], att_tol(ref, Sk, torch.float16, kv), f"{Sq} queries")


# ------------------------------------------- streams, graphs, the whole path ---
def layer(x, H, Hkv, gq, gk, pos, f, sections, cache, at, lens, out):
    """One attention layer over a cache: norms and rotation (keys into the cache), attention."""
    k, v = cache
    S = x.shape[1]
    q, _ = ops.qk_norm_rotary(x[:, :, :H], x[:, :, H:H + Hkv], gq, gk, pos, f, sections, k_out=k[:, at:at + S])
    v[:, at:at + S].copy_(x[:, :, H + Hkv:])
    return ops.attention_masked(q, k, v, q_pos=lens, causal=True, cap=30.0, out=out)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_a_prompt_and_its_tokens_through_the_operators(gpu, dt):
    """A prompt of 90 tokens, then single tokens, against the whole sequence in float64: queries
    and keys turned by three axes, kept rounded to the type as the cache does."""
    B, S, H, Hkv, Dh, n = 2, 96, 8, 2, 64, 90
    sections = [8, 12, 12]
    x = rnd((B, S, H + 2 * Hkv, Dh), 71, dt)
    gq, gk = rnd((Dh,), 72, dt, 0.2) + 1, rnd((Dh,), 73, dt, 0.2) + 1
    pos = positions(B, S, 3, torch.int32)
    f = ops.rotary_freqs(sections)
    cache = [torch.full((B, 128, Hkv, Dh), float("nan"), dtype=dt, device="cuda") for _ in range(2)]
    outs = []
    for at, m in [(0, n)] + [(i, 1) for i in range(n, S)]:
        announce(f"tokens {at} to {at + m} {dt}")
        lens = torch.arange(at, at + m, dtype=torch.int32, device="cuda").expand(B, m).contiguous()
        outs.append(layer(x[:, at:at + m].cuda(), H, Hkv, gq.cuda(), gk.cuda(), pos[:, at:at + m].cuda(), f, sections, cache,
                          at, lens, None))
    got = torch.cat(outs, 1)
    q, sq = M.rotary(M.norm(x[:, :, :H], gq, 1e-6), pos, f.cpu(), sections, False)
    k, sk = M.rotary(M.norm(x[:, :, H:H + Hkv], gk, 1e-6), pos, f.cpu(), sections, False)
    ref = M.attention(q, k, x[:, :, H + Hkv:], causal=True, cap=30.0)
    # queries and keys each off by their bound: the scores by |q| |dk| + |dq| |k|
    dq, dk = turn_tol(q, sq, dt), turn_tol(k, sk, dt)
    kk = k.abs().repeat_interleave(H // Hkv, 2).permute(0, 2, 3, 1)
    dkk = dk.repeat_interleave(H // Hkv, 2).permute(0, 2, 3, 1)
    ds = (q.abs().transpose(1, 2) @ dkk + dq.transpose(1, 2) @ (kk + dkk)) * Dh ** -0.5
    ds = ds.masked_fill(~M.visible(B, S, S, causal=True)[0][:, None], 0.0).amax(-1, keepdim=True).transpose(1, 2)
    ref["err"] = ref["err"] + ds * 2.0 ** 24
    within(got, ref["o"], att_tol(ref, S, dt, x), "the layer")


def test_captured_calls_replay(gpu):
    """Two graphs that split over the keys, replayed in turn and with eager calls between."""
    announce("two captured graphs with workspaces")
    f = ops.rotary_freqs([32])
    state = []
    for i, Sk in enumerate((3000, 2000)):
        x, k, v = (t.cuda() for t in qkv(2, 1, Sk, 8, 2, 64, torch.float16, 80 + i))
        pos = torch.full((2, 1, 1), Sk - 1, dtype=torch.int32, device="cuda")
        lens = torch.full((2, 1), Sk - 1, dtype=torch.int32, device="cuda")
        out = torch.empty_like(x)

        def go(x=x, k=k, v=v, pos=pos, lens=lens, out=out):
            q, _ = ops.qk_norm_rotary(x, None, None, None, pos, f, [32])
            ops.attention_masked(q, k, v, q_pos=lens, causal=True, out=out)

        go()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go()
        state.append((x, lens, pos, out, go, g, Sk))
    for turn in range(4):
        for x, lens, pos, out, go, g, Sk in state:
            x.copy_(rnd(tuple(x.shape), 90 + turn, torch.float16).cuda())
            lens.fill_(Sk - 1 - 37 * turn)
            pos.fill_(Sk - 1 - 37 * turn)
            go()
            want = out.clone()
            out.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), f"replay {turn}"
    # both replays in flight at once, on streams of their own
    wants = []
    for x, lens, pos, out, go, g, Sk in state:
        go()
        wants.append(out.clone())
        out.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, (x, lens, pos, out, go, g, Sk) in zip(streams, state):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, st in zip(wants, state):
        assert torch.equal(st[3], w)


def test_calls_on_another_stream_and_repeated(gpu):
    announce("a side stream, and the same bits every time")
    q, k, v = (t.cuda() for t in qkv(2, 40, 3000, 8, 2, 128, torch.bfloat16, 95))
    want = ops.attention_masked(q, k, v, causal=True, cap=20.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.attention_masked(q, k, v, causal=True, cap=20.0) for _ in range(3)]
    s.synchronize()
    for g in got:
        assert torch.equal(g, want)


def test_two_calls_at_once(gpu):
    """Calls with parts of the keys on two streams, each with a workspace of its own."""
    announce("two streams, parts of 20000 keys")
    q, k, v = (t.cuda() for t in qkv(1, 4, 20000, 32, 8, 128, torch.bfloat16, 31))
    other = q * 0.5
    want = [ops.attention_masked(x, k, v) for x in (q, other)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, x in enumerate((q, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.attention_masked(x, k, v))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_wrappers_refuse_on_the_gpu(gpu):
    announce("refused calls")
    q, k, v = (t.cuda() for t in qkv(2, 4, 9, 4, 2, 64, torch.float16))
    A = ops.attention_masked
    for bad, kw in [
        (lambda: A(q.float(), k, v), "float16 or bfloat16"),
        (lambda: A(q, k.bfloat16(), v), "float16"),
        (lambda: A(q.cpu(), k, v), "current GPU"),
        (lambda: A(q, k[:, :, :, :32], v), "must be"),
        (lambda: A(q, k, v[:, :8]), "must be"),
        (lambda: A(q, k, v, q_pos=torch.zeros(2, 4, device="cuda")), "int32"),
        (lambda: A(q, k, v, key_range=torch.zeros(3, 4, 2, dtype=torch.int32, device="cuda")), "key_range"),
        (lambda: A(q, k, v, rel_bias=torch.zeros(4, 8, device="cuda")), "2R"),
        (lambda: A(q, k, v, slopes=torch.zeros(3, device="cuda")), "slopes"),
        (lambda: A(q, k, v, out=torch.empty(2, 4, 4, 32, dtype=torch.float16, device="cuda")), "out"),
        (lambda: A(q.transpose(2, 3).contiguous().transpose(2, 3), k, v), "consecutive"),
    ]:
        with pytest.raises(ValueError, match=kw):
            bad()
    for bad, kw in [
        (lambda: A(q, k, v, out=q), "overlaps q"),
        (lambda: A(q, k, v, scale=0.0), "scale"),
        (lambda: A(q, k, v, cap=-1.0), "cap"),
        (lambda: A(q[:, :, :3], k, v), "multiple of Hkv"),
    ]:
        with pytest.raises(_lib.DlmError, match=kw):
            bad()
    f = ops.rotary_freqs([16, 16])
    pos = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for bad, kw in [
        (lambda: ops.rotary_axes(q, pos, f, [16]), "positions"),
        (lambda: ops.rotary_axes(q, pos, f[:8], [16, 16]), "freqs"),
        (lambda: ops.rotary_axes(q, pos, f.float(), [16, 16]), "freqs"),
        (lambda: ops.rotary_axes(q, pos.short(), f, [16, 16]), "positions"),
        (lambda: ops.rotary_axes(q, pos, f, [16, -16]), "negative"),
        (lambda: ops.qk_norm_rotary(q, None, k_out=k), "need k"),
        (lambda: ops.qk_norm_rotary(q, None, torch.ones(32, device="cuda").half()), "q_gamma"),
    ]:
        with pytest.raises(ValueError, match=kw):
            bad()
    with pytest.raises(_lib.DlmError, match="more pairs"):
        ops.rotary_axes(q, pos, ops.rotary_freqs([16, 17]), [16, 17])
    with pytest.raises(_lib.DlmError, match="overlaps"):
        ops.rotary_axes(q[:, :2], pos[:2], f, [16, 16], out=q[:, 1:3])
