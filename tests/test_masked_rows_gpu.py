"""Masked attention's rows beside one another: no row's result shows what another row's query, keys or
place hold, nor what keys hold that a table hides from it; scores, values, slopes and caps at the ends of their
ranges; row blocks that workgroups share (GPU)."""
import ctypes
import math

import pytest
import torch

from dollama_amd import _lib, ops
from oracle import masked_ref as M
from test_masked_gpu import HALF, NAMES, announce, att_tol, attend, qkv, rnd, turn_tol, within

pytestmark = pytest.mark.gpu

MODES = ["plain", "cap", "slopes", "table", "cap and slopes", "cap and table"]


def scores_kw(mode, H):
    kw = {"cap": 30.0} if "cap" in mode else {}
    if "slopes" in mode:
        kw["slopes"] = torch.exp2(-8 * torch.arange(1, H + 1) / H).cuda()
    if "table" in mode:
        kw["rel_bias"] = rnd((H, 41), 1).cuda()
    return kw


# queries, keys, heads, Dh: few rows, many rows with their keys in parts, many rows whole; every width
ROWS = [(24, 640, 40, 64), (150, 640, 40, 64), (150, 640, 40, 128), (700, 640, 48, 64), (20, 640, 20, 256), (150, 640, 20, 256),
        (150, 640, 20, 80)]


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("mode", MODES)
def test_other_rows_change_no_bit(gpu, mode, dt):
    """Every other row of a wave has small scores, or large ones that grow from tile to tile, so that its
    base moves and a capped score takes its second form: the rows between keep their bits."""
    for Sq, Sk, H, Dh in ROWS:
        announce(f"scores of neighbours, {mode}, {Sq}x{Sk}x{H}x{Dh} {dt}")
        q, k, v = qkv(1, Sq, Sk, H, H, Dh, dt, 3)
        q, v = q.cuda(), v.cuda()
        k = (k.float() * torch.linspace(0.3, 2, Sk)[None, :, None, None]).to(dt).cuda()
        q[:, ::2] *= 0.5
        want = None
        for f in (0.0, 0.5, 8.0, math.inf, math.nan):
            x = q.clone()
            x[:, 1::2] *= f
            got = ops.attention_masked(x, k, v, **scores_kw(mode, H))[:, ::2]
            want = got if want is None else want
            assert torch.equal(got, want), f"{mode}, neighbours times {f}: {int((got != want).sum())} values differ"


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("mode", MODES)
def test_keys_that_only_other_rows_see_change_no_bit(gpu, mode, dt):
    for Sq, Sk, H, Dh in ROWS:
        announce(f"keys of neighbours, {mode}, {Sq}x{Sk}x{H}x{Dh} {dt}")
        q, k, v = (t.cuda() for t in qkv(1, Sq, Sk, H, H, Dh, dt, 4))
        r = torch.tensor([0, Sk], dtype=torch.int32, device="cuda").repeat(Sq, 1)
        r[::2, 1] = Sk - 200
        want = None
        for f in (1.0, 8.0, float("nan")):
            k2, v2 = k.clone(), v.clone()
            k2[:, Sk - 200:] *= f
            v2[:, Sk - 200:] *= f
            got = ops.attention_masked(q, k2, v2, key_range=r, **scores_kw(mode, H))[:, ::2]
            want = got if want is None else want
            assert torch.equal(got, want), f"{mode}, keys times {f}: {int((got != want).sum())} values differ"


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("mode", [m for m in MODES if "slopes" in m or "table" in m])
def test_places_of_other_rows_change_no_bit(gpu, mode, dt):
    for Sq, Sk, H, Dh in ROWS:
        announce(f"places of neighbours, {mode}, {Sq}x{Sk}x{H}x{Dh} {dt}")
        q, k, v = (t.cuda() for t in qkv(1, Sq, Sk, H, H, Dh, dt, 5))
        p = (torch.arange(Sq, dtype=torch.int32, device="cuda") * 7 + 11) % 331
        want = None
        for far in (0, 300, -(1 << 30), 1 << 30):
            at = p.clone()
            at[1::2] += far
            got = ops.attention_masked(q, k, v, q_pos=at, **scores_kw(mode, H))[:, ::2]
            want = got if want is None else want
            assert torch.equal(got, want), f"{mode}, neighbours {far} away: {int((got != want).sum())} values differ"


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("R", [20, 40, 400])  # R = 400: more than LDS holds of both heads
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_keys_that_a_table_hides_may_hold_anything(gpu, cap, R, dt):
    """Entries of -infinity among others, NaN and infinities in keys and values at their distance: rows that
    have them hidden keep their bits, and rows that see them show them where the definition does."""
    t = rnd((2, 2 * R + 1), 6)
    t[0, 1::4] = -math.inf
    t[1, R + 3:] = -math.inf  # no key three or more behind the query
    t[1, :R // 2] = -math.inf
    for Sq, Sk in ((1, 90), (5, 700), (150, 300), (200, 130)):
        q, k, v = qkv(1, Sq, Sk, 2, 2, 64, dt, 7)
        clean = ops.attention_masked(q.cuda(), k.cuda(), v.cuda(), cap=cap, rel_bias=t.cuda()).cpu()
        ref = M.attention(q, k, v, cap=cap, rel_bias=t)
        within(clean, ref["o"], att_tol(ref, Sk, dt, v), f"{Sq}x{Sk}, R = {R}, cap {cap}")
        at = [Sk - 1, Sk - 2, Sk // 2, 3]
        d = torch.tensor(at)[None] - torch.arange(Sk - Sq, Sk)[:, None]
        sees = (t[:, d.clamp(-R, R) + R] != -math.inf).any(-1).T  # [query, head]
        for x in (math.nan, math.inf, -math.inf):
            announce(f"hidden keys and values of {x}, {Sq}x{Sk}, R = {R}, cap {cap}, {dt}")
            k2, v2, v3 = k.clone(), v.clone(), v.clone()
            k2[:, at] = v2[:, at] = x
            v3[:, at, :, 1] = x
            both = ops.attention_masked(q.cuda(), k2.cuda(), v2.cuda(), cap=cap, rel_bias=t.cuda()).cpu()
            assert torch.equal(both[0][~sees], clean[0][~sees]), f"{int((both != clean)[0][~sees].sum())} values differ"
            one = ops.attention_masked(q.cuda(), k.cuda(), v3.cuda(), cap=cap, rel_bias=t.cuda()).cpu()
            assert torch.equal(one[0][~sees], clean[0][~sees])
            shown = one[0][sees][..., 1]
            assert (shown.isnan() if x != x else shown == x).all()
            rest = [e for e in range(64) if e != 1]
            assert torch.equal(one[..., rest], clean[..., rest])


@pytest.mark.parametrize("power", [126, 100, 0, -64])
@pytest.mark.parametrize("scores", ["equal", "growing", "falling"])
def test_bf16_values_of_any_size(gpu, scores, power):
    """Finite values have finite results up to the type's largest, whatever the weights' sum: 500 keys in
    one part, thousands in several, few rows and many."""
    for Sq, Sk, H in ((1, 500, 1), (2, 6000, 1), (100, 700, 1), (100, 5000, 1), (100, 500, 260)):
        announce(f"values of 2^{power}, {scores} scores, {Sq}x{Sk}x{H}")
        q, k, v = qkv(1, Sq, Sk, H, H, 64, torch.bfloat16, 8)
        k = k.float() * {"equal": torch.zeros(Sk), "growing": torch.linspace(0.2, 3, Sk),
                         "falling": torch.linspace(3, 0.2, Sk)}[scores][None, :, None, None]
        k = k.bfloat16()
        v = v.abs().clamp(0.5, 1.9) if scores == "equal" else v.clamp(-1.9, 1.9)
        ref = M.attention(q, k, v)
        big = (v.double() * 2.0 ** power).bfloat16()
        assert torch.isfinite(big).all() and torch.equal(big.double() * 2.0 ** -power, v.double())
        got = ops.attention_masked(q.cuda(), k.cuda(), big.cuda()).double() * 2.0 ** -power
        within(got, ref["o"], att_tol(ref, Sk, torch.bfloat16, v), f"values of 2^{power}")


@pytest.mark.parametrize("slope", [3e38, math.inf, -math.inf, 1e-45])
@pytest.mark.parametrize("mode", ["slopes", "cap and slopes"])
def test_slopes_of_any_size(gpu, slope, mode):
    """A slope past every score leaves a query the nearest of its keys alone (the farthest where it is
    negative); the smallest ones leave the plain result."""
    for Sq, Sk in ((1, 130), (150, 200)):
        announce(f"{mode} of {slope}, {Sq}x{Sk}")
        q, k, v = qkv(1, Sq, Sk, 1, 1, 64, torch.bfloat16, 9)
        p = torch.arange(Sq, dtype=torch.int32) + Sk - Sq
        kw = {"cap": 30.0} if "cap" in mode else {}
        dev = dict(slopes=torch.tensor([slope], device="cuda"), q_pos=p.cuda(), causal=True, **kw)
        got = ops.attention_masked(q.cuda(), k.cuda(), v.cuda(), **dev).cpu()
        if abs(slope) < 1:
            ref = M.attention(q, k, v, causal=True, **kw)
            within(got, ref["o"], att_tol(ref, Sk, torch.bfloat16, v), "a tiny slope")
            continue
        if slope > 0:
            assert torch.equal(got[0, :, 0], v[0, p.long(), 0])
        else:
            assert torch.equal(got[0, :, 0], v[0, :1, 0].expand(Sq, 64))


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
def test_an_output_among_its_operands(gpu, dt):
    """Queries, keys, values and the output as slices of one tensor: whole heads, or heads' parts."""
    B, S, H, Hkv, Dh = 2, 100, 4, 2, 64
    for shape, cut in (((B, S, 2 * H + 2 * Hkv, Dh), lambda t: t.split([H, Hkv, Hkv, H], 2)),
                       ((B, 2 * H + 2 * Hkv, S, Dh), lambda t: [x.transpose(1, 2) for x in t.split([H, Hkv, Hkv, H], 1)]),
                       ((B, S, H, 4 * Dh), lambda t: t.split(Dh, 3))):
        announce(f"slices of {shape} {dt}")
        x = rnd(shape, 10, dt).cuda()
        q, k, v, out = cut(x)
        want = ops.attention_masked(q, k, v, causal=True)
        before = [t.clone() for t in (q, k, v)]
        got = ops.attention_masked(q, k, v, causal=True, out=out)
        assert got is out and torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip((q, k, v), before))


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("eps", [1e-50, 1e-45, 1e-40, 1e-37])
def test_heads_of_zeros_under_the_smallest_eps(gpu, eps, dt):
    """0 / sqrt(0 + eps) is 0 for every eps but 0."""
    announce(f"norm of zeros, eps = {eps}, {dt}")
    x = rnd((1, 4, 2, 80), 11, dt)
    x[0, 1] = 0
    x[0, 3, 0] = 0
    got, _ = ops.qk_norm_rotary(x.cuda(), eps=eps)
    y = M.norm(x, None, eps)
    within(got, y, turn_tol(y, y.abs(), dt) + 2.0 ** -126, "norm")


def test_caps_below_every_number_are_refused(gpu):
    announce("a cap that is no fp32 number")
    q, k, v = (t.cuda() for t in qkv(1, 3, 9, 2, 2, 64, torch.float16))
    with pytest.raises(ValueError, match="cap"):
        ops.attention_masked(q, k, v, cap=1e-46)
    with pytest.raises(_lib.DlmError, match="cap"):
        ops.attention_masked(q, k, v, cap=1e-45)
    ops.attention_masked(q, k, v, cap=1e-45, scale=1e-30)


def in_parts(B, Sq, Sk, H, Hkv, Dh):
    """Whether a call of these sizes splits its keys."""
    a = _lib.AttentionMaskedArgs()
    a.B, a.Sq, a.Sk, a.H, a.Hkv, a.Dh = B, Sq, Sk, H, Hkv, Dh
    return _lib.hip_lib().dlm_attention_masked_workspace_bytes(ctypes.byref(a)) > 0


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("B,H,Hkv,Dh,lengths", [
    (1, 43, 43, 64, [310, 300, 90]), (2, 24, 24, 80, [257, 330, 3, 111]), (1, 48, 12, 64, [40, 360, 300]),
    (1, 37, 37, 40, [500, 260, 10]), (2, 37, 37, 64, [333, 1, 366]), (1, 30, 30, 128, [600, 520, 20]), (1, 29, 29, 256, [400, 390, 360]),
])
def test_documents_that_share_row_blocks_of_whole_keys(gpu, B, H, Hkv, Dh, lengths, dt):
    """More row blocks than CUs, so that keys stay whole: two workgroups store the rows of a block that holds
    the end of one long document and the start of another, started in the order of their lengths."""
    S = sum(lengths)
    blocks = B * Hkv * ((S * (H // Hkv) + 127) // 128)
    assert blocks > 255 and not in_parts(B, S, S, H, Hkv, Dh)
    q, k, v = qkv(B, S, S, H, Hkv, Dh, dt, S)
    r = ops.document_ranges(lengths, device="cpu")
    name = f"documents {lengths} x{B}x{H}/{Hkv}x{Dh} {dt}, {blocks} row blocks"
    out = torch.full((B, S, H, Dh), float("nan"), dtype=dt, device="cuda")
    attend(q, k, v, name, key_range=r, out=out)
    if Dh != 128:
        out.fill_(float("nan"))
        attend(q, k, v, f"{name}, causal", key_range=r, causal=True, out=out)


@pytest.mark.parametrize("B,S,H,Hkv,Dh", [(3, 260, 40, 40, 64), (1, 700, 47, 47, 64), (4, 130, 70, 70, 64), (1, 400, 84, 28, 80),
                                          (2, 513, 30, 30, 128), (5, 129, 29, 29, 40), (1, 1100, 31, 31, 64)])
def test_row_blocks_by_length_where_keys_are_whole(gpu, B, S, H, Hkv, Dh):
    """Causal row blocks beyond a first round on 256 CUs, in numbers that 8 divides and does not: each is
    taken once."""
    blocks = B * Hkv * ((S * (H // Hkv) + 127) // 128)
    assert 256 < blocks <= 8 * 256 and not in_parts(B, S, S, H, Hkv, Dh)
    q, k, v = qkv(B, S, S, H, Hkv, Dh, torch.float16, S)
    out = torch.full((B, S, H, Dh), float("nan"), dtype=torch.float16, device="cuda")
    attend(q, k, v, f"causal {B}x{S}x{H}/{Hkv}x{Dh}, {blocks} row blocks", causal=True, out=out)


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("mode", MODES)
def test_intervals_of_other_rows_change_no_bit(gpu, mode, dt):
    """Tiles that are whole for a row, and not for its neighbours."""
    for Sq, Sk, H, Dh in ROWS:
        announce(f"intervals of neighbours, {mode}, {Sq}x{Sk}x{H}x{Dh} {dt}")
        q, k, v = (t.cuda() for t in qkv(1, Sq, Sk, H, H, Dh, dt, 12))
        r = torch.tensor([0, Sk], dtype=torch.int32, device="cuda").repeat(Sq, 1)
        want = None
        for lo, hi in ((0, Sk), (0, Sk - 70), (100, Sk), (7, 7), (300, 330)):
            r[1::2, 0], r[1::2, 1] = lo, hi
            got = ops.attention_masked(q, k, v, key_range=r, **scores_kw(mode, H))[:, ::2]
            want = got if want is None else want
            assert torch.equal(got, want), f"{mode}, neighbours see [{lo}, {hi}): {int((got != want).sum())} values differ"


@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_a_table_shows_its_nan(gpu, cap):
    """An entry of NaN makes NaN of the rows that see a key at its distance, and of no other."""
    R = 20
    t = rnd((1, 2 * R + 1), 13)
    t[0, R - 7] = math.nan
    for Sq, Sk in ((2, 90), (150, 200)):
        announce(f"NaN in a table, {Sq}x{Sk}, cap {cap}")
        q, k, v = qkv(1, Sq, Sk, 1, 1, 64, torch.float16, 14)
        p = (torch.arange(Sq) * 9 % Sk).to(torch.int32)
        clean = p < 7  # no key seven behind them
        got = ops.attention_masked(q.cuda(), k.cuda(), v.cuda(), rel_bias=t.cuda(), cap=cap, q_pos=p.cuda()).cpu()
        assert got[0, ~clean].isnan().all()
        ref = M.attention(q[:, clean], k, v, rel_bias=t.nan_to_num(), cap=cap, q_pos=p[clean])
        within(got[:, clean], ref["o"], att_tol(ref, Sk, torch.float16, v), "the others")


@pytest.mark.parametrize("power,dt", [(n, dt) for dt in HALF for n in (20, 27, 33, 36, 70, 110)
                                      if n <= 36 or dt == torch.bfloat16], ids=str)
@pytest.mark.parametrize("mode", ["plain", "slopes", "table"])
def test_scores_far_beyond_their_differences(gpu, mode, power, dt):
    """Scores of 1.875 2^20 to 2^110, which no sum rounds, times log2 e, which every product rounds: equal
    ones share their weight, and the largest have it alone."""
    a = (power - 6) // 2
    b = power - 6 - a
    kw = {"slopes": torch.zeros(2)} if mode == "slopes" else {"rel_bias": torch.zeros(2, 41)} if mode == "table" else {}
    kw = {n: t.cuda() for n, t in kw.items()}
    for Sq, Sk in ((3, 100), (2, 3000), (150, 300), (150, 2000)):
        announce(f"scores of 2^{power}, {mode}, {Sq}x{Sk} {dt}")
        q, k, v = qkv(1, Sq, Sk, 2, 2, 64, dt, 16)
        q.fill_(1.25 * 2.0 ** a)
        k.fill_(1.5 * 2.0 ** b)
        keep = torch.zeros(Sk, dtype=torch.bool)
        keep[[Sk // 3, Sk // 2, Sk - 2]] = True
        half = torch.where(keep, 1.0, 0.5)[None, :, None, None]
        for what, f, seen in (("equal", 1.0, keep | True), ("equal, below 0", -1.0, keep | True), ("three", half, keep),
                              ("three, below 0", half - 1.5, keep)):
            got = ops.attention_masked(q.cuda(), (k.float() * f).to(dt).cuda(), v.cuda(), scale=1.0, **kw)
            want = v[:, seen].double().mean(1, keepdim=True).expand(1, Sq, 2, 64)
            ref = {"o": want, "A": v[:, seen].double().abs().mean(1, keepdim=True), "err": torch.zeros(1)}
            within(got, want, att_tol(ref, Sk, dt, v), f"{what} {Sq}x{Sk}")


@pytest.mark.parametrize("cap", [3e38, 1e38, 2.0 ** 125])
def test_scores_beyond_half_of_the_largest_caps(gpu, cap):
    for Sq, Sk in ((1, 100), (140, 100)):
        announce(f"scores of 1.9e38 under a cap of {cap}, {Sq}x{Sk}")
        q, k, v = qkv(1, Sq, Sk, 1, 1, 64, torch.bfloat16, 15)
        q.zero_(), k.zero_()
        q[..., 0] = 1.5 * 2.0 ** 63
        k[..., 0] = -1.5 * 2.0 ** 62
        k[0, 10, 0, 0], k[0, 70, 0, 0] = 1.5 * 2.0 ** 62, 1.5 * 2.0 ** 63
        got = ops.attention_masked(q.cuda(), k.cuda(), v.cuda(), scale=1.0, cap=cap).cpu()
        assert torch.equal(got, v[:, 70:71].expand(1, Sq, 1, 64)), "the largest score's value alone"


@pytest.mark.parametrize("mode", ["plain", "table"])
@pytest.mark.parametrize("dt,high,first,rise", [(torch.float16, 12, 32, 18), (torch.bfloat16, 13, 64, 20)], ids=["fp16", "bf16"])
def test_bases_that_round(gpu, dt, high, first, rise, mode):
    """One key above 60000 others by a few powers of two, all scores near 2^24 or 2^25, where every number is a
    multiple of 2 or 4: what was summed against the first base counts against the second as its score says."""
    scale = float(torch.tensor(math.log(2)))  # to powers of two: 1
    Sk, at = 60000, 50000
    for Sq in (1, 70):
        for B in (1, 260):  # with the keys in parts, and whole
            if B > 1 and (Sq == 1) != (mode == "plain"):
                continue
            announce(f"scores of {first} to {first + rise} above 2^{12 + high}, {mode}, {B}x{Sq} {dt}")
            q = torch.zeros(1, Sq, 1, 16, dtype=dt)
            k = torch.zeros(1, Sk, 1, 16, dtype=dt)
            q[..., 0], q[..., 1] = 2.0 ** high, 1.0
            k[..., 0], k[..., 1] = 2.0 ** 12, first
            k[0, at, 0, 1] = first + rise
            v = torch.ones(1, Sk, 1, 16, dtype=dt)
            v[0, at] = 0
            kw = {"rel_bias": torch.zeros(B, 1).cuda()} if mode == "table" else {}
            # the batches as heads, so that one tensor does for all
            got = ops.attention_masked(q.expand(1, Sq, B, 16).contiguous().cuda(), k.cuda().expand(1, Sk, B, 16),
                                       v.cuda().expand(1, Sk, B, 16), scale=scale, **kw).double().cpu()
            w = (Sk - 1) * 2.0 ** -rise
            want = torch.full((1, Sq, B, 16), w / (1 + w), dtype=torch.float64)
            ref = {"o": want, "A": want, "err": torch.zeros(1)}
            within(got, want, att_tol(ref, Sk, dt, v), f"{B}x{Sq}")


@pytest.mark.parametrize("dt", HALF, ids=NAMES.get)
@pytest.mark.parametrize("Dh", [64, 256])
def test_places_near_and_far_in_one_workgroup(gpu, Dh, dt):
    """Waves whose rows' places lie within a table's margin beside waves whose places do not: each takes its
    own way through the tiles, and all meet at every tile."""
    table = rnd((3, 2 * 40 + 1), 17)
    for Sq, Sk, H in ((128, 700, 3), (300, 512, 3), (130, 900, 90)):
        q, k, v = qkv(1, Sq, Sk, H, H, Dh, dt, 18)
        g = torch.Generator().manual_seed(Sq)
        p = torch.arange(Sq, dtype=torch.int32) + 100
        for at in (0, 64, 160):
            n = len(p[at:at + 32])
            p[at:at + 32] = torch.randint(0, Sk, (n,), generator=g).to(torch.int32)
        t = table.repeat(H // 3, 1)
        attend(q, k, v, f"places near and far, {Sq}x{Sk}x{H}x{Dh} {dt}", q_pos=p, rel_bias=t)
        r = torch.tensor([17, Sk - 5], dtype=torch.int32).repeat(Sq, 1)
        attend(q, k, v, f"places near and far, interval, {Sq}x{Sk}x{H}x{Dh} {dt}", q_pos=p, rel_bias=t, key_range=r)
