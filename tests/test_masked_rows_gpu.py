"""Masked attention's rows beside one another: no row's result shows what another row's query, keys or
place hold (GPU)."""
import pytest
import torch

from dollama_amd import ops
from test_masked_gpu import HALF, NAMES, announce, qkv, rnd

pytestmark = pytest.mark.gpu

MODES = ["plain", "cap", "slopes", "table", "cap and slopes", "cap and table"]


def scores_kw(mode, H):
    kw = {"cap": 30.0} if "cap" in mode else {}
    if "slopes" in mode:
        kw["slopes"] = torch.exp2(-8 * torch.arange(1, H + 1) / H).cuda()
    if "table" in mode:
        kw["rel_bias"] = rnd((H, 41), 1).cuda()
    return kw


# queries, keys, heads, Dh: few rows, many rows with their keys in parts, many rows whole
ROWS = [(24, 640, 40, 64), (150, 640, 40, 64), (150, 640, 40, 128), (700, 640, 48, 64)]


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
        for f in (0.0, 0.5, 8.0):
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
