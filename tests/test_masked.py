"""Argument checks of the rotary, norm and masked-attention entry points, at the C
boundary and without a device: every refused call returns before anything is launched;
the mask helpers, and the oracle's float64 definitions against closed forms (CPU only)."""
import ctypes
import math
import os
import struct

import pytest
import torch

from dollama_amd import _lib, ops
from oracle import masked_ref as M

A = 1 << 24  # addresses that no refused call reads
INVALID = _lib.DLM_ERR_INVALID_ARG


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.HIP_LIB_PATH):
        pytest.fail("libdlm_hip.so is not built")
    return _lib.hip_lib()


def err():
    return _lib.last_error()


def test_packed_arguments_have_the_structures_layout():
    for fmt, cls in ((_lib.ROTARY_FORMAT, _lib.RotaryArgs), (_lib.ATTENTION_MASKED_FORMAT, _lib.AttentionMaskedArgs)):
        s = struct.Struct(fmt)
        assert s.size == ctypes.sizeof(cls)
        n = len(s.unpack(bytes(s.size)))
        values = list(range(1, n + 1))
        a = cls.from_buffer_copy(s.pack(*values))
        got = []
        for name, _ in cls._fields_:
            x = getattr(a, name)
            got += list(x) if isinstance(x, ctypes.Array) else [x]
        assert [int(x) for x in got] == values


def rotary_args(**kw):
    a = _lib.RotaryArgs()
    B, S, H, Hkv, Dh = 2, 8, 4, 2, 64
    a.q, a.k, a.q_out, a.k_out = A, 2 * A, 3 * A, 4 * A
    for x, h in (("q", H), ("qo", H), ("k", Hkv), ("ko", Hkv)):
        setattr(a, x + "_sb", S * h * Dh)
        setattr(a, x + "_ss", h * Dh)
        setattr(a, x + "_sh", Dh)
    a.pos, a.pos_sb, a.pos_ss, a.freqs, a.pos_type, a.axes = 5 * A, S * 2, 2, 6 * A, 0, 2
    a.sections[0], a.sections[1] = 16, 16
    a.norm, a.eps, a.dtype = 1, 1e-6, 0
    a.B, a.S, a.H, a.Hkv, a.Dh = B, S, H, Hkv, Dh
    for n, v in kw.items():
        if n == "sections":
            for i, x in enumerate(v):
                a.sections[i] = x
        else:
            setattr(a, n, v)
    return a


def test_rotary_entries_refuse(lib):
    def qk(**kw):
        return lib.dlm_qk_norm_rotary(ctypes.byref(rotary_args(**kw)), None)

    assert lib.dlm_qk_norm_rotary(None, None) == INVALID and "NULL" in err()
    assert lib.dlm_rotary_axes(None, None) == INVALID
    for dim in ("B", "S", "H", "Dh"):  # nothing to do
        assert qk(**{dim: 0}, q=None) == 0
    for text, kw in [
        ("NULL", dict(q=None)), ("NULL", dict(q_out=None)), ("together", dict(k=None)), ("together", dict(k_out=None)),
        ("heads", dict(Hkv=0)), ("dtype", dict(dtype=2)), ("Dh", dict(Dh=65)), ("Dh", dict(Dh=258)), ("axes", dict(axes=5)),
        ("axes", dict(axes=-1)), ("negative", dict(sections=[-1, 4])), ("more pairs", dict(sections=[17, 16])),
        ("more pairs", dict(sections=[2 ** 31 - 1, 2 ** 31 - 1])), ("positions", dict(pos=None)), ("positions", dict(freqs=None)),
        ("type of positions", dict(pos_type=3)), ("aligned", dict(pos=5 * A + 2)), ("aligned", dict(freqs=6 * A + 4)),
        ("aligned", dict(pos=5 * A + 4, pos_type=1)), ("stride", dict(pos_ss=-1)), ("eps", dict(eps=-1.0)),
        ("eps", dict(eps=float("nan"))), ("eps", dict(eps=float("inf"))), ("aligned", dict(q=A + 1)),
        ("aligned", dict(k_out=4 * A + 1)), ("aligned", dict(q_gamma=7 * A + 1)), ("negative stride", dict(q_ss=-64)),
        ("2^46", dict(q_sb=1 << 60)), ("2^26", dict(B=1 << 13, S=1 << 13)), ("65535", dict(H=65536)),
        ("q_out overlaps itself", dict(qo_sh=32)), ("k_out overlaps itself", dict(ko_ss=0)),
        # outputs on inputs, and on one another
        ("q_out overlaps q", dict(q_out=A + 2)), ("q_out overlaps k", dict(q_out=2 * A)), ("k_out overlaps q", dict(k_out=A)),
        ("k_out overlaps q_out", dict(k_out=3 * A)), ("k_out overlaps k", dict(k_out=2 * A + 128)),
        ("q_out overlaps q", dict(q_out=A, qo_ss=512, qo_sb=8 * 512)),  # in place, but for the strides
    ]:
        assert qk(**kw) == INVALID and text in err(), (kw, err())
    assert lib.dlm_rotary_axes(ctypes.byref(rotary_args()), None) == INVALID and "norm" in err()
    assert lib.dlm_rotary_axes(ctypes.byref(rotary_args(norm=0, q_gamma=7 * A)), None) == INVALID and "gamma" in err()
    assert qk(norm=0) == INVALID and "rotation" in err()


def test_slices_of_one_tensor_do_not_overlap(lib):
    """The overlap check against the sets of addresses: k and q_out lie among one another
    by chance; k_out is q_out, so that every call is refused in the end."""
    import itertools
    import random
    rng = random.Random(3)
    told = {True: 0, False: 0}
    for _ in range(600):
        B, S, Dh = rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([2, 4, 8])
        Hkv = rng.choice([1, 2])
        H = Hkv + rng.choice([0, 1])
        size, st = Dh + rng.choice([0, 4]), {}
        for d in reversed(rng.choice(["bsh", "bhs", "sbh"])):
            st[d] = size
            size *= {"b": B, "s": S, "h": 8}[d]
        k, q_out = (rng.randrange(0, 8) * st["h"] + rng.randrange(0, S) * st["s"] + rng.choice([0, 0, 0, Dh // 2])
                    for _ in range(2))

        def cells(at, heads):
            return {at + b * st["b"] + s * st["s"] + h * st["h"] + d
                    for b, s, h, d in itertools.product(range(B), range(S), range(heads), range(Dh))}

        kw = dict(q=A - 1024 * 1024, k=A + 2 * k, q_out=A + 2 * q_out, k_out=A + 2 * q_out, B=B, S=S, H=H, Hkv=Hkv, Dh=Dh,
                  sections=[0, 0])
        for x in ("q", "qo", "k", "ko"):
            kw[x + "_sb"], kw[x + "_ss"], kw[x + "_sh"] = st["b"], st["s"], st["h"]
        clash = bool(cells(k, Hkv) & cells(q_out, H))
        told[clash] += 1
        assert lib.dlm_qk_norm_rotary(ctypes.byref(rotary_args(**kw)), None) == INVALID
        assert ("q_out overlaps k" if clash else "k_out overlaps q_out") in err(), (kw, err())
    assert min(told.values()) > 100


def attention_args(**kw):
    a = _lib.AttentionMaskedArgs()
    B, Sq, Sk, H, Hkv, Dh = 2, 8, 16, 4, 2, 64
    a.q, a.k, a.v, a.o = A, 2 * A, 3 * A, 4 * A
    for x, s, h in (("q", Sq, H), ("o", Sq, H), ("k", Sk, Hkv), ("v", Sk, Hkv)):
        setattr(a, x + "_sb", s * h * Dh)
        setattr(a, x + "_ss", h * Dh)
        setattr(a, x + "_sh", Dh)
    a.scale, a.B, a.Sq, a.Sk, a.H, a.Hkv, a.Dh = 0.125, B, Sq, Sk, H, Hkv, Dh
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_attention_entry_refuses(lib):
    def go(ws=None, n=0, **kw):
        return lib.dlm_attention_masked(ctypes.byref(attention_args(**kw)), ws, n, None)

    assert lib.dlm_attention_masked(None, None, 0, None) == INVALID and "NULL" in err()
    assert lib.dlm_attention_masked_workspace_bytes(None) == 0
    for dim in ("B", "Sq", "H", "Dh"):
        assert go(**{dim: 0}, q=None) == 0
    for text, kw in [
        ("NULL", dict(q=None)), ("NULL", dict(k=None)), ("NULL", dict(v=None)), ("NULL", dict(o=None)), ("dtype", dict(dtype=2)),
        ("number of keys", dict(Sk=-1)), ("Dh", dict(Dh=60)), ("Dh", dict(Dh=264)), ("multiple of Hkv", dict(Hkv=3)),
        ("multiple of Hkv", dict(Hkv=0)), ("scale", dict(scale=0.0)), ("scale", dict(scale=float("inf"))),
        ("scale", dict(scale=float("nan"))), ("cap", dict(cap=-1.0)), ("cap", dict(cap=float("nan"))), ("cap is too small", dict(cap=1e-38, scale=1.0)),
        ("one bias", dict(slopes=5 * A, rel_bias=6 * A)), ("R must", dict(rel_bias=6 * A, R=-1)),
        ("R must", dict(rel_bias=6 * A, R=(1 << 24) + 1)), ("2^28", dict(Sk=(1 << 28) + 1)), ("rows", dict(Sq=1 << 28)),
        ("rows", dict(B=70000)), ("rows", dict(B=30000, Sq=100000)), ("q: address", dict(q=A + 8)),
        ("k: address", dict(k_ss=132)), ("v: address", dict(v_sh=68)), ("o: address", dict(o=4 * A + 4)),
        ("o: address", dict(o_ss=258)), ("negative", dict(q_sb=-64)), ("stride must", dict(k_ss=56)),
        ("stride must", dict(v_ss=0)), ("stride must", dict(k_ss=1 << 23)), ("2^46", dict(o_sb=1 << 50)),
        ("o overlaps itself", dict(o_sh=32)), ("o overlaps itself", dict(o_sb=0)), ("o overlaps q", dict(o=A)),
        ("o overlaps k", dict(o=2 * A + 128)), ("o overlaps v", dict(o=3 * A - 8)), ("aligned", dict(key_range=7 * A + 4)),
        ("aligned", dict(q_pos=7 * A + 2)), ("aligned", dict(slopes=7 * A + 2)), ("batch strides", dict(key_range=7 * A, kr_sb=3)),
        ("batch strides", dict(q_pos=7 * A, qp_sb=-1)),
    ]:
        assert go(**kw) == INVALID and text in err(), (kw, err())
    # few queries against many keys: the parts need room
    kw = dict(Sq=1, Sk=4096, k_sb=4096 * 128, v_sb=4096 * 128, v=8 * A)
    n = lib.dlm_attention_masked_workspace_bytes(ctypes.byref(attention_args(**kw)))
    assert n > 0 and n % (2 * 4 * 66 * 4) == 0  # parts of B x H rows of Dh + 2 floats
    assert go(None, n, **kw) == INVALID and "workspace" in err()
    assert go(A * 16, n - 1, **kw) == INVALID and "workspace" in err()
    assert go(A * 16 + 8, n, **kw) == INVALID and "16-byte" in err()
    assert lib.dlm_attention_masked_workspace_bytes(ctypes.byref(attention_args())) == 0


@pytest.mark.parametrize("B,Sq,Sk,H,Hkv,Dh,parts", [
    (1, 8192, 8192, 10, 10, 64, False),  # 640 workgroups without parts
    (2, 4096, 4096, 10, 10, 64, False), (1, 4096, 4096, 32, 8, 128, False), (4, 512, 512, 64, 64, 64, False),
    (2, 2051, 2051, 12, 12, 80, False), (1 << 10, 1, 4096, 32, 8, 128, False), (1, 1, 511, 32, 8, 128, False),
    (1, 1, 4096, 32, 8, 128, True), (1, 64, 30001, 32, 32, 128, True), (40, 1, 32768, 32, 8, 128, True),
])
def test_keys_are_split_where_workgroups_are_few(lib, B, Sq, Sk, H, Hkv, Dh, parts):
    a = attention_args(B=B, Sq=Sq, Sk=Sk, H=H, Hkv=Hkv, Dh=Dh)
    assert (lib.dlm_attention_masked_workspace_bytes(ctypes.byref(a)) > 0) == parts


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu():
    q = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    for call in (lambda: ops.attention_masked(q, q, q), lambda: ops.qk_norm_rotary(q),
                 lambda: ops.rotary_axes(q, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(32), [32])):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_mask_helpers():
    r = ops.document_ranges([2, 0, 3], tokens=7, device="cpu")
    assert r.tolist() == [[0, 2], [0, 2], [2, 5], [2, 5], [2, 5], [0, 0], [0, 0]]
    assert ops.document_ranges([], device="cpu").shape == (0, 2)
    assert ops.document_ranges([], 3, device="cpu").tolist() == [[0, 0]] * 3
    with pytest.raises(ValueError):
        ops.document_ranges([3, 3], tokens=5, device="cpu")
    with pytest.raises(ValueError):
        ops.document_ranges([3, -1], device="cpu")
    p = ops.prefix_ranges([0, 2, 9], 4, device="cpu")
    assert p[..., 0].abs().sum() == 0
    assert p[..., 1].tolist() == [[1, 2, 3, 4], [2, 2, 3, 4], [4, 4, 4, 4]]
    assert ops.prefix_ranges([3], 2, 6, device="cpu")[..., 1].tolist() == [[5, 6]]
    f = ops.rotary_freqs([2, 3], theta=16.0, device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1, 0.25, 1, 16 ** (-1 / 3), 16 ** (-2 / 3)], dtype=torch.float64))
    f = ops.rotary_freqs([2, 2], theta=16.0, shared=True, device="cpu")
    assert torch.allclose(f, torch.tensor([1, 0.5, 0.25, 0.125], dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.rotary_freqs([2, -2], device="cpu")


def test_oracle_closed_forms():
    # a quarter turn, halves and interleaved
    x = torch.tensor([1.0, 2.0, 3.0, 4.0, 9.0]).view(1, 1, 1, 5)[..., :4]
    f = torch.tensor([math.pi / 2, 0.0], dtype=torch.float64)
    pos = torch.ones(1, 1, 1)
    assert torch.allclose(M.rotary(x, pos, f, [2], False)[0].flatten(), torch.tensor([-3.0, 2, 1, 4], dtype=torch.float64))
    assert torch.allclose(M.rotary(x, pos, f, [2], True)[0].flatten(), torch.tensor([-2.0, 1, 3, 4], dtype=torch.float64))
    # only differences of positions matter to a product
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(2, 1, 6, 1, 8, generator=g).double().unbind(0)
    f = ops.rotary_freqs([1, 3], device="cpu")
    p = torch.randint(0, 50, (1, 6, 2), generator=g)
    dots = [(M.rotary(q, p + s, f, [1, 3], False)[0][0, :, 0] @ M.rotary(k, p + s, f, [1, 3], False)[0][0, :, 0].T)
            for s in (0, 17)]
    assert torch.allclose(*dots)
    assert torch.allclose(M.norm(torch.full((1, 4), 3.0), None, 0.0), torch.ones(1, 4, dtype=torch.float64))
    # equal scores: the mean over what is seen; nothing seen: 0
    q = torch.zeros(1, 3, 2, 8)
    v = torch.randn(1, 3, 1, 8, generator=g)
    o = M.attention(q, q[:, :, :1], v, causal=True)["o"]
    assert torch.allclose(o[0, 1, 0], v[0, :2, 0].double().mean(0)) and torch.allclose(o[0, 2, 1], v[0, :, 0].double().mean(0))
    o = M.attention(q, q[:, :, :1], v, key_range=torch.tensor([[0, 3], [1, 1], [2, 9]]))["o"]
    assert (o[0, 1] == 0).all() and torch.allclose(o[0, 2, 0], v[0, 2, 0].double())
    # a slope of ln 2 halves a weight each step away
    o = M.attention(q, q[:, :, :1], v, slopes=torch.full((2,), math.log(2)))["o"]
    w = torch.tensor([0.25, 0.5, 1.0], dtype=torch.float64)
    assert torch.allclose(o[0, 2, 0], (w / w.sum()) @ v[0, :, 0].double())
