"""More argument checks of the rotary, norm and masked-attention entry points at the C boundary, without a
device: every refused call returns before anything is launched (CPU only)."""
import ctypes
import struct

import msgpack

from dollama_amd import _lib
from test_masked import A, INVALID, attention_args, err, lib, rotary_args  # noqa: F401 (lib: a fixture)


def qk(lib, **kw):
    return lib.dlm_qk_norm_rotary(ctypes.byref(rotary_args(**kw)), None)


def test_tokens_that_a_grid_takes(lib):
    """64 lanes a token where heads are wide or unaligned, in whole blocks of four tokens: fewer than 2^32."""
    for tokens in ((1 << 26) - 3, (1 << 26) - 1, 1 << 26):
        assert qk(lib, B=1, S=tokens) == INVALID and "2^26 - 4 tokens" in err(), (tokens, err())
    assert qk(lib, B=1, S=(1 << 26) - 4, H=65536) == INVALID and "65535" in err()


def test_rotary_outputs_on_what_every_head_reads(lib):
    """Gammas, positions and frequencies on an output are refused; in the gaps between its heads they are not
    (those calls are refused for their last operand: k_out is q_out)."""
    qo = 3 * A  # [2, 8, 4, 64], contiguous: 8192 bytes; k_out at 4 A: 4096
    last = 8192
    for text, kw in [
        ("q_out overlaps q_gamma", dict(q_gamma=qo)), ("q_out overlaps q_gamma", dict(q_gamma=qo - 126)),
        ("q_out overlaps q_gamma", dict(q_gamma=qo + last - 2)), ("q_out overlaps k_gamma", dict(k_gamma=qo + 1000)),
        ("k_out overlaps k_gamma", dict(k_gamma=4 * A + 4094)), ("k_out overlaps q_gamma", dict(q_gamma=4 * A - 2)),
        ("q_out overlaps pos", dict(pos=qo + last - 4)), ("q_out overlaps pos", dict(pos=qo - 124)),  # 16 x 2 int32
        ("q_out overlaps pos", dict(pos=qo - 248, pos_type=1, pos_sb=16)), ("k_out overlaps pos", dict(pos=4 * A)),
        ("q_out overlaps freqs", dict(freqs=qo + 8)), ("k_out overlaps freqs", dict(freqs=4 * A - 248)),
        ("k_out overlaps q_out", dict(q_gamma=qo - 128, k_gamma=qo + last, pos=qo - 256, freqs=qo + last, k_out=qo)),
        ("span more", dict(pos_sb=1 << 60)),
    ]:
        assert qk(lib, **kw) == INVALID and text in err(), (kw, err())


def test_bytes_on_a_view_against_its_addresses(lib):
    """q_gamma among the elements of q_out by chance, against the sets of addresses; every call is refused in
    the end, k_out being q_out."""
    import itertools
    import random
    rng = random.Random(5)
    told = {True: 0, False: 0}
    for _ in range(800):
        B, S, H, Dh = rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([1, 2, 3]), rng.choice([2, 4, 8])
        size, st = Dh + rng.choice([0, 4, 20]), {}
        for d in reversed(rng.choice(["bsh", "bhs", "sbh"])):
            st[d] = size
            size = size * {"b": B, "s": S, "h": H}[d] + rng.choice([0, 10, 30])
        at = rng.randrange(-Dh - 2, size + 4)
        cells = {b * st["b"] + s * st["s"] + h * st["h"] + d
                 for b, s, h, d in itertools.product(range(B), range(S), range(H), range(Dh))}
        kw = dict(q=A - 1024 * 1024, k=A + 1024 * 1024, q_out=A, k_out=A, q_gamma=A + 2 * at, B=B, S=S, H=H, Hkv=H, Dh=Dh,
                  sections=[0, 0])
        for x in ("q", "qo", "k", "ko"):
            kw[x + "_sb"], kw[x + "_ss"], kw[x + "_sh"] = st["b"], st["s"], st["h"]
        clash = bool(cells & set(range(at, at + Dh)))
        told[clash] += 1
        assert qk(lib, **kw) == INVALID
        assert ("q_out overlaps q_gamma" if clash else "k_out overlaps q_out") in err(), (kw, err())
    assert min(told.values()) > 100, told


def attend(lib, ws=None, n=0, **kw):
    return lib.dlm_attention_masked(ctypes.byref(attention_args(**kw)), ws, n, None)


def test_attention_outputs_on_masks_and_biases(lib):
    o, size = 4 * A, 2 * 8 * 4 * 64 * 2  # [2, 8, 4, 64], contiguous
    table = dict(R=3)  # [4, 7]
    for text, kw in [
        ("o overlaps key_range", dict(key_range=o)), ("o overlaps key_range", dict(key_range=o - 56)),
        ("o overlaps key_range", dict(key_range=o - 112, kr_sb=16)), ("o overlaps key_range", dict(key_range=o + size - 8)),
        ("o overlaps q_pos", dict(q_pos=o - 28)), ("o overlaps q_pos", dict(q_pos=o - 60, qp_sb=8)),
        ("o overlaps slopes", dict(slopes=o - 12)), ("o overlaps slopes", dict(slopes=o + size - 4)),
        ("o overlaps rel_bias", dict(rel_bias=o - 108, **table)), ("o overlaps rel_bias", dict(rel_bias=o + size - 4, **table)),
        # in the gaps between heads of 64 in 128 they are free (those calls are refused for their table)
        ("o overlaps rel_bias", dict(o_sh=128, o_ss=512, o_sb=4096, key_range=o + 128, rel_bias=o, **table)),
        ("o overlaps rel_bias", dict(o_sh=128, o_ss=512, o_sb=4096, q_pos=o + 128, rel_bias=o, **table)),
        ("span more", dict(q_pos=7 * A, qp_sb=1 << 50)),
    ]:
        assert attend(lib, **kw) == INVALID and text in err(), (kw, err())


def test_workspaces_on_operands(lib):
    many = dict(Sq=1, Sk=4096, k_sb=4096 * 128, v_sb=4096 * 128, v=8 * A, q_sb=256, o_sb=256)
    n = lib.dlm_attention_masked_workspace_bytes(ctypes.byref(attention_args(**many)))
    assert n > 0
    keys = 2 * 4096 * 128 * 2
    for text, ws, kw in [
        ("workspace overlaps q", A, {}), ("workspace overlaps q", A - n + 16, {}), ("workspace overlaps q", A + 1008, {}),
        ("workspace overlaps k", 2 * A + keys - 16, {}), ("workspace overlaps v", 8 * A - 16, {}), ("workspace overlaps o", 4 * A, {}),
        ("workspace overlaps key_range", 9 * A, dict(key_range=9 * A + n - 16)),
        ("workspace overlaps q_pos", 9 * A, dict(q_pos=9 * A)), ("workspace overlaps slopes", 9 * A, dict(slopes=9 * A - 12)),
        ("workspace overlaps rel_bias", 9 * A + 16 * 4, dict(rel_bias=9 * A, R=3)),
    ]:
        assert attend(lib, ws, n, **{**many, **kw}) == INVALID and text in err(), (ws, kw, err())


def test_attention_outputs_among_operands(lib):
    """The output may be a slice of the tensor that the operands are slices of; against the sets of addresses.
    Calls without an overlap are refused for their places' alignment."""
    import itertools
    import random
    rng = random.Random(9)
    told = {True: 0, False: 0}
    for _ in range(800):
        B, Sq, Sk, Dh = rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([1, 2, 4]), 8
        Hkv = rng.choice([1, 2])
        H = Hkv * rng.choice([1, 2])
        size, st = Dh + rng.choice([0, 8]), {}
        for d in reversed(rng.choice(["bsh", "bhs", "sbh"])):
            st[d] = size
            size *= {"b": B, "s": 6, "h": 8}[d]
        k, o = (rng.randrange(0, 6) * st["h"] + rng.randrange(0, 3) * st["s"] for _ in range(2))

        def cells(at, tokens, heads):
            return {at + b * st["b"] + s * st["s"] + h * st["h"] + d
                    for b, s, h, d in itertools.product(range(B), range(tokens), range(heads), range(Dh))}

        kw = dict(q=A - 1024 * 1024, v=A + 1024 * 1024, k=A + 2 * k, o=A + 2 * o, B=B, Sq=Sq, Sk=Sk, H=H, Hkv=Hkv, Dh=Dh,
                  q_pos=7 * A + 2)
        for x in "qkvo":
            kw[x + "_sb"], kw[x + "_ss"], kw[x + "_sh"] = st["b"], st["s"], st["h"]
        clash = bool(cells(k, Sk, Hkv) & cells(o, Sq, H))
        told[clash] += 1
        assert attend(lib, **kw) == INVALID
        assert ("o overlaps k" if clash else "aligned") in err(), (kw, err())
    assert min(told.values()) > 100, told


def test_scales_whose_powers_of_two_leave_fp32(lib):
    """scale log2 e has to be finite: infinity times a product of 0 is NaN."""
    for cap in (0.0, 1e38):
        assert attend(lib, scale=3e38, cap=cap) == INVALID and "scale" in err()
        assert attend(lib, scale=2.0 ** 127, cap=cap, q_pos=7 * A + 2) == INVALID and "aligned" in err()


def code_objects(path):
    """The gfx950 code objects that the library holds."""
    with open(path, "rb") as f:
        d = f.read()
    at = d.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        n, p = struct.unpack_from("<Q", d, at + 24)[0], at + 32
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", d, p)
            if b"gfx950" in d[p + 24:p + 24 + length]:
                yield d[at + offset:at + offset + size]
            p += 24 + length
        at = d.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 24)


def kernels(elf):
    """Their kernels' metadata: the note of type 32 of a note section."""
    sections, = struct.unpack_from("<Q", elf, 40)
    entry, count = struct.unpack_from("<HH", elf, 58)
    for i in range(count):
        if struct.unpack_from("<I", elf, sections + i * entry + 4)[0] != 7:
            continue
        p, size = struct.unpack_from("<QQ", elf, sections + i * entry + 24)
        end = p + size
        while p < end:
            name, desc, kind = struct.unpack_from("<III", elf, p)
            p += 12 + (name + 3) // 4 * 4
            if kind == 32:
                yield from msgpack.unpackb(elf[p:p + desc])["amdhsa.kernels"]
            p += (desc + 3) // 4 * 4


def test_no_kernel_spills_to_both_kinds_of_place(lib):
    """A tuple of registers that is spilled to AGPRs in part and to scratch memory in part has come back without
    one of the former: kernels with AGPRs use no scratch memory."""
    found = [k for e in code_objects(_lib.HIP_LIB_PATH) for k in kernels(e)]
    wide = [k for k in found if "attn_masked" in k[".name"] and "Li512E" in k[".name"]]
    assert len(wide) == 20  # two kernels, five kinds of score, two types
    both = [k[".name"] for k in found if k[".agpr_count"] and k[".private_segment_fixed_size"]]
    assert not both, both
