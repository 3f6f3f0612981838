"""Argument checks of the 8-bit entry points, at the C boundary and without a
device: every refused call returns before anything is launched, and the oracle's
float64 definitions agree with closed forms (CPU only)."""
import ctypes
import os

import pytest
import torch

from dollama_amd import _lib, ops
from oracle import quant_ref as Q

A = 1 << 24  # addresses that no refused call reads
INVALID = _lib.DLM_ERR_INVALID_ARG


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.HIP_LIB_PATH):
        pytest.fail("libdlm_hip.so is not built")
    return _lib.hip_lib()


def err():
    return _lib.last_error()


def test_row_entries_refuse(lib):
    for t, e in (("fp16", 2), ("f32", 4)):
        qz = getattr(lib, f"dlm_quantize_rows_{t}")
        assert qz(None, 64, None, 64, None, 0, 64, None) == 0  # no rows: nothing to do
        assert qz(None, 64, None, 64, None, 4, -1, None) == 0
        assert qz(None, 64, A, 64, A * 2, 4, 64, None) == INVALID and "NULL" in err()
        assert qz(A, 63, 2 * A, 64, 3 * A, 4, 64, None) == INVALID and "stride" in err()
        assert qz(A, 64, 2 * A, 63, 3 * A, 4, 64, None) == INVALID and "stride" in err()
        assert qz(A + 1, 64, 2 * A, 64, 3 * A, 4, 64, None) == INVALID and "aligned" in err()
        assert qz(A, 64, 2 * A, 64, 3 * A + 2, 4, 64, None) == INVALID and "aligned" in err()
        assert qz(A, 64, A + 4 * 64 * e - 1, 64, 3 * A, 4, 64, None) == INVALID and "q overlaps x" in err()
        assert qz(A, 64, 2 * A, 64, A, 4, 64, None) == INVALID and "scale overlaps x" in err()
        assert qz(A, 64, 2 * A, 64, 2 * A + 8, 4, 64, None) == INVALID and "overlaps" in err()
        for name, beta in (("rms", ()), ("layer", (None,))):
            nm = getattr(lib, f"dlm_{name}_norm_q8_{t}")

            def call(x=A, ldx=64, R=2 * A, ldr=64, H=3 * A, ldh=64, gamma=None, eps=1e-5):
                return nm(x, ldx, R, ldr, H, ldh, gamma, *beta, 5 * A, 64, 6 * A, 4, 64, eps, None)

            assert call(ldr=63) == INVALID and "stride" in err()
            assert call(ldh=63) == INVALID and "stride" in err()
            assert call(R=None) == INVALID and "residual" in err()
            assert call(eps=-1.0) == INVALID and "eps" in err()
            assert call(eps=float("nan")) == INVALID and "eps" in err()
            assert call(gamma=4 * A + 1) == INVALID and "aligned" in err()
            assert call(H=2 * A + 64 * e) == INVALID and "sum overlaps residual" in err()
            assert call(H=A, ldh=128) == INVALID and "sum overlaps x" in err()  # another row stride
            assert call(H=5 * A) == INVALID and "overlaps q" in err()
        dq = getattr(lib, f"dlm_dequantize_rows_{t}")
        assert dq(A, 64, 2 * A, 3 * A, 63, 4, 64, None) == INVALID and "stride" in err()
        assert dq(A, 64, None, 3 * A, 64, 4, 64, None) == INVALID and "NULL" in err()
        assert dq(A, 64, 2 * A, A + 16, 64, 4, 64, None) == INVALID and "overlaps" in err()


def test_linear_entries_refuse(lib):
    for f in (lib.dlm_linear_q8_fp16, lib.dlm_linear_q8_f32out):
        def call(X=A, ldx=64, sx=2 * A, W=3 * A, ldw=64, sw=4 * A, bias=None, R=None, ldr=0, Y=6 * A, ldy=32, M=4, N=32,
                 K=64, act=0):
            return f(X, ldx, sx, W, ldw, sw, bias, R, ldr, Y, ldy, M, N, K, 1.0, act, None)

        assert call(X=None, M=0) == 0 and call(X=None, N=-1) == 0 and call(X=None, K=0) == 0
        for k in ("X", "W", "sx", "sw", "Y"):
            assert call(**{k: None}) == INVALID and "NULL" in err()
        assert call(act=4) == INVALID and "activation" in err()
        assert call(act=-1) == INVALID and "activation" in err()
        assert call(act=2, N=24) == INVALID and "GEGLU" in err()
        assert call(K=131072, ldx=131072, ldw=131072) == INVALID and "K" in err()
        assert call(ldx=(1 << 22) + 16) == INVALID and "4194304" in err()
        assert call(N=(1 << 25) + 1, ldy=(1 << 25) + 1) == INVALID and "33554432" in err()
        assert call(X=A + 8) == INVALID and "16-byte" in err()
        assert call(ldw=72) == INVALID and "16-byte" in err()
        assert call(K=65) == INVALID and "rounded up" in err()
        assert call(ldy=31) == INVALID and "stride" in err()
        assert call(R=7 * A, ldr=31) == INVALID and "stride" in err()
        assert call(Y=6 * A + 1) == INVALID and "aligned" in err()
        assert call(bias=7 * A + 1) == INVALID and "aligned" in err()
        assert call(sx=2 * A + 2) == INVALID and "aligned" in err()
        for k in ("X", "W", "sx", "sw", "bias"):
            assert call(**{k: 6 * A}) == INVALID and "Y overlaps " + k in err()
        assert call(R=6 * A, ldr=48) == INVALID and "Y overlaps R" in err()


def test_the_sum_may_be_neither_gamma_nor_beta(lib):
    for t in ("fp16", "f32"):
        for rows, K, ldh in ((4, 64, 64), (1, 64, 64), (4, 64, 128), (1, 128, 128)):
            rms, layer = getattr(lib, f"dlm_rms_norm_q8_{t}"), getattr(lib, f"dlm_layer_norm_q8_{t}")
            H, tail = 3 * A, (5 * A, K, 6 * A, rows, K, 1e-5, None)
            assert rms(A, K, 2 * A, K, H, ldh, H, *tail) == INVALID and "sum overlaps gamma" in err()
            assert layer(A, K, 2 * A, K, H, ldh, H, None, *tail) == INVALID and "sum overlaps gamma" in err()
            assert layer(A, K, 2 * A, K, H, ldh, None, H, *tail) == INVALID and "sum overlaps beta" in err()


def test_only_the_residual_may_be_the_output(lib):
    for f, e in ((lib.dlm_linear_q8_fp16, 2), (lib.dlm_linear_q8_f32out, 4)):
        def call(X=A, sx=2 * A, W=3 * A, sw=4 * A, bias=None, act=0):
            # R is Y, with the same row stride; the operand named below is there too
            return f(X, 64, sx, W, 64, sw, bias, 6 * A, 64, 6 * A, 64, 4, 32, 64, 1.0, act, None)

        for k in ("X", "W", "sx", "sw", "bias"):
            for act in (0, 2):
                assert call(**{k: 6 * A}, act=act) == INVALID and "Y overlaps " + k in err()


def test_interleaved_slices_that_share_a_column_are_refused(lib):
    for t, e in (("fp16", 2), ("f32", 4)):
        # rows of 64 columns: x and the sum take 40 each, from column 0 and from 24 or 39
        for at in (24, 39):
            st = getattr(lib, f"dlm_rms_norm_q8_{t}")(A, 64, 2 * A, 64, A + at * e, 64, None, 5 * A, 64, 6 * A, 4, 40,
                                                      1e-5, None)
            assert st == INVALID and "sum overlaps x" in err()
            # ... the sum first, and x wrapping into the row after it
            st = getattr(lib, f"dlm_rms_norm_q8_{t}")(A + at * e, 64, 2 * A, 64, A, 64, None, 5 * A, 64, 6 * A, 4, 40,
                                                      1e-5, None)
            assert st == INVALID and "sum overlaps x" in err()
        f = lib.dlm_linear_q8_fp16 if e == 2 else lib.dlm_linear_q8_f32out
        for at in (1, 31, 33, 63):
            assert f(A, 64, 2 * A, 3 * A, 64, 4 * A, None, 6 * A + at * e, 64, 6 * A, 64, 4, 32, 64, 1.0, 0,
                     None) == INVALID and "Y overlaps R" in err()


def test_forced_tiles_are_those_there_are(lib):
    for tile in (-1, 15, 1 << 20):
        assert lib.dlm_q8_force_tile(tile) == INVALID and "[0, 14]" in err()
    assert lib.dlm_q8_force_tile(14) == 0 and lib.dlm_q8_force_tile(0) == 0


def test_wrappers_refuse_host_tensors():
    x, s = torch.zeros(4, 64, dtype=torch.float16), torch.ones(4)
    q = torch.zeros(4, 64, dtype=torch.int8)
    for f, args in ((ops.quantize_rows, (x,)), (ops.dequantize_rows, (q, s)), (ops.rms_norm_q8, (x,)),
                    (ops.layer_norm_q8, (x,)), (ops.linear_q8, (q, s, q, s))):
        with pytest.raises(ValueError):
            f(*args)


def test_oracle_rows():
    v = torch.tensor([[254.0, 1.0, 3.0, -1.0, -3.0, -254.0], [0.0] * 6], dtype=torch.float64)
    t, q, s = Q.rows(v)
    assert q[0].tolist() == [127, 0, 2, 0, -2, -127]  # halves to even
    assert q[1].tolist() == [0] * 6 and s.tolist() == [2.0, 0.0]


def test_oracle_linear_geglu_groups():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randint(-9, 9, (3, 8), generator=g), torch.randint(-9, 9, (16, 8), generator=g)
    one = torch.ones(16)
    y, _ = Q.linear(x, one[:3], w, one * 0.1, act="geglu")
    z = 0.1 * (x.double() @ w.double().t())
    for j in range(8):
        v, t = z[:, j // 4 * 8 + j % 4], z[:, j // 4 * 8 + 4 + j % 4]
        assert torch.allclose(y[:, j], v * 0.5 * t * (1 + torch.erf(t / 2 ** 0.5)), atol=1e-6)
