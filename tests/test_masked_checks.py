"""More argument checks of the rotary, norm and masked-attention entry points at the C boundary, without a
device: every refused call returns before anything is launched (CPU only)."""
import ctypes

from test_masked import A, INVALID, attention_args, err, lib, rotary_args  # noqa: F401 (lib: a fixture)


def qk(lib, **kw):
    return lib.dlm_qk_norm_rotary(ctypes.byref(rotary_args(**kw)), None)


def test_tokens_that_a_grid_takes(lib):
    """64 lanes a token where heads are wide or unaligned, in whole blocks of four tokens: fewer than 2^32."""
    for tokens in ((1 << 26) - 3, (1 << 26) - 1, 1 << 26):
        assert qk(lib, B=1, S=tokens) == INVALID and "2^26 - 4 tokens" in err(), (tokens, err())
    assert qk(lib, B=1, S=(1 << 26) - 4, H=65536) == INVALID and "65535" in err()
