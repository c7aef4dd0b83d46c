"""What the prompt attention and the 4-bit cache refuse at the ends of their ranges, and their build, without a GPU."""

import ctypes

import pytest

D16 = ctypes.c_void_p(16)


def _prompt(lib, q_rows=8, k_rows=8, n=2, heads=20, kv=20, dim=64, dtype=0, scale=0.125):
    strides = (heads * dim, dim)
    return lib.fw_prompt_attention(D16, *strides, D16, kv * dim, dim, D16, kv * dim, dim, D16, *strides, D16, D16, n, q_rows, k_rows,
                                   heads, kv, dim, dtype, scale, 1, None)


@pytest.mark.parametrize('scale', [2.5e38, -3.4e38])
def test_prompt_scale_past_the_exponent(built_lib, scale):
    """Scores are kept in powers of two: scale log2(e) has to be a number."""
    from flash_whisper_amd import _lib

    assert _prompt(built_lib, scale=scale) == _lib.FW_EINVAL
    assert b'scale must be finite' in built_lib.fw_last_error()
