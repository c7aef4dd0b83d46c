"""The prompt attention and the 4-bit cache without a GPU: what their entry points refuse, at the C ABI and at the
torch level, and the float64 oracle of the cache against its layout's definition."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import serving

D16 = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)
CACHE = (D16, D16, D16, D16)


def _prompt(lib, q=D16, k=D16, out=D16, strides=(1280, 64), cu=D16, n=2, rows=8, heads=20, kv=20, dim=64, dtype=0):
    return lib.fw_prompt_attention(q, *strides, k, *strides, D16, *strides, out, *strides, cu, cu, n, rows, rows, heads, kv,
                                   dim, dtype, 0.125, 1, None)


@pytest.mark.parametrize('what, message', [
    (dict(n=0), b'n_seq must be positive'), (dict(rows=-1), b'rows not negative'), (dict(heads=20, kv=8), b'multiple of kv_heads'),
    (dict(heads=0, kv=1), b'multiple of kv_heads'), (dict(kv=0), b'multiple of kv_heads'), (dict(dim=80), b'64 or 128'),
    (dict(dtype=2), b'FW_F16 or FW_BF16'), (dict(cu=None), b'null'), (dict(q=None), b'null'), (dict(k=None), b'null'),
    (dict(out=None), b'null'), (dict(q=ODD), b'16-byte aligned'), (dict(out=ODD), b'16-byte aligned'),
    (dict(strides=(1284, 64)), b'multiples of 8'), (dict(strides=(1280, 66)), b'multiples of 8')])
def test_prompt_attention_refuses(built_lib, what, message):
    from flash_whisper_amd import _lib

    assert _prompt(built_lib, **what) == _lib.FW_EINVAL
    assert message in built_lib.fw_last_error()


def _append(lib, k=D16, cu=D16, rows=8, cache=CACHE, n=2, heads=20, max_len=448, dim=64, dtype=0, strides=(1280, 64)):
    return lib.fw_kv_q4_append(k, *strides, D16, *strides, rows, cu, D16, *cache, n, heads, max_len, dim, dtype, None)


def _read(lib, k=D16, cu=D16, rows=8, cache=CACHE, n=2, heads=20, max_len=448, dim=64, dtype=0, strides=(1280, 64)):
    return lib.fw_kv_q4_read(*cache, n, heads, max_len, dim, cu, D16, rows, k, *strides, D16, *strides, dtype, None)


def _decode(lib, q=D16, lens=D16, cache=CACHE, n=2, heads=20, kv=20, max_len=448, dim=64, dtype=0, strides=(1280, 64),
            k_new=None, v_new=None, ws=D16, ws_floats=1 << 40):
    return lib.fw_decode_attention_q4(q, *strides, *cache, lens, D16, *strides, k_new, *strides, v_new, *strides, n, heads, kv,
                                      max_len, dim, dtype, 0.125, ws, ws_floats, None)


CACHE_REFUSALS = [(dict(max_len=440), b'multiple of 32'), (dict(max_len=0), b'multiple of 32'), (dict(dim=32), b'64 or 128'),
                  (dict(n=0), b'must be positive'), (dict(cache=(D16, None, D16, D16)), b'null'),
                  (dict(cache=(D16, D16, ODD, D16)), b'16-byte aligned'), (dict(dtype=-1), b'FW_F16 or FW_BF16'),
                  (dict(strides=(1284, 64)), b'multiples of 8')]


@pytest.mark.parametrize('call', [_append, _read])
@pytest.mark.parametrize('what, message', CACHE_REFUSALS + [(dict(rows=-1), b'not be negative'), (dict(k=None), b'null'),
                                                            (dict(cu=None), b'null'), (dict(heads=0), b'must be positive'),
                                                            (dict(k=ODD), b'16-byte aligned'),
                                                            (dict(rows=1 << 40), b'too many rows')])
def test_cache_rows_refuse(built_lib, call, what, message):
    from flash_whisper_amd import _lib

    assert call(built_lib, **what) == _lib.FW_EINVAL
    assert message in built_lib.fw_last_error()


@pytest.mark.parametrize('what, message', CACHE_REFUSALS + [
    (dict(q=None), b'null'), (dict(lens=None), b'null'), (dict(heads=20, kv=8), b'multiple of kv_heads'), (dict(q=ODD), b'16-byte aligned'),
    (dict(k_new=D16), b'given together'), (dict(v_new=D16), b'given together'), (dict(k_new=ODD, v_new=D16), b'16-byte aligned'),
    (dict(ws=None), b'workspace needs'), (dict(ws=ODD), b'workspace needs'), (dict(ws_floats=0), b'workspace needs')])
def test_decode_refuses(built_lib, what, message):
    from flash_whisper_amd import _lib

    assert _decode(built_lib, **what) == _lib.FW_EINVAL
    assert message in built_lib.fw_last_error()


def test_no_rows_is_no_launch(built_lib):
    """A call without rows returns before any HIP call, null pointers or not."""
    from flash_whisper_amd import _lib

    assert _prompt(built_lib, rows=0, q=None, k=None, out=None) == _lib.FW_OK
    assert _append(built_lib, rows=0, k=None) == _lib.FW_OK and _read(built_lib, rows=0, k=None) == _lib.FW_OK


def test_workspace_sizes(built_lib):
    need = built_lib.fw_decode_attention_q4_ws_floats
    assert need(1, 20, 20, 448, 64) > 0 and need(64, 32, 8, 8192, 128) > 0
    for bad in ((0, 20, 20, 448, 64), (1, 20, 8, 448, 64), (1, 20, 20, 440, 64), (1, 20, 20, 448, 96), (1, 0, 20, 448, 64)):
        assert need(*bad) == 0


def test_torch_level_checks(built_lib):
    """Tensors off the GPU, of another type or shape raise before the library is called."""
    from flash_whisper_amd.ext import load_ext

    ext = load_ext()
    q, cu = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match='current device'):
        ext.prompt_attention(q, q, q, q.clone(), cu, cu, 0.125)
    with pytest.raises(RuntimeError, match='fp16 or bf16'):
        ext.prompt_attention(q.float(), q, q, q, cu, cu, 0.125)
    with pytest.raises(RuntimeError, match='64 or 128'):
        ext.prompt_attention(q[..., :32], q, q, q, cu, cu, 0.125)
    with pytest.raises(RuntimeError):
        ext.prompt_attention(None, q, q, q, cu, cu, 0.125)
    cache = ext.kv_q4_cache(2, 2, 50, 64, device='cpu')
    assert cache.k_codes.shape == (2, 2, 64, 32) and cache.v_meta.shape == (2, 2, 8, 2, 2, 8)
    with pytest.raises(RuntimeError, match='current device'):
        ext.kv_q4_append(q, q, cu, cu[:2], cache)
    with pytest.raises(RuntimeError, match='current device'):
        ext.decode_attention_q4(q[:2], cache, cu[:2], q[:2].clone(), torch.zeros(4), 0.125)
    with pytest.raises(RuntimeError, match='head_dim'):
        ext.kv_q4_cache(2, 2, 50, 80, device='cpu')
    with pytest.raises(RuntimeError, match='multiple of the cache'):
        ext.decode_attention_q4_workspace(2, 3, cache)


@pytest.mark.parametrize('dim', [64, 128])
def test_oracle_cache_rows(dim):
    """The oracle's rows come back within half a step (plus the roundings of low, step and the value), and its
    extreme groups stay finite; a group with an infinity reads back as NaN, its neighbours do not."""
    rng = np.random.default_rng(dim)
    cache = serving.empty_cache(2, 3, 32, dim, fill=0xAB)
    x = np.float16(rng.standard_normal((11, 2, 3, dim)) * np.exp(rng.standard_normal((11, 2, 3, 1)) * 2))
    x[0, 0, 0, :32] = np.tile(np.float16([-65504, 65504]), 16)
    x[1, 0, 0, :32] = 0.25
    for i in range(11):
        serving.write_row(cache, 1, 5 + i, x[i, 0], x[i, 1])
    for which, got in enumerate(serving.read_rows(cache, 1, range(5, 16))):
        want = x[:, which].astype(np.float64)
        g = want.reshape(11, 3, -1, 32)
        width = (g.max(-1) - g.min(-1)) / 15
        # half a step; the step is up to 2^-10 of itself short (15 times that at the top); the value rounded to fp16
        tol = (0.5 * width + 15 * 2.0 ** -10 * width)[..., None] + 2.0 ** -11 * np.abs(g).max(-1, keepdims=True) + 2.0 ** -25
        assert np.isfinite(got).all() and (np.abs(got.reshape(g.shape).astype(np.float64) - g) <= tol).all()
    untouched = serving.empty_cache(2, 3, 32, dim, fill=0xAB)
    assert np.array_equal(cache[0][0], untouched[0][0]) and np.array_equal(cache[2][1, :, 2:], untouched[2][1, :, 2:])
    x[2, 0, 1, 40] = np.inf
    serving.write_row(cache, 1, 7, x[2, 0], x[2, 1])
    k, _ = serving.read_rows(cache, 1, [7])
    assert np.isnan(k[0, 1, 32:64]).all() and np.isfinite(k[0, 1, :32]).all() and np.isfinite(k[0, 0]).all()


def test_binding_refuses_without_a_call(built_lib):
    """The compiled binding answers False, and makes no call, for anything that is not a valid call on the GPU named."""
    from flash_whisper_amd import _bind
    from flash_whisper_amd.ext import load_ext

    cache = load_ext().kv_q4_cache(2, 2, 64, 64, device='cpu')
    q, cu = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int64)
    for args in ((), (q, q, q, q, cu, cu, 0.125, True, 0, 0), (q, q, q, q, cu, cu, 'x', True, 0, 0), (None,) * 10,
                 (q, q, q, q, cu, cu, 0.125, True, 1 << 70, 0)):
        assert _bind.prompt_attention(*args) is False
    assert _bind.kv_q4_append(q, q, cu, cu[:2], cache, 0, 0) is False
    assert _bind.kv_q4_read(cache, cu, cu[:2], q, q, 0, 0) is False and _bind.kv_q4_read(None, cu, cu[:2], q, q, 0, 0) is False
    assert _bind.decode_attention_q4(q[:2], cache, cu[:2], q[:2], torch.zeros(4), 0.125, None, None, 0, 0) is False
    with pytest.raises(ValueError):
        _bind.set_entry('fw_other', 0)


@pytest.mark.parametrize('scale', [float('inf'), float('-inf'), float('nan')])
def test_scale_is_finite(built_lib, scale):
    from flash_whisper_amd import _lib

    strides = (1280, 64)
    assert built_lib.fw_prompt_attention(D16, *strides, D16, *strides, D16, *strides, D16, *strides, D16, D16, 2, 8, 8, 20, 20, 64,
                                         0, scale, 1, None) == _lib.FW_EINVAL
    assert b'scale must be finite' in built_lib.fw_last_error()
    assert built_lib.fw_decode_attention_q4(D16, *strides, *CACHE, D16, D16, *strides, None, *strides, None, *strides, 2, 20, 20,
                                            448, 64, 0, scale, D16, 1 << 40, None) == _lib.FW_EINVAL
    assert b'scale must be finite' in built_lib.fw_last_error()


@pytest.mark.parametrize('call, what, message', [
    (_prompt, dict(rows=1 << 31, heads=20, kv=20), b'too many rows'),          # rows of a sequence in 32 bits
    (_prompt, dict(rows=1 << 30, heads=64, kv=64), b'too many rows'),          # 2^23 blocks x 64 heads x 256 threads
    (_append, dict(rows=1 << 26, heads=8, dim=64), b'too many rows'),          # 2^23 x 8 waves of 64 threads: 2^32 and a few
    (_read, dict(rows=1 << 28, heads=8, dim=128), b'too many rows'),
    (_append, dict(rows=1 << 62), b'too many rows'),
    (_append, dict(max_len=(1 << 30) + 32), b'up to 2^30'),
    (_decode, dict(max_len=(1 << 30) + 32), b'up to 2^30'),
    (_decode, dict(n=65536), b'too many sequences'),
    (_decode, dict(n=65535, heads=512, kv=512), b'too many sequences')])       # 2^25 blocks of 256 threads
def test_calls_past_a_grid(built_lib, call, what, message):
    from flash_whisper_amd import _lib

    assert call(built_lib, **what) == _lib.FW_EINVAL
    assert message in built_lib.fw_last_error()
