"""What the prompt attention and the 4-bit cache refuse at the ends of their ranges, and their build, without a GPU."""

import ctypes

import pytest
import torch

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


@pytest.mark.parametrize('n, heads, kv, max_len, dim', [(1, 1 << 20, 1, 1 << 28, 64), (1, 1 << 18, 1, 1 << 30, 64), (4, 1 << 20, 4, 1 << 28, 128),
                                                        (1, 16, 1, 1 << 30, 64), (4096, 64, 8, 1 << 17, 128), (64, 32, 8, 131072, 128)])
def test_decode_workspace_is_bounded(built_lib, n, heads, kv, max_len, dim):
    """However many keys there are in all items, they are at most 8192 chunks and one more an item: (m, l, O) of each."""
    group = heads // kv
    items, cols = kv * -(-group // 16), min(16, group)
    floats = built_lib.fw_decode_attention_q4_ws_floats(n, heads, kv, max_len, dim)
    assert 0 < floats <= (8192 + n * items) * cols * (dim + 2) + 4


@pytest.mark.parametrize('rows, heads, kv', [(1 << 62, 80, 20), (1 << 61, 8, 1), (0x7FFFFF01, 20, 20), (0x7FFFFF00 // 4 + 1, 80, 20)])
def test_prompt_rows_times_heads(built_lib, rows, heads, kv):
    """The rows of a group's heads are counted in 32 bits; more are refused however large, also where the product wraps round."""
    from flash_whisper_amd import _lib

    assert _prompt(built_lib, q_rows=rows, heads=heads, kv=kv) == _lib.FW_EINVAL
    assert b'too many rows' in built_lib.fw_last_error()


@pytest.mark.parametrize('rows, heads, dim', [((1 << 40) - 32, 1 << 27, 64), ((1 << 40) - 32, 1 << 26, 128), (1 << 62, 1 << 30, 128), (1 << 10, 1 << 30, 128),
                                              (1 << 62, 1, 64)])
def test_cache_rows_times_heads(built_lib, rows, heads, dim):
    """An append or a read of more waves than a grid has is refused, also where their number wraps round 64 bits."""
    from flash_whisper_amd import _lib

    strides, cache, sizes = (64, 64), (D16, D16, D16, D16), (2, heads, 32, dim)
    assert built_lib.fw_kv_q4_append(D16, *strides, D16, *strides, rows, D16, D16, *cache, *sizes, 0, None) == _lib.FW_EINVAL
    assert b'too many rows' in built_lib.fw_last_error()
    assert built_lib.fw_kv_q4_read(*cache, *sizes, D16, D16, rows, D16, *strides, D16, *strides, 0, None) == _lib.FW_EINVAL
    assert b'too many rows' in built_lib.fw_last_error()


def test_decode_heads_past_a_grid(built_lib):
    """More heads than the joining launch has blocks for are refused before anything is launched."""
    from flash_whisper_amd import _lib

    strides = (64, 64)
    assert built_lib.fw_decode_attention_q4(D16, *strides, D16, D16, D16, D16, D16, D16, *strides, None, *strides, None, *strides, 1, 1 << 25, 1,
                                            4096, 64, 0, 0.125, D16, 1 << 60, None) == _lib.FW_EINVAL
    assert b'too many heads' in built_lib.fw_last_error()


@pytest.mark.parametrize('cache', [None, (), 7, (torch.zeros(1, 1, 32, 32),) * 3, (None,) * 4, [None] * 4])
def test_not_a_cache(built_lib, cache):
    """Anything but a cache's four arrays is a RuntimeError, as every invalid argument is."""
    from flash_whisper_amd.ext import load_ext

    ext = load_ext()
    x, cu = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ext.kv_q4_append(x, x, cu, cu[:1], cache), lambda: ext.kv_q4_read(cache, cu, cu[:1], x, x),
                 lambda: ext.decode_attention_q4(x[:1], cache, cu[:1], x[:1], torch.zeros(4), 0.125),
                 lambda: ext.decode_attention_q4_workspace(1, 2, cache)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize('missing', ['compiler', 'headers', 'torch'])
def test_build_without_the_binding(monkeypatch, tmp_path, capsys, missing):
    """No C++ compiler, one that fails, no torch to compile against: the build says so, leaves no binding of an earlier one
    behind and goes on."""
    import sys

    from flash_whisper_amd import build

    monkeypatch.setattr(build, 'BIND_LIB', tmp_path / '_bind.so')
    (tmp_path / '_bind.so').write_bytes(b'an earlier one')
    if missing == 'torch':
        monkeypatch.setitem(sys.modules, 'torch.utils.cpp_extension', None)
    else:
        monkeypatch.setenv('CXX', str(tmp_path / 'none') if missing == 'compiler' else 'false')
    assert build._compile_bind(False) is False
    assert not list(tmp_path.iterdir()) and 'ctypes' in capsys.readouterr().err


def test_prompt_forms(built_lib):
    """What the library says of sizes on either side of its rule, and of sizes that it refuses."""
    from flash_whisper_amd import _lib

    form = built_lib.fw_prompt_attention_form
    assert form(1, 4, 4, 20, 20, 64, 1) == _lib.PROMPT_WAVES and form(64, 64 * 32, 64 * 32, 20, 20, 64, 1) == _lib.PROMPT_WAVES
    assert form(64, 64 * 33, 64 * 33, 20, 20, 64, 1) == _lib.PROMPT_128_ROWS and form(4, 4 * 33, 4 * 33, 20, 20, 64, 1) == _lib.PROMPT_2_SHORT_PARTS
    assert form(1, 4, 1500, 20, 20, 64, 0) == _lib.PROMPT_8_PARTS and form(1, 4, 511, 20, 20, 64, 0) == _lib.PROMPT_2_PARTS
    assert form(1, 2000, 2000, 20, 20, 64, 1) == _lib.PROMPT_2_PARTS and form(1, 2000, 2000, 20, 20, 64, 0) == _lib.PROMPT_2_SHORT_PARTS
    assert form(1, 8192, 8192, 32, 8, 128, 1) == _lib.PROMPT_128_ROWS
    for bad in ((0, 4, 4, 20, 20, 64), (1, -1, 4, 20, 20, 64), (1, 4, 4, 20, 8, 64), (1, 4, 4, 20, 20, 80), (1, 1 << 31, 4, 20, 20, 64)):
        assert form(*bad, 1) == _lib.FW_EINVAL


def test_views_without_rows():
    """The strides of a tensor without rows mean nothing; its heads, head size and type are still asked for."""
    from flash_whisper_amd import ext

    none, f16 = torch.empty(0).half().as_strided((0, 2, 64), (1, 3, 2)), torch.float16
    for view in (ext._heads_view, ext._out_view):
        assert view(none, 'k', f16, -1, 2, 64) == (0, 0) and view(none, 'k', f16, -1, None, 64) == (0, 0)
        for args in ((f16, -1, 3, 64), (f16, -1, 2, 128), (torch.bfloat16, -1, 2, 64), (f16, 0, 2, 64)):
            with pytest.raises(RuntimeError):
                view(none, 'k', *args)
        with pytest.raises(RuntimeError):
            view(torch.zeros(400, dtype=f16).as_strided((1, 2, 64), (1, 3, 2)), 'k', f16, -1, 2, 64)
