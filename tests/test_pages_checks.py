"""The cache in pages and the rules on logits without a GPU: what their entry points refuse, at the C ABI and at the torch
level, and the oracle against hand-made cases."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import pages as oracle

D16, ODD = ctypes.c_void_p(16), ctypes.c_void_p(24)


def _map(lib, pos=D16, table=D16, own=None, stack=D16, slots=D16, n=2, width=4, size=8, rows=3, page=16):
    return lib.fw_kv_page_map(pos, D16, table, D16, own, stack, D16, D16, D16, slots, n, width, size, rows, page, None)


def _append(lib, k=D16, slots=D16, cache=D16, strides=(128, 64), rows=3, n=4, heads=2, page=16, dim=64):
    return lib.fw_kv_page_append(k, *strides, D16, *strides, slots, rows, cache, D16, n, heads, page, dim, None)


def _attend(lib, q=D16, k=D16, table=D16, cu=None, shared=None, strides=(128, 64), n=2, heads=2, kv=2, pages=4, page=16, width=4,
            groups=0, dim=64, dtype=0, scale=0.125, ws=D16, floats=1 << 40):
    return lib.fw_decode_attention_paged(q, *strides, k, D16, table, D16, cu, shared, D16, *strides, n, heads, kv, pages, page, width,
                                         groups, dim, dtype, scale, ws, floats, None)


def _rules(lib, x=D16, rows=2, vocab=100, dtype=0, tokens=None, n_tokens=0, cu=None, rep=None, ids=None, bias=None, n_bias=0,
           cu_bias=None, masks=None, words=4, sets=1, of=None):
    return lib.fw_logits_rules(x, vocab, D16, vocab, rows, vocab, dtype, tokens, n_tokens, cu, None, rep, None, None, ids, bias, n_bias,
                               cu_bias, masks, words, sets, of, None)


@pytest.mark.parametrize('call, what, message', [
    (_map, dict(page=8), b'page must be'), (_map, dict(page=48), b'page must be'), (_map, dict(n=0), b'must be positive'),
    (_map, dict(width=0), b'must be positive'), (_map, dict(rows=-1), b'not negative'), (_map, dict(size=-1), b'not negative'),
    (_map, dict(width=(1 << 20) + 1), b'2^20'), (_map, dict(rows=1 << 31), b'2^31'), (_map, dict(pos=None), b'null'),
    (_map, dict(table=None), b'null'), (_map, dict(stack=None), b'null'), (_map, dict(slots=None), b'null'),
    (_append, dict(page=512), b'page must be'), (_append, dict(dim=96), b'64 or 128'), (_append, dict(n=0), b'must be positive'),
    (_append, dict(heads=0), b'must be positive'), (_append, dict(rows=-1), b'not negative'), (_append, dict(k=None), b'null'),
    (_append, dict(slots=None), b'null'), (_append, dict(cache=None), b'null'), (_append, dict(k=ODD), b'aligned'),
    (_append, dict(cache=ODD), b'aligned'), (_append, dict(strides=(132, 64)), b'multiples of 8'), (_append, dict(rows=1 << 40), b'too many rows'),
    (_append, dict(rows=1 << 62), b'too many rows'), (_append, dict(rows=8, heads=1 << 30), b'too many rows'),
    (_attend, dict(page=0), b'page must be'), (_attend, dict(dim=80), b'64 or 128'), (_attend, dict(n=0), b'must be positive'),
    (_attend, dict(width=0), b'must be positive'), (_attend, dict(groups=-1), b'not negative'), (_attend, dict(heads=3), b'multiple of kv_heads'),
    (_attend, dict(kv=0), b'multiple of kv_heads'), (_attend, dict(heads=0), b'multiple of kv_heads'), (_attend, dict(width=1 << 27), b'2^30'),
    (_attend, dict(n=65536), b'too many sequences'), (_attend, dict(heads=(1 << 14) + 2), b'too many heads'), (_attend, dict(pages=0), b'n_pages'),
    (_attend, dict(dtype=2), b'FW_F16 or FW_BF16'), (_attend, dict(q=None), b'null'), (_attend, dict(k=None), b'null'),
    (_attend, dict(table=None), b'null'), (_attend, dict(groups=1), b'null'), (_attend, dict(groups=1, cu=D16), b'null'),
    (_attend, dict(scale=float('nan')), b'scale must be finite'), (_attend, dict(scale=2.5e38), b'scale must be finite'),
    (_attend, dict(q=ODD), b'aligned'), (_attend, dict(k=ODD), b'aligned'), (_attend, dict(strides=(130, 64)), b'multiples of 8'),
    (_attend, dict(ws=None), b'workspace needs'), (_attend, dict(ws=ODD), b'workspace needs'), (_attend, dict(floats=0), b'workspace needs'),
    (_attend, dict(n=65535, heads=1 << 14, kv=1 << 14), b'too many sequences'),
    (_rules, dict(dtype=3), b'FW_F16, FW_BF16 or FW_F32'), (_rules, dict(rows=-1), b'not be negative'), (_rules, dict(vocab=0), b'vocab positive'),
    (_rules, dict(x=None), b'null'), (_rules, dict(tokens=D16), b'penalties need'), (_rules, dict(cu=D16), b'penalties need'),
    (_rules, dict(rep=D16), b'penalties need'), (_rules, dict(n_tokens=-1), b'negative'), (_rules, dict(n_bias=1 << 31), b'too many'),
    (_rules, dict(ids=D16), b'given together'), (_rules, dict(bias=D16), b'given together'), (_rules, dict(ids=D16, bias=D16), b'given together'),
    (_rules, dict(of=D16), b'masks must hold'), (_rules, dict(masks=D16, words=3), b'masks must hold'), (_rules, dict(masks=D16, sets=0), b'masks must hold'),
    (_rules, dict(masks=D16, rows=3, sets=2), b'masks must hold'), (_rules, dict(rows=1 << 30, vocab=100000), b'too many rows')])
def test_refused(built_lib, call, what, message):
    from flash_whisper_amd import _lib

    assert call(built_lib, **what) == _lib.FW_EINVAL
    assert message in built_lib.fw_last_error()


def test_no_rows_is_no_launch(built_lib):
    from flash_whisper_amd import _lib

    assert _append(built_lib, rows=0, k=None, slots=None) == _lib.FW_OK and _rules(built_lib, rows=0, x=None) == _lib.FW_OK


def test_workspace_sizes(built_lib):
    need = built_lib.fw_decode_attention_paged_ws_floats
    assert need(5, 20, 20, 28, 16, 1, 64) > 0 and need(64, 32, 8, 288, 32, 1, 128) > need(64, 32, 8, 288, 32, 0, 128) > 0
    for bad in ((0, 20, 20, 28, 16, 1, 64), (5, 20, 8, 28, 16, 1, 64), (5, 20, 20, 28, 24, 1, 64), (5, 20, 20, 0, 16, 1, 64),
                (5, 20, 20, 28, 16, -1, 64), (5, 20, 20, 28, 16, 1, 96), (1 << 20, 20, 20, 28, 16, 1, 64)):
        assert need(*bad) == 0
    # results of every piece there may be: 512 blocks' worth, one more for a run of a group's columns, one more a sequence; and the plan
    for n, heads, kv, groups, dim in ((1, 1, 1, 0, 64), (65535, 64, 8, 60000, 128), (4096, 16384, 1, 3, 64), (64, 16384, 16384, 60, 64), (64, 32, 8, 1, 128)):
        group, want = heads // kv, max(1, 512 // kv)
        slots = max(c // 16 * (want + n * group // c + groups) for c in (16, 64, 128)) + n * -(-group // 16) + 1
        assert 0 < need(n, heads, kv, 1 << 20, 256, groups, dim) <= slots * (kv * 16 * (dim + 2) + 8) + 11 * n + 5 * groups + 16


def _cpu_cache(ext, dtype=torch.float16):
    return ext.kv_pages(4, 2, 16, 64, dtype, device='cpu')


def test_torch_level_checks(built_lib):
    """Tensors off the GPU, of another type or shape raise before the library is called."""
    from flash_whisper_amd.ext import KvPages, load_ext

    ext = load_ext()
    cache = _cpu_cache(ext)
    assert cache.k.shape == (4, 2, 16, 64) and cache.v.shape == (4, 2, 2, 64, 8)
    q, i64, i32 = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int32)
    f32 = torch.zeros(3)
    calls = [lambda: ext.kv_page_map(i64[:3], i64, i32, i64[:3], i32[0], i64[:2], i64, 16),
             lambda: ext.kv_page_append(q, q, i64[:3], cache), lambda: ext.decode_attention_paged(q, cache, i32, i64[:3], q, f32, 0.1),
             lambda: ext.logits_rules(f32[None], f32[None])]
    for call in calls:
        with pytest.raises(RuntimeError, match='current device'):
            call()
    for bad in (None, (), (cache.k,), (cache.k, None), KvPages(cache.k, cache.v.float()), 7):
        for call in (lambda: ext.kv_page_append(q, q, i64[:3], bad), lambda: ext.decode_attention_paged(q, bad, i32, i64[:3], q, f32, 0.1)):
            with pytest.raises(RuntimeError):
                call()
    for bad in ((0, 2, 16, 64), (4, 0, 16, 64), (4, 2, 24, 64), (4, 2, 16, 80), (4, 2, 16, 64, torch.float32)):
        with pytest.raises(RuntimeError, match='page one of'):
            ext.kv_pages(*bad, device='cpu')
    with pytest.raises(RuntimeError, match='multiple of kv_heads'):
        ext.decode_attention_paged_workspace(3, 3, cache, 2)
    assert ext.decode_attention_paged_workspace(3, 4, cache, 2, 1).dtype == torch.float32
    for args in ((None, None), (f32, None), (None, f32)):
        with pytest.raises(RuntimeError):
            ext.logits_rules(*args)


def test_binding_refuses_without_a_call(built_lib):
    """The compiled binding answers False, and makes no call, for anything that is not a valid call on the GPU named."""
    from flash_whisper_amd import _bind
    from flash_whisper_amd.ext import load_ext

    cache = _cpu_cache(load_ext())
    q, i64, i32, f32 = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3)
    none = (None,) * 3
    for call, args in ((_bind.kv_page_map, (i64[:3], i64, i32, i64[:3], i32[0], i64[:2], i64, 16, *none, 0, 0)), (_bind.kv_page_append, (q, q, i64[:3], cache, 0, 0)),
                       (_bind.decode_attention_paged, (q, cache, i32, i64[:3], q, f32, 0.1, None, None, 0, 0)),
                       (_bind.logits_rules, (f32[None], f32[None], *none, *none, *none, None, None, 0, 0))):
        assert call(*args) is False and call() is False and call(*args[:-1]) is False and call(*(None,) * len(args)) is False
        assert call(*args[:-2], 1 << 70, 0) is False


def test_oracle_map():
    """A sequence that ends gives its pages to one that grows; shared entries are only dropped; what is missing is counted."""
    table = [[5, 6, 7], [1, 0, 0], [2, 3, 0]]
    got = oracle.page_map([0, 16, -1], [0, 0, 33, 35], table, [3, 1, 2], [1, 0, 0], [9] * 4, 0, 36, 16)
    assert got[0].tolist() == [[5, 6, 7], [1, 7, 6], [2, 3, 0]] and got[1] == [0, 3, 2] and got[2] == [6, 7, 9, 9] and got[3] == [0, 1]
    assert got[4] == [112 + i for i in range(16)] + [96 + i for i in range(16)] + [-1, -1, -1, None]


def test_oracle_rules():
    x = np.array([[2.0, -2.0, 1.0, 0.0]])
    got, _ = oracle.rules(x, tokens=np.array([0, 1, 2, 2, 9]), cu=[0, 5], prompt=[2], repetition=[2.0], presence=[0.5], frequency=[0.25],
                          bias_ids=np.array([3, 3]), bias=[7.0, 1.0], cu_bias=[0, 2], masks=np.array([[0b1110]], np.int32))
    assert got.tolist() == [[float('-inf'), -4.0, 0.5 - 0.5 - 0.5, 1.0]]


def test_oracle_rows():
    """Rows appended to a cache come back by table, in their order."""
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 40, 2, 64))
    table = np.array([3, 0, 2])
    slots = [int(table[j // 16]) * 16 + j % 16 for j in range(40)]
    cache = oracle.append(np.zeros((4, 2, 16, 64)), np.zeros((4, 2, 2, 64, 8)), k, v, slots)
    got = oracle.rows_of(*cache, table, 40)
    assert np.array_equal(got[0], k) and np.array_equal(got[1], v)
    table[1] = -1
    assert np.array_equal(oracle.rows_of(*cache, table, 40)[0], np.concatenate([k[:16], k[32:]]))


def test_workspace_of_padded_groups(built_lib):
    """As many groups as sequences, or more, may be a few large ones among empty ones: there is room for what these leave."""
    need = built_lib.fw_decode_attention_paged_ws_floats
    for n in (2, 5, 64, 300):
        assert need(n, 32, 8, 288, 32, n, 128) > need(n, 32, 8, 288, 32, 0, 128) < need(n, 32, 8, 288, 32, 4 * n, 128)
    assert need(1, 32, 8, 288, 32, 1, 128) == need(1, 32, 8, 288, 32, 0, 128)  # nobody to share with
