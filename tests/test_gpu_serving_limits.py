"""The prompt attention and the 4-bit cache at the ends of what their entry points take: scales, values and sizes."""

import numpy as np
import pytest
import torch

from oracle import serving
from serving_tools import TYPES, check_attention, check_prompts, rounded, starts, to_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ext(hip_device):
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def _index(x, dev):
    return torch.tensor(x, dtype=torch.int64, device=dev)


def _cache_of(k, v, max_len, dim, dev):
    """A cache whose one sequence holds rows k, v [rows, heads, dim], on the device and as the oracle's arrays."""
    want = serving.empty_cache(1, k.shape[1], max_len, dim, fill=0xFF)
    for i in range(len(k)):
        serving.write_row(want, 0, i, k[i].float().numpy(), v[i].float().numpy())
    return to_device(want, dev), want


@pytest.mark.parametrize('keys', [1, 32, 37, 300])
@pytest.mark.parametrize('exponent', [-126, -60, 0, 100])
def test_decode_scale_of_zero(ext, hip_device, exponent, keys):
    """A scale of zero weighs all keys alike, however small or large a bf16 query is, and where the last tile is not whole."""
    dev, rng = hip_device, np.random.default_rng(keys)
    k, v = (rounded(rng, (keys, 1, 64), torch.float16)[0] for _ in range(2))
    cache, want = _cache_of(k, v, 320, 64, dev)
    q = (rounded(rng, (1, 2, 64), torch.bfloat16)[0].float() * 2.0 ** exponent).bfloat16()
    out = torch.full((1, 2, 64), 9.0, dtype=torch.bfloat16, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index([keys], dev), out, ext.decode_attention_q4_workspace(1, 2, cache), 0.0)
    k64, v64 = serving.read_rows(want, 0, range(keys))
    o, spread, size = serving.attend(q.double().numpy(), k64, v64, 0.0, False)
    check_attention(out.double().cpu().numpy(), o, spread, size, np.abs(v64.astype(np.float64)).max(), keys, torch.bfloat16)


@pytest.mark.parametrize('scale', [1.0, -1.0, 0.125])
def test_decode_large_queries(ext, hip_device, scale):
    """The largest bf16 queries over keys that are zero where they are not: scores of zero stay zero, all keys weigh alike."""
    dev, rng = hip_device, np.random.default_rng(2)
    k, v = (rounded(rng, (37, 1, 64), torch.float16)[0] for _ in range(2))
    k[:, :, :32] = 0
    cache, want = _cache_of(k, v, 64, 64, dev)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    q[:, :, 3] = 3e38
    out = torch.full((1, 2, 64), 9.0, dtype=torch.bfloat16, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index([37], dev), out, ext.decode_attention_q4_workspace(1, 2, cache), scale)
    k64, v64 = serving.read_rows(want, 0, range(37))
    o, spread, size = serving.attend(q.double().numpy(), k64, v64, scale, False)
    assert not size.any()
    check_attention(out.double().cpu().numpy(), o, spread, size, np.abs(v64.astype(np.float64)).max(), 37, torch.bfloat16)


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('scale', [0.0, -0.0, 2.0 ** -119, -2.0 ** -119])
def test_prompt_small_scales_of_large_scores(ext, hip_device, scale, causal, dim):
    """bf16 queries and keys whose products are near 2^120: a scale of zero weighs all keys alike all the same, and one of
    2^-119 gives ordinary scores."""
    dev, rng = hip_device, np.random.default_rng(dim)
    q, k = ((rounded(rng, (90, 2, dim), torch.bfloat16)[0].float() * 2.0 ** 57).bfloat16() for _ in range(2))
    v, v64 = rounded(rng, (90, 2, dim), torch.bfloat16)
    out, cu = torch.empty(90, 2, dim, dtype=torch.bfloat16, device=dev), starts([50, 40], dev)
    ext.prompt_attention(q.to(dev), k.to(dev), v.to(dev), out, cu, cu, scale, causal)
    check_prompts(out.double().cpu().numpy(), q.double().numpy(), k.double().numpy(), v64, [50, 40], [50, 40], scale, causal, torch.bfloat16)


def test_prompt_scale_of_zero_no_numbers(ext, hip_device):
    """A scale of zero does not turn a query that is no number into one."""
    dev, rng = hip_device, np.random.default_rng(6)
    q, k, v = (rounded(rng, (40, 2, 64), torch.float16)[0].to(dev) for _ in range(3))
    q[3, 1, 5], q[4, 0, 6] = float('nan'), float('inf')
    out, cu = torch.empty_like(q), starts([40], dev)
    ext.prompt_attention(q, k, v, out, cu, cu, 0.0)
    bad = out.isnan().all(-1)
    assert bad[3, 1] and bad[4, 0] and bad.sum() == 2 and out.isnan().sum() == 128


@pytest.mark.parametrize('fresh', [False, True])
@pytest.mark.parametrize('values, good', [([65280.0, -65280.0, 1.0], True), ([65536.0, 0.0, 1.0], False), ([1e6, 7e4, 9e4, 100.0], False),
                                          ([-65536.0, 5.0], False), ([-3e38, 3e38], False), ([1e-30, -2e-9], True), ([3e-5, 0.0, 1e-5], True)])
def test_cache_bf16_past_fp16(ext, hip_device, values, good, fresh):
    """A bf16 group whose values fp16 does not reach reads back as NaN, none of it as other numbers, and as what the codes
    stand for below; the row's other group and the other head stay what they are. By an append, and by the decode's fresh row."""
    dev = hip_device
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    x[0, 0, :len(values)] = torch.tensor(values, dtype=torch.bfloat16)
    x[0, 0, 32:], x[0, 1] = torch.arange(32) / 8, torch.arange(64) / 16
    cache, cu, pos = ext.kv_q4_cache(1, 2, 32, 64), starts([1], dev), _index([0], dev)
    if fresh:
        out = torch.empty_like(x, device=dev)
        ext.decode_attention_q4(torch.zeros_like(x, device=dev), cache, pos, out, ext.decode_attention_q4_workspace(1, 2, cache), 0.125,
                                x.to(dev), x.to(dev))
    else:
        ext.kv_q4_append(x.to(dev), x.to(dev), cu, pos, cache)
    want = serving.empty_cache(1, 2, 32, 64)
    serving.write_row(want, 0, 0, x[0].float().numpy(), x[0].float().numpy())
    got = torch.empty_like(x, device=dev), torch.empty_like(x, device=dev)
    ext.kv_q4_read(cache, cu, pos, *got)
    for g, w in zip(got, serving.read_rows(want, 0, [0])):
        g, w = g.cpu(), torch.from_numpy(w).to(torch.bfloat16)
        bad = torch.zeros(1, 2, 64, dtype=torch.bool)
        bad[0, 0, :32] = not good
        assert torch.equal(w.isnan(), bad) and torch.equal(g.isnan(), bad) and torch.equal(g[~bad], w[~bad])


def test_decode_heads_times_rows(ext, hip_device):
    """2^20 query heads over one key/value head of 2^28 rows: 2^44 keys in all items, the chunk still a number of rows."""
    dev, rng = hip_device, np.random.default_rng(7)
    rows = 1 << 28
    empty = lambda dtype, *shape: torch.empty(1, 1, *shape, dtype=dtype, device=dev)
    cache = (empty(torch.uint8, rows, 32), empty(torch.float16, rows, 2, 2), empty(torch.uint8, rows // 8, 16, 16),
             empty(torch.float16, rows // 8, 2, 2, 8))
    k, v = (rounded(rng, (70, 1, 64), torch.float16)[0] for _ in range(2))
    ext.kv_q4_append(k.to(dev), v.to(dev), starts([70], dev), _index([0], dev), cache)
    want = serving.empty_cache(1, 1, 96, 64)
    for i in range(70):
        serving.write_row(want, 0, i, k[i].float().numpy(), v[i].float().numpy())
    few, q64 = rounded(rng, (1, 16, 64), torch.float16)
    q = few.to(dev).repeat(1, 1 << 16, 1)
    out = torch.full_like(q, 9.0)
    ext.decode_attention_q4(q, cache, _index([70], dev), out, ext.decode_attention_q4_workspace(1, 1 << 20, cache), 0.125)
    o, spread, size = serving.attend(q64, *serving.read_rows(want, 0, range(70)), 0.125, False)
    got = out.view(1, 1 << 16, 16, 64)
    assert torch.equal(got, got[:, :1].expand_as(got))
    check_attention(got[0, :1].double().cpu().numpy(), o, spread, size, np.abs(v.double().numpy()).max() * 1.1, 70, torch.float16)


@pytest.mark.parametrize('fresh', [False, True])
@pytest.mark.parametrize('kind, dim, n, heads, kv_heads, max_len', [('fp16', 64, 32, 256, 1, 40960), ('bf16', 128, 130, 8, 4, 40960),
                                                                    ('fp16', 64, 256, 32, 2, 40960)])
def test_decode_many_items_in_long_caches(ext, hip_device, kind, dim, n, heads, kv_heads, max_len, fresh):
    """512 items and more whose capacity would make chunks long: the few long sequences among them in chunks by the lengths,
    the fresh row at a chunk's end and the first of one; a captured call replayed with other lengths gives the bits of an eager
    one, and both the float64 values."""
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(n)
    cache = ext.kv_q4_cache(n, kv_heads, max_len, dim)
    ws = torch.full_like(ext.decode_attention_q4_workspace(n, heads, cache), float('nan'))
    q, q64 = rounded(rng, (n, heads, dim), dtype)
    k1, v1 = (torch.zeros(n, kv_heads, dim, dtype=dtype, device=dev) for _ in range(2))
    q, lens, out = q.to(dev), torch.full((n,), -1, dtype=torch.int64, device=dev), torch.empty(n, heads, dim, dtype=dtype, device=dev)
    call = lambda: ext.decode_attention_q4(q, cache, lens, out, ws, dim ** -0.5, *((k1, v1) if fresh else ()))
    rows = [3000, 5] + [int(x) for x in rng.integers(0, 40, n - 2)]
    rows[n // 2], rows[n - 1] = 9000, 2047
    k, v = (rounded(rng, (sum(rows), kv_heads, dim), dtype)[0].to(dev) for _ in range(2))
    ext.kv_q4_append(k, v, starts(rows, dev), torch.zeros_like(lens), cache)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    held_k, held_v = torch.empty_like(k, dtype=torch.float16), torch.empty_like(v, dtype=torch.float16)
    ext.kv_q4_read(cache, starts(rows, dev), torch.zeros_like(lens), held_k, held_v)
    for few in (0, 256, 255, 1 << 20):  # the long ones cut to some rows, or not at all
        now = [min(x, few) if x > 2047 else x for x in rows]
        now[3] = -1
        lens.copy_(_index([x - 1 if fresh and x > 0 else x for x in now], dev))
        if fresh:  # the row that is there already, written again
            for s, (x, at) in enumerate(zip(now, np.cumsum([0] + rows[:-1]))):
                k1[s], v1[s] = (k[at + x - 1], v[at + x - 1]) if x > 0 else (0, 0)
            lens[[s for s, x in enumerate(now) if x == 0]] = -1
        out.fill_(9.0)
        graph.replay()
        got = out.clone()
        out.fill_(7.0)
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        got = got.double().cpu().numpy()
        for s in {0, 1, 2, 3, 4, n // 2, n - 2, n - 1}:
            a, x = sum(rows[:s]), max(now[s], 0)
            ks, vs = (h[a:a + x].double().cpu().numpy() for h in (held_k, held_v))
            o, spread, size = serving.attend(q64[s][None], ks, vs, dim ** -0.5, False)
            check_attention(got[s][None], o, spread, size, np.abs(vs).max(initial=0), x, dtype)


@pytest.mark.parametrize('causal', [True, False])
def test_rows_before_the_first_sequence(ext, hip_device, causal):
    """Starts need not begin at the first row: rows before it are neither read into a sequence nor written, by any of the ops."""
    dev, rng, at = hip_device, np.random.default_rng(8), [37, 40, 40, 140]
    q, q64 = rounded(rng, (150, 4, 64), torch.float16)
    k, k64 = rounded(rng, (150, 2, 64), torch.float16)
    v, v64 = rounded(rng, (150, 2, 64), torch.float16)
    k[:37], v[:37], k[140:], v[140:] = float('nan'), float('inf'), float('inf'), float('nan')
    cu, k, v, out = _index(at, dev), k.to(dev), v.to(dev), torch.full((150, 4, 64), 5.0, dtype=torch.float16, device=dev)
    ext.prompt_attention(q.to(dev), k, v, out, cu, cu, 0.125, causal)
    got = out.double().cpu().numpy()
    assert (got[:37] == 5.0).all() and (got[140:] == 5.0).all()
    check_prompts(got[37:140], q64[37:], k64[37:], v64[37:], [3, 0, 100], [3, 0, 100], 0.125, causal, torch.float16)
    cache, want = ext.kv_q4_cache(3, 2, 128, 64), ext.kv_q4_cache(3, 2, 128, 64)
    pos = _index([125, 0, 9], dev)
    ext.kv_q4_append(k, v, cu, pos, cache)
    ext.kv_q4_append(k[37:140], v[37:140], cu - 37, pos, want)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, want))
    back = [torch.full_like(k, 5.0) for _ in range(2)]
    ext.kv_q4_read(cache, cu, pos, *back)
    held = [torch.zeros_like(k[37:140]) for _ in range(2)]
    ext.kv_q4_read(want, cu - 37, pos, *held)
    for b, h in zip(back, held):
        assert torch.equal(b[37:140], h) and (b[:37] == 5.0).all() and (b[140:] == 5.0).all()


def test_calls_of_two_threads(ext, hip_device):
    """Two threads that call the ops at once, a stream and a workspace each: the bits of calls one after another."""
    import threading

    dev, sets = hip_device, []
    for seed in range(2):
        rng = np.random.default_rng(seed)
        q, k, v = (rounded(rng, (200, h, 64), torch.float16)[0].to(dev) for h in (4, 2, 2))
        cache = ext.kv_q4_cache(3, 2, 4128, 64)
        sets.append((q, k, v, cache, ext.decode_attention_q4_workspace(3, 4, cache), starts([100, 0, 100 - seed], dev), _index([4000, 0, 7], dev)))
    torch.cuda.synchronize()

    def run(s, turns):
        q, k, v, cache, ws, cu, pos = s
        out, one = torch.zeros_like(q), torch.zeros(3, 4, 64, dtype=torch.float16, device=dev)
        for _ in range(turns):
            ext.prompt_attention(q, k, v, out, cu, cu, 0.125)
            ext.kv_q4_append(k, v, cu, pos, cache)
            ext.decode_attention_q4(q[:3], cache, pos + 50, one, ws, 0.125)
        torch.cuda.current_stream().synchronize()
        return out, one

    want, got = [run(s, 1) for s in sets], [None, None]

    def thread(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = run(sets[i], 20)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


def test_tensors_without_rows(ext, hip_device):
    """Empty tensors of any strides: an append, a read and queries of no rows do nothing, keys of no rows give zeros."""
    dev = hip_device
    none = torch.empty(0, dtype=torch.float16, device=dev).as_strided((0, 2, 64), (1, 3, 2))
    cache, cu, pos = ext.kv_q4_cache(2, 2, 32, 64), _index([0, 0, 0], dev), _index([3, 0], dev)
    q, out = torch.ones(2, 2, 64, dtype=torch.float16, device=dev), torch.full((2, 2, 64), 5.0, dtype=torch.float16, device=dev)
    ext.kv_q4_append(none, none, cu, pos, cache)
    ext.kv_q4_read(cache, cu, pos, none, none)
    ext.prompt_attention(none, q, q, none, cu, _index([0, 1, 2], dev), 0.125)
    assert not any(t.any() for t in cache)
    ext.prompt_attention(q, none, none, out, _index([0, 1, 2], dev), cu, 0.125)
    assert not out.any()
