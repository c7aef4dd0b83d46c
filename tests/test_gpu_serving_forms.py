"""Every way in which the prompt attention shares out its rows, named by the library for the sizes at hand, and the decode
over caches that are cut into chunks: against the float64 oracle, within the bound of serving_tools.check_attention."""

import numpy as np
import pytest
import torch

from flash_whisper_amd import _lib
from oracle import serving
from serving_tools import TYPES, check_attention, check_prompts, rounded, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ext(hip_device):
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def _index(x, dev):
    return torch.tensor(x, dtype=torch.int64, device=dev)


# form: the queries and keys of the sequences, heads and key/value heads. Partial blocks and tiles in each; single waves with
# sequences of many tiles among the short ones; blocks of 128 rows over more than 1500 keys and over few
FORMS = {'waves': (_lib.PROMPT_WAVES, [150] + [1] * 20, [200] + [3] * 20, 8, 4), 'waves_last': (_lib.PROMPT_WAVES, [1, 0, 2] * 9 + [333], [1, 5, 0] * 9 + [333], 6, 2),
         'long_wide': (_lib.PROMPT_128_ROWS, [1300, 1201], [1500, 2100], 40, 20), 'short_wide': (_lib.PROMPT_128_ROWS, [60, 1, 133] * 22, [100, 1, 140] * 22, 40, 20),
         'two_parts': (_lib.PROMPT_2_PARTS, [300, 70], [900, 601], 20, 20), 'two_short_parts': (_lib.PROMPT_2_SHORT_PARTS, [150, 33, 90], [150, 70, 210], 20, 20),
         'eight_parts': (_lib.PROMPT_8_PARTS, [4, 37, 1], [1000, 531, 777], 8, 2)}


def _form(ext, nq, nk, heads, kv_heads, dim, causal):
    return ext.lib.fw_prompt_attention_form(len(nq), sum(nq), sum(nk), heads, kv_heads, dim, causal)


def _check_some(ext, dev, form, dim, kind, causal, edit=None):
    """The call of a form; the query heads of the first and the last key/value head are compared."""
    want, nq, nk, heads, kv_heads = FORMS[form]
    assert _form(ext, nq, nk, heads, kv_heads, dim, causal) == want
    dtype, rng, group = TYPES[kind], np.random.default_rng(dim + causal), heads // kv_heads
    q, q64 = rounded(rng, (sum(nq), heads, dim), dtype)
    k, k64 = rounded(rng, (sum(nk), kv_heads, dim), dtype)
    v, v64 = rounded(rng, (sum(nk), kv_heads, dim), dtype)
    if edit:
        edit(k, v, nk)
        k64, v64 = k.double().numpy(), v.double().numpy()
    out = torch.full((sum(nq), heads, dim), float('nan'), dtype=dtype, device=dev)
    ext.prompt_attention(q.to(dev), k.to(dev), v.to(dev), out, starts(nq, dev), starts(nk, dev), dim ** -0.5, causal)
    got = out.double().cpu().numpy()
    assert edit or not np.isnan(got).any()
    for h in (0, kv_heads - 1):
        own = slice(h * group, (h + 1) * group)
        check_prompts(got[:, own], q64[:, own], k64[:, h:h + 1], v64[:, h:h + 1], nq, nk, dim ** -0.5, causal, dtype)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('form', FORMS)
def test_prompt_forms(ext, hip_device, form, causal, kind, dim):
    _check_some(ext, hip_device, form, dim, kind, causal)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('form', FORMS)
def test_prompt_forms_no_numbers(ext, hip_device, form, causal, kind, dim):
    """Infinities and NaN near the end of each sequence, whose last causal queries alone see them, and in its middle."""
    def edit(k, v, nk):
        for end, n in zip(np.cumsum(nk), nk):
            if n > 20:
                k[end - 2, 0, 9] = float('inf')
                v[end - 1, -1, 3], v[end - 3, -1, 4], v[end - 2, -1, dim - 1] = float('nan'), float('inf'), float('-inf')
                v[end - 17, -1, 5], v[end - n // 2, -1, 7] = float('inf'), float('nan')

    _check_some(ext, hip_device, form, dim, kind, causal, edit)


def _rows_in_cache(ext, dev, rng, lens, heads, max_len, dim, spread=1.0):
    """A cache with random rows, and what it holds of them, float64 [rows, heads, dim]."""
    cache = ext.kv_q4_cache(len(lens), heads, max_len, dim)
    k, v = (rounded(rng, (sum(lens), heads, dim), torch.float16, spread)[0].to(dev) for _ in range(2))
    cu, zero = starts(lens, dev), _index([0] * len(lens), dev)
    ext.kv_q4_append(k, v, cu, zero, cache)
    ext.kv_q4_read(cache, cu, zero, k, v)
    return cache, k.double().cpu().numpy(), v.double().cpu().numpy()


def _chunked_workspace(ext, n, heads, cache):
    ws = ext.decode_attention_q4_workspace(n, heads, cache)
    assert ws.numel() > 4  # else the cache is one chunk
    return ws.fill_(float('nan'))


def _check_rows(got, q64, k, v, held, lens, scale, dtype):
    """Sequence s over the first lens[s] of its held[s] rows."""
    for s, n in enumerate(lens):
        at, n = sum(held[:s]), max(n, 0)
        ks, vs = k[at:at + n], v[at:at + n]
        out, spread, size = serving.attend(q64[s][None], ks, vs, scale, False)
        check_attention(got[s][None], out, spread, size, np.abs(vs).max(initial=0), n, dtype)


@pytest.mark.parametrize('dim, heads, kv_heads, max_len', [(64, 4, 2, 4128), (128, 8, 2, 16384), (64, 20, 20, 16384)])
def test_chunked_decode_streams_and_graph(ext, hip_device, dim, heads, kv_heads, max_len):
    """Two streams with a workspace each, and two captured calls, also with one each, replayed in turn with lengths that go from
    one chunk to several and back, with eager calls of a third workspace between: the eager call's bits, and the oracle's values."""
    dev, rng, held = hip_device, np.random.default_rng(max_len), [4000, 64, 3900, 0]
    n, dtype, scale = len(held), torch.float16, dim ** -0.5
    cache, k, v = _rows_in_cache(ext, dev, rng, held, kv_heads, max_len, dim)
    qs = [rounded(rng, (n, heads, dim), dtype) for _ in range(2)]
    q = [x[0].to(dev) for x in qs]
    lens = _index(held, dev)
    want, eager_ws = [], _chunked_workspace(ext, n, heads, cache)
    for x in q:
        want.append(torch.empty_like(x))
        ext.decode_attention_q4(x, cache, lens, want[-1], eager_ws, scale)
    torch.cuda.synchronize()
    wss, outs = [_chunked_workspace(ext, n, heads, cache) for _ in q], [torch.zeros_like(x) for x in q]
    torch.cuda.synchronize()
    for x, out, ws in zip(q, outs, wss):
        with torch.cuda.stream(torch.cuda.Stream()):
            ext.decode_attention_q4(x, cache, lens, out, ws, scale)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for x, out, ws in zip(q, outs, wss):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ext.decode_attention_q4(x, cache, lens, out, ws, scale)
    for now in ([400, 64, 31, 0], [600, 0, 512, -1], [4000, 64, 3900, 0], [0, -1, 1, 0], [3871, 1, 2048, -5]):
        lens.copy_(_index(now, dev))
        for out in outs:
            out.fill_(9.0)
        for graph in graphs:
            graph.replay()
        for x, x64, out, w in zip(q, (y for _, y in qs), outs, want):
            ext.decode_attention_q4(x, cache, lens, w, eager_ws, scale)
            torch.cuda.synchronize()
            assert torch.equal(out, w)
            _check_rows(out.double().cpu().numpy(), x64, k, v, held, now, scale, dtype)


@pytest.mark.parametrize('q_scale', [0.0, 1e-3, 30.0, 1000.0])
@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('bf16', 128)])
def test_chunked_decode_score_sizes(ext, hip_device, kind, dim, q_scale):
    """All scores equal, nearly equal, and so large that one key in one chunk takes all the weight."""
    dev, dtype, rng, held = hip_device, TYPES[kind], np.random.default_rng(9), [4000, 3, 2500]
    cache, k, v = _rows_in_cache(ext, dev, rng, held, 1, 4128, dim)
    q, q64 = rounded(rng, (3, 4, dim), dtype, q_scale)
    out = torch.full((3, 4, dim), float('nan'), dtype=dtype, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index(held, dev), out, _chunked_workspace(ext, 3, 4, cache), dim ** -0.5)
    _check_rows(out.double().cpu().numpy(), q64, k, v, held, held, dim ** -0.5, dtype)


def test_chunked_decode_many_sequences(ext, hip_device):
    """150 sequences of 0 to 4000 rows in chunked caches: three rounds of lengths."""
    dev, rng = hip_device, np.random.default_rng(12)
    held = [int(x) for x in rng.integers(0, 60, 150)]
    held[3], held[77], held[128], held[149] = 4000, 0, 2100, 640
    cache, k, v = _rows_in_cache(ext, dev, rng, held, 2, 4128, 64)
    q, q64 = rounded(rng, (150, 2, 64), torch.float16)
    out = torch.full((150, 2, 64), float('nan'), dtype=torch.float16, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index(held, dev), out, _chunked_workspace(ext, 150, 2, cache), 0.125)
    _check_rows(out.double().cpu().numpy(), q64, k, v, held, held, 0.125, torch.float16)


def test_chunked_decode_views(ext, hip_device):
    """q, k_new and v_new as slices of a packed projection and out in rows of its own stride: the bits of dense ones."""
    dev, rng, held = hip_device, np.random.default_rng(10), [4000, 5, 0]
    packed = rounded(rng, (3, 8 * 64), torch.float16)[0].to(dev)
    q, k, v = (packed[:, a:b].unflatten(1, (-1, 64)) for a, b in ((0, 256), (256, 384), (384, 512)))
    outs, caches = [], []
    for dense in (True, False):
        cache = _rows_in_cache(ext, dev, np.random.default_rng(1), held, 2, 4128, 64)[0]
        out = torch.zeros(3, 4, 64 if dense else 80, dtype=torch.float16, device=dev)
        args = [t.contiguous() if dense else t for t in (q, k, v)]
        ext.decode_attention_q4(args[0], cache, _index(held, dev), out[..., :64], _chunked_workspace(ext, 3, 4, cache), 0.125, *args[1:])
        assert not out[..., 64:].any()
        outs.append(out[..., :64].clone())
        caches.append(cache)
    assert torch.equal(*outs) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*caches))
