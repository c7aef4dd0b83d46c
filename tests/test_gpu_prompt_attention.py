"""prompt_attention on the GPU against the float64 oracle, at the lengths, masks, strides and values where it can go
wrong. The bound on every element is serving_tools.check_attention's."""

import numpy as np
import pytest
import torch

from serving_tools import TYPES, check_prompts, rounded, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ext(hip_device):
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def _run(ext, dev, nq, nk, heads, kv_heads, dim, kind, causal, seed=0, q_scale=1.0, edit=None):
    dtype, rng = TYPES[kind], np.random.default_rng(seed)
    q, q64 = rounded(rng, (sum(nq), heads, dim), dtype, q_scale)
    k, k64 = rounded(rng, (sum(nk), kv_heads, dim), dtype)
    v, v64 = rounded(rng, (sum(nk), kv_heads, dim), dtype)
    if edit:
        edit(k, v)
        k64, v64 = k.double().numpy(), v.double().numpy()
    out = torch.full((sum(nq), heads, dim), float('nan'), dtype=dtype, device=dev)
    ext.prompt_attention(q.to(dev), k.to(dev), v.to(dev), out, starts(nq, dev), starts(nk, dev), dim ** -0.5, causal)
    check_prompts(out.double().cpu().numpy(), q64, k64, v64, nq, nk, dim ** -0.5, causal, dtype)


# one token, the prompt's 4, a query more and less than the tiles of 16 to 256 rows, keys likewise
@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('n', [1, 2, 4, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 400])
def test_square(ext, hip_device, n, causal, kind, dim):
    _run(ext, hip_device, [n], [n], 2, 2, dim, kind, causal, seed=n)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('heads, kv_heads', [(20, 20), (8, 1), (10, 2), (12, 4), (3, 1), (48, 1)])
def test_grouped_heads(ext, hip_device, heads, kv_heads, kind, dim):
    _run(ext, hip_device, [70, 3], [70, 3], heads, kv_heads, dim, kind, True, seed=heads)


# keys longer than the queries (a prompt that goes on), queries longer than the keys (rows that see nothing), no
# keys, no queries, empty sequences first, last and between
@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('nq, nk', [([5, 100, 1, 64], [300, 164, 1000, 65]), ([100, 40, 200], [37, 1, 130]), ([3, 70, 9], [0, 200, 0]),
                                    ([0, 5, 0, 0, 130, 0], [0, 7, 9, 0, 130, 100]), ([1] * 70, list(range(70))),
                                    ([1, 200, 3] * 30, [150, 200, 3] * 30)])
def test_ragged(ext, hip_device, nq, nk, causal, kind, dim):
    _run(ext, hip_device, nq, nk, 4, 2, dim, kind, causal, seed=len(nq))


@pytest.mark.parametrize('kind, dim, nq, nk', [('fp16', 64, 1100, 1500), ('bf16', 128, 1025, 1025), ('fp16', 128, 3, 5000)])
def test_long(ext, hip_device, kind, dim, nq, nk):
    _run(ext, hip_device, [nq], [nk], 4, 2, dim, kind, True, seed=7)


@pytest.mark.parametrize('q_scale', [0.0, 1e-3, 30.0, 300.0])
def test_score_sizes(ext, hip_device, q_scale):
    """All scores equal, nearly equal, and so large that a key or two take all the weight; the maximum rises along
    the keys for some rows."""
    _run(ext, hip_device, [150, 33], [400, 33], 2, 2, 64, 'fp16', True, seed=3, q_scale=q_scale)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('at', [0, 5, 63, 64, 90, 129])
def test_values_not_seen(ext, hip_device, at, kind, dim):
    """Infinities and NaN in keys and values reach only the queries that see them: causal rows before them, and
    the other sequence's, stay what they are."""
    def edit(k, v):
        k[at, 0, 3] = float('nan')
        v[at, 1, 5], v[at, 1, 6], v[at, 1, 7] = float('inf'), float('-inf'), float('nan')
        v[at + 1, 1, 5] = float('inf')

    _run(ext, hip_device, [130, 40], [131, 40], 2, 2, dim, kind, True, seed=at, edit=edit)


def test_values_past_the_sequences(ext, hip_device):
    """NaN in rows of k and v behind the last sequence, and rows of out there, are left alone."""
    dev, rng = hip_device, np.random.default_rng(1)
    q, q64 = rounded(rng, (90, 2, 64), torch.float16)
    k, k64 = rounded(rng, (120, 2, 64), torch.float16)
    v, v64 = rounded(rng, (120, 2, 64), torch.float16)
    k[77:], v[77:] = float('nan'), float('inf')
    for causal in (True, False):
        out = torch.full((90, 2, 64), 5.0, dtype=torch.float16, device=dev)
        ext.prompt_attention(q.to(dev), k.to(dev), v.to(dev), out, starts([30, 41], dev), starts([36, 41], dev), 0.125, causal)
        got = out.double().cpu().numpy()
        assert (got[71:] == 5.0).all()
        check_prompts(got[:71], q64, k64, v64, [30, 41], [36, 41], 0.125, causal, torch.float16)


def test_starts_out_of_range(ext, hip_device):
    """Starts outside the rows are clamped to them: no access leaves the tensors, the sequences that are whole are right."""
    dev, rng = hip_device, np.random.default_rng(2)
    q, q64 = rounded(rng, (50, 2, 64), torch.float16)
    cu = torch.tensor([-9, 20, 1 << 40], dtype=torch.int64, device=dev)
    out = torch.full((50, 2, 64), float('nan'), dtype=torch.float16, device=dev)
    x = q.to(dev)
    ext.prompt_attention(x, x, x, out, cu, cu, 0.125)
    check_prompts(out.double().cpu().numpy(), q64, q64, q64, [20, 30], [20, 30], 0.125, True, torch.float16)
    out.fill_(3.0)
    falling = torch.tensor([40, 10, 5], dtype=torch.int64, device=dev)  # no sequence has a row
    ext.prompt_attention(x, x, x, out, falling, falling, 0.125)
    assert (out == 3.0).all()


@pytest.mark.parametrize('kind', ['fp16', 'bf16'])
def test_strided_views(ext, hip_device, kind):
    """q, k and v as slices of one packed projection, out head-major: the same bits as from dense copies."""
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(4)
    nq = [100, 37, 1]
    packed = rounded(rng, (sum(nq), (4 + 2 + 2) * 64), dtype)[0].to(dev)
    q, k, v = (packed[:, a:b].unflatten(1, (-1, 64)) for a, b in ((0, 256), (256, 384), (384, 512)))
    cu = starts(nq, dev)
    dense = torch.empty(sum(nq), 4, 64, dtype=dtype, device=dev)
    ext.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), dense, cu, cu, 0.125)
    by_head = torch.empty(4, sum(nq), 64, dtype=dtype, device=dev).transpose(0, 1)
    ext.prompt_attention(q, k, v, by_head, cu, cu, 0.125)
    assert torch.equal(by_head, dense)
    wide = torch.zeros(sum(nq), 4, 72, dtype=dtype, device=dev)
    ext.prompt_attention(q, k, v, wide[..., :64], cu, cu, 0.125)
    assert torch.equal(wide[..., :64], dense) and not wide[..., 64:].any()
    broadcast = k[:, :1].expand(-1, 2, -1)  # one stored head read as two
    ext.prompt_attention(q, broadcast, v, by_head, cu, cu, 0.125)
    ext.prompt_attention(q, broadcast.contiguous(), v, dense, cu, cu, 0.125)
    assert torch.equal(by_head, dense)


def test_refusals_on_the_device(ext, hip_device):
    dev = hip_device
    q = torch.zeros(8, 4, 64, dtype=torch.float16, device=dev)
    k, cu = q[:, :2].contiguous(), starts([8], dev)
    out = torch.empty_like(q)
    for args in ((q, k, k[:7], out, cu, cu), (q, k, k, out[:7], cu, cu), (q, k, k.bfloat16(), out, cu, cu),
                 (q, k[:, :, ::2], k, out, cu, cu), (q, k, k, out[:1].expand(8, -1, -1), cu, cu), (q, q[:, :3], q[:, :3], out, cu, cu),
                 (q, k, k, out, cu.int(), cu), (q, k, k, out, cu, cu[:1]), (q, k, k, out, cu.cpu(), cu),
                 (q.flatten()[4:4 + 7 * 256].view(7, 4, 64), k, k, out[:7], cu, cu)):
        with pytest.raises(RuntimeError):
            ext.prompt_attention(*args, 0.125)


def test_streams_and_graph(ext, hip_device):
    """Two calls at once on two streams, and a captured call replayed with changed inputs and lengths: each the bits
    of an eager call."""
    dev, rng = hip_device, np.random.default_rng(5)
    sets = []
    for nq in ([300, 5], [40, 265]):
        q, k, v = (rounded(rng, (305, 4, 64), torch.float16)[0].to(dev) for _ in range(3))
        sets.append([q, k, v, torch.zeros_like(q), starts(nq, dev), starts(nq, dev)])
    want = []
    for s in sets:
        ext.prompt_attention(*s, 0.125)
        want.append(s[3].clone())
        s[3].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for stream, s in zip(streams, sets):
        with torch.cuda.stream(stream):
            ext.prompt_attention(*s, 0.125)
    torch.cuda.synchronize()
    assert all(torch.equal(s[3], w) for s, w in zip(sets, want))
    bufs = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.prompt_attention(*bufs, 0.125)
    for turn in (0, 1, 0, 1):
        for b, t in zip(bufs, sets[turn]):
            b.copy_(t)
        bufs[3].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bufs[3], want[turn])


def test_far_rows(ext, hip_device):
    """Rows more than 2^31 elements behind the first, of every tensor."""
    dev, rng = hip_device, np.random.default_rng(6)
    stride = (1 << 31) // 96 // 8 * 8 + 64  # 100 rows of this stride pass 2^31 elements
    big = torch.empty(99 * stride + 4 * 64 * 4, dtype=torch.float16, device=dev)
    view = lambda at: big.as_strided((100, 4, 64), (stride, 64, 1), at)
    q, k, v, out = (view(256 * i) for i in range(4))
    h = [rounded(rng, (100, 4, 64), torch.float16) for _ in range(3)]
    for t, (x, _) in zip((q, k, v), h):
        t.copy_(x)
    ext.prompt_attention(q, k, v, out, starts([60, 40], dev), starts([60, 40], dev), 0.125)
    check_prompts(out.double().cpu().numpy(), *(x for _, x in h), [60, 40], [60, 40], 0.125, True, torch.float16)


# every way of sharing out the rows, by the sizes that choose it: 128-row blocks, 64 rows and two parts of 64 or 32
# keys, 32 rows and 8 parts, single waves; partial blocks and tiles in each
FORMS = {'wide': ([500, 33, 700, 129], [500, 160, 700, 130], 40, 20), 'wide_long': ([1030, 40], [1500, 2100], 40, 20),
         'two_parts': ([300, 70], [900, 601], 20, 20), 'two_short_parts': ([150, 33, 90], [150, 70, 210], 20, 20),
         'eight_parts': ([4, 37, 1], [1000, 531, 777], 8, 2), 'single_waves': ([33, 8, 64, 1], [40, 20, 64, 64], 8, 4)}


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('form', FORMS)
def test_forms(ext, hip_device, form, causal, kind, dim):
    nq, nk, heads, kv_heads = FORMS[form]
    _run(ext, hip_device, nq, nk, heads, kv_heads, dim, kind, causal, seed=dim)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('form', FORMS)
def test_forms_values_not_seen(ext, hip_device, form, kind, dim):
    """Infinities and NaN in the keys and values near each sequence's end: seen by its last queries, not by the others."""
    nq, nk, heads, kv_heads = FORMS[form]

    def edit(k, v):
        for end in np.cumsum(nk):
            k[end - 2, 0, 9] = float('inf')
            v[end - 1, -1, 3], v[end - 3, -1, 4], v[end - 2, -1, dim - 1] = float('nan'), float('inf'), float('-inf')
            v[end - 17, -1, 5] = float('inf')

    _run(ext, hip_device, nq, nk, heads, kv_heads, dim, kind, True, seed=dim, edit=edit)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('scale', [0.0, -0.125, 1.0, -1e-3])
def test_scales(ext, hip_device, scale, kind, dim):
    """A scale of zero weighs all keys alike, a negative one turns the order of the scores round."""
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(17)
    q, q64 = rounded(rng, (90, 2, dim), dtype)
    k, k64 = rounded(rng, (90, 2, dim), dtype)
    v, v64 = rounded(rng, (90, 2, dim), dtype)
    out, cu = torch.empty(90, 2, dim, dtype=dtype, device=dev), starts([50, 40], dev)
    ext.prompt_attention(q.to(dev), k.to(dev), v.to(dev), out, cu, cu, scale)
    check_prompts(out.double().cpu().numpy(), q64, k64, v64, [50, 40], [50, 40], scale, True, dtype)


def test_no_rows(ext, hip_device):
    """No queries: nothing happens; no keys at all: zeros."""
    dev = hip_device
    q, none = torch.ones(6, 2, 64, dtype=torch.float16, device=dev), torch.empty(0, 2, 64, dtype=torch.float16, device=dev)
    out, cu, cu0 = torch.ones_like(q), starts([2, 4], dev), starts([0, 0], dev)
    ext.prompt_attention(none, q, q, none.clone(), cu0, cu, 0.125)
    for causal in (True, False):
        ext.prompt_attention(q, none, none, out.fill_(1), cu, cu0, 0.125, causal)
        assert not out.any()


@pytest.mark.parametrize('value', [float('nan'), float('inf')])
def test_queries_that_are_no_numbers(ext, hip_device, value):
    """They make their own row and head NaN, and no other."""
    dev, rng = hip_device, np.random.default_rng(18)
    q, k, v = (rounded(rng, (70, 2, 64), torch.float16)[0].to(dev) for _ in range(3))
    cu, want = starts([70], dev), torch.empty(70, 2, 64, dtype=torch.float16, device=dev)
    ext.prompt_attention(q, k, v, want, cu, cu, 0.125)
    q[33, 1, 7] = value
    got = torch.empty_like(want)
    ext.prompt_attention(q, k, v, got, cu, cu, 0.125)
    assert got[33, 1].isnan().all()
    got[33, 1] = want[33, 1]
    assert torch.equal(got, want)


def test_starts_that_fall_and_rise(ext, hip_device):
    """Starts must ascend; where they do not, no access leaves the rows: the ones around them stay as they were."""
    dev = hip_device
    x = torch.randn(1000, 2, 64, generator=torch.Generator().manual_seed(3)).half().to(dev)
    for cu in ([300, 0, 50, 400], [390, 399, 10, 20], [200, 0, 0, 0]):
        starts_of = torch.tensor(cu, dtype=torch.int64, device=dev)
        for causal in (True, False):
            out = torch.full_like(x, 3.0)
            ext.prompt_attention(x[300:700], x[300:700], x[300:700], out[300:700], starts_of, starts_of, 0.125, causal)
            assert (out[:300] == 3.0).all() and (out[700:] == 3.0).all() and not out.isnan().any()


# sizes on either side of where one way of sharing out the rows takes over from another
SIDES = {'full_blocks': ([700, 33, 900], [700, 160, 900], 40, 20), 'few_full_blocks': ([640, 129], [700, 130], 40, 20),
         'one_tile': ([32, 8, 2, 1], [32, 20, 4, 7], 8, 4), 'past_one_tile': ([33, 8, 64, 1], [33, 31, 64, 4], 8, 4),
         'keys_383': ([383], [383], 8, 8), 'keys_384': ([384], [384], 8, 8), 'keys_511': ([40], [511], 8, 4), 'keys_512': ([40], [512], 8, 4),
         'eight_parts_full': ([200, 31], [600, 600], 26, 26), 'past_eight_parts': ([225, 31], [600, 600], 26, 26)}


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('sides', SIDES)
def test_sides_of_forms(ext, hip_device, sides, causal, kind, dim):
    nq, nk, heads, kv_heads = SIDES[sides]
    _run(ext, hip_device, nq, nk, heads, kv_heads, dim, kind, causal, seed=dim + 1)
