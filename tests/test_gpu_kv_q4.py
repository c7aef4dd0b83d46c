"""The 4-bit cache on the GPU: rows written and read back bit for bit as the oracle's, every other byte left as it is,
and the single-token attention over it against float64 (the bound of serving_tools.check_attention)."""

import numpy as np
import pytest
import torch

from oracle import serving
from serving_tools import TYPES, check_attention, check_prompts, rounded, same_bits, starts, to_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ext(hip_device):
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def _index(x, dev):
    return torch.tensor(x, dtype=torch.int64, device=dev)


# single tokens, whole blocks of 8 rows, runs that begin and end inside one; rows before the cache and past its end
@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('lengths, pos', [([1], [0]), ([1, 1, 1], [7, 8, 63]), ([8, 16, 5], [0, 8, 3]), ([20, 0, 64], [13, 5, 0]),
                                          ([9, 30], [60, -7]), ([10, 3], [64, -3]), ([0, 0, 6], [0, 1 << 40, 29]), ([2] * 70, [31] * 70)])
def test_rows_in_and_out(ext, hip_device, lengths, pos, kind, dim):
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(sum(lengths) + dim)
    n, heads, max_len, total = len(lengths), 3, 64, sum(lengths)
    k, _ = rounded(rng, (total, heads, dim), dtype)
    v, _ = rounded(rng, (total, heads, dim), dtype, 0.02)
    k[0, 0, :32], v[-1, -1, 32:64] = 0.75, 0.0  # groups of one value
    k[:, :, 5] += 8.0  # a channel that stands out
    want = serving.empty_cache(n, heads, max_len, dim, fill=0x5C)
    cache = to_device(want, dev)
    cu = starts(lengths, dev)
    ext.kv_q4_append(k.to(dev), v.to(dev), cu, _index(pos, dev), cache)
    kf, vf, at = k.float().numpy(), v.float().numpy(), 0
    k_want, v_want = np.zeros(k.shape, np.float16), np.zeros(v.shape, np.float16)
    for s, (length, p) in enumerate(zip(lengths, pos)):
        for i in range(length):
            if 0 <= p + i < max_len:
                serving.write_row(want, s, p + i, kf[at + i], vf[at + i])
                k_want[at + i], v_want[at + i] = (x[0] for x in serving.read_rows(want, s, [p + i]))
        at += length
    assert same_bits(cache, want)
    k_got, v_got = (torch.full((total + 1, heads, dim), 9.0, dtype=dtype, device=dev) for _ in range(2))
    ext.kv_q4_read(cache, cu, _index(pos, dev), k_got, v_got)
    assert torch.equal(k_got[:-1].cpu(), torch.from_numpy(k_want).to(dtype)) and torch.equal(v_got[:-1].cpu(), torch.from_numpy(v_want).to(dtype))
    assert (k_got[-1] == 9.0).all() and (v_got[-1] == 9.0).all()  # behind the last sequence
    assert same_bits(cache, want)


@pytest.mark.parametrize('kind', ['fp16', 'bf16'])
def test_extreme_rows(ext, hip_device, kind):
    """The largest and smallest values of fp16, subnormal ones, signed zeros, infinities and NaN: the oracle's bits where
    they are numbers, NaN in the groups that hold one that is not, and nowhere else."""
    dev, dtype = hip_device, TYPES[kind]
    x = torch.zeros(8, 1, 64, dtype=torch.float32)
    x[0, 0, :32] = torch.tensor([-65024.0, 65024.0]).repeat(16)
    x[1, 0, :32] = torch.arange(32) * 2.0 ** -24
    x[2, 0] = torch.tensor([0.0, -0.0]).repeat(32)
    x[3, 0, :32] = 1.0 + torch.arange(32) * 2.0 ** -7
    x[4, 0, 40], x[5, 0, 3], x[6, 0, 63] = float('inf'), float('-inf'), float('nan')
    x[7, 0] = -60000.0
    x = x.to(dtype)
    want = serving.empty_cache(1, 1, 32, 64)
    cache = to_device(want, dev)
    cu, pos = starts([8], dev), _index([3], dev)
    ext.kv_q4_append(x.to(dev), x.to(dev), cu, pos, cache)
    for i in range(8):
        serving.write_row(want, 0, 3 + i, x[i].float().numpy(), x[i].float().numpy())
    k_got, v_got = torch.empty_like(x, device=dev), torch.empty_like(x, device=dev)
    ext.kv_q4_read(cache, cu, pos, k_got, v_got)
    for got, w in zip((k_got, v_got), serving.read_rows(want, 0, range(3, 11))):
        w = torch.from_numpy(w).to(dtype)
        assert torch.equal(got.cpu().isnan(), w.isnan()) and torch.equal(got.cpu().nan_to_num(), w.nan_to_num())
        assert w.isnan().sum() == 96


def test_strided_rows(ext, hip_device):
    """k and v as slices of a packed projection, read back into slices of a wider one."""
    dev, rng = hip_device, np.random.default_rng(8)
    packed = rounded(rng, (40, 3 * 128), torch.float16)[0].to(dev)
    k, v = (packed[:, a:a + 128].unflatten(1, (2, 64)) for a in (128, 256))
    cu, pos = starts([13, 27], dev), _index([4, 0], dev)
    one, two = ext.kv_q4_cache(2, 2, 32, 64), ext.kv_q4_cache(2, 2, 32, 64)
    ext.kv_q4_append(k, v, cu, pos, one)
    ext.kv_q4_append(k.contiguous(), v.contiguous(), cu, pos, two)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    wide = torch.zeros(40, 2, 2, 72, dtype=torch.float16, device=dev)
    ext.kv_q4_read(one, cu, pos, wide[:, 0, :, :64], wide[:, 1, :, :64])
    k_got, v_got = torch.empty(40, 2, 64, dtype=torch.float16, device=dev), torch.empty(40, 2, 64, dtype=torch.float16, device=dev)
    ext.kv_q4_read(one, cu, pos, k_got, v_got)
    assert torch.equal(wide[:, 0, :, :64], k_got) and torch.equal(wide[:, 1, :, :64], v_got) and not wide[..., 64:].any()


def _filled(rng, n, heads, max_len, dim, lens, fill=0xFF):
    """A cache whose rows below lens[s] are set, the others' bytes `fill` (0xFF: NaN steps and lows)."""
    cache = serving.empty_cache(n, heads, max_len, dim, fill=fill)
    for s, length in enumerate(lens):
        if length <= 0:
            continue
        k_codes, k_meta, v_codes, v_meta = (c[s] for c in cache)
        k, v = (rng.standard_normal((length, heads, dim)).astype(np.float32) + rng.standard_normal((heads, dim)) for _ in range(2))
        step, low, c = serving.quantise(k)
        k_codes[:, :length] = (c[..., 0::2] | c[..., 1::2] << 4).transpose(1, 0, 2)
        k_meta[:, :length, :, 0], k_meta[:, :length, :, 1] = step.transpose(1, 0, 2), low.transpose(1, 0, 2)
        step, low, c = serving.quantise(v)
        t, b = np.arange(length), c[..., 0::2] | c[..., 1::2] << 4  # [t, heads, dim / 2]
        for j in range(dim // 2):
            v_codes[:, t // 8, j // 2, 2 * (t % 8) + j % 2] = b[:, :, j].T
        v_meta[:, t // 8, :, 0, t % 8], v_meta[:, t // 8, :, 1, t % 8] = step, low
    return cache


def _check_decode(got, q64, cache, lens, scale, dtype):
    for s, length in enumerate(lens):
        length = max(length, 0)
        k, v = serving.read_rows(cache, s, range(length))
        out, spread, size = serving.attend(q64[s][None], k, v, scale, False)
        check_attention(got[s][None], out, spread, size, np.abs(v.astype(np.float64)).max(initial=0), length, dtype)


# one key, around the 8, 16, 32 and 64 keys of a tile, around the 512 keys of a small cache, several tiles a wave
@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('max_len, lens', [(32, [1, 32, 0]), (96, [7, 8, 9, 15, 17, 33, 96]), (448, [225, 448, 63, 65, 0]),
                                           (512, [512, 511, 300]), (544, [544, 543, 1]), (1504, [1500, 129, 700, 0, 31]),
                                           (6016, [6000, 2, 4097])])
def test_decode(ext, hip_device, max_len, lens, kind, dim):
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(max_len + dim)
    n, heads, kv_heads = len(lens), 4, 2
    want = _filled(rng, n, kv_heads, max_len, dim, lens)
    cache = to_device(want, dev)
    q, q64 = rounded(rng, (n, heads, dim), dtype)
    out = torch.full((n, heads, dim), float('nan'), dtype=dtype, device=dev)
    ws = ext.decode_attention_q4_workspace(n, heads, cache)
    ext.decode_attention_q4(q.to(dev), cache, _index(lens, dev), out, ws, dim ** -0.5)
    _check_decode(out.double().cpu().numpy(), q64, want, lens, dim ** -0.5, dtype)
    assert same_bits(cache, want)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('heads, kv_heads', [(20, 20), (3, 1), (10, 2), (16, 1), (17, 1), (40, 1), (64, 2)])
@pytest.mark.parametrize('max_len', [224, 1216])
def test_decode_grouped_heads(ext, hip_device, max_len, heads, kv_heads, kind, dim):
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(heads)
    lens = [max_len - 1, 37]
    want = _filled(rng, 2, kv_heads, max_len, dim, lens)
    cache = to_device(want, dev)
    q, q64 = rounded(rng, (2, heads, dim), dtype)
    k, v = (rounded(rng, (2, kv_heads, dim), dtype)[0] for _ in range(2))
    out = torch.empty(2, heads, dim, dtype=dtype, device=dev)
    ws = ext.decode_attention_q4_workspace(2, heads, cache)
    ext.decode_attention_q4(q.to(dev), cache, _index(lens, dev), out, ws, dim ** -0.5, k.to(dev), v.to(dev))
    for s, length in enumerate(lens):
        serving.write_row(want, s, length, k[s].float().numpy(), v[s].float().numpy())
    assert same_bits(cache, want)
    _check_decode(out.double().cpu().numpy(), q64, want, [x + 1 for x in lens], dim ** -0.5, dtype)


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 64), ('fp16', 128), ('bf16', 128)])
@pytest.mark.parametrize('max_len, lens', [(64, [0, 7, 8, 31, 32, 63]), (64, [64, 1 << 40, -1, -(1 << 40), 5]), (640, [0, 511, 512, 639, 640, -3])])
def test_decode_fresh_row(ext, hip_device, max_len, lens, kind, dim):
    """The fresh row goes to lens[s] and is attended to; a full cache has its last row overwritten; idle sequences keep
    their cache and get zeros. Written as an append would, every other byte as it was."""
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(max_len)
    n, heads = len(lens), 2
    want = _filled(rng, n, heads, max_len, dim, [min(x, max_len) for x in lens])
    cache = to_device(want, dev)
    q, q64 = rounded(rng, (n, heads, dim), dtype)
    k, v = (rounded(rng, (n, heads, dim), dtype)[0] for _ in range(2))
    out = torch.full((n, heads, dim), float('nan'), dtype=dtype, device=dev)
    at = _index(lens, dev)
    ext.decode_attention_q4(q.to(dev), cache, at, out, ext.decode_attention_q4_workspace(n, heads, cache), dim ** -0.5,
                            k.to(dev), v.to(dev))
    rows = [min(x, max_len - 1) for x in lens]
    for s, row in enumerate(rows):
        if row >= 0:
            serving.write_row(want, s, row, k[s].float().numpy(), v[s].float().numpy())
    assert same_bits(cache, want) and at.tolist() == lens
    _check_decode(out.double().cpu().numpy(), q64, want, [r + 1 if r >= 0 else 0 for r in rows], dim ** -0.5, dtype)


def test_decode_many_sequences(ext, hip_device):
    """150 sequences of 0 to 900 rows: more than one wave's worth of lengths, work shared out over all blocks."""
    dev, rng = hip_device, np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(0, 60, 150)]
    lens[3], lens[77], lens[149] = 900, 0, 640
    want = _filled(rng, 150, 2, 928, 64, lens)
    cache = to_device(want, dev)
    q, q64 = rounded(rng, (150, 2, 64), torch.float16)
    out = torch.full((150, 2, 64), float('nan'), dtype=torch.float16, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index(lens, dev), out, ext.decode_attention_q4_workspace(150, 2, cache), 0.125)
    _check_decode(out.double().cpu().numpy(), q64, want, lens, 0.125, torch.float16)


@pytest.mark.parametrize('q_scale', [0.0, 1e-3, 30.0, 1000.0])
@pytest.mark.parametrize('kind', ['fp16', 'bf16'])
def test_decode_score_sizes(ext, hip_device, kind, q_scale):
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(9)
    want = _filled(rng, 2, 1, 1024, 64, [1000, 200])
    q, q64 = rounded(rng, (2, 4, 64), dtype, q_scale)
    cache, out = to_device(want, dev), torch.empty(2, 4, 64, dtype=dtype, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index([1000, 200], dev), out, ext.decode_attention_q4_workspace(2, 4, cache), 0.125)
    _check_decode(out.double().cpu().numpy(), q64, want, [1000, 200], 0.125, dtype)


def test_decode_views(ext, hip_device):
    """q, k_new and v_new as slices of a packed projection and out in rows of its own stride: the bits of dense ones."""
    dev, rng = hip_device, np.random.default_rng(10)
    want = _filled(rng, 3, 2, 608, 64, [600, 5, 0])
    lens = _index([600, 5, 0], dev)
    packed = rounded(rng, (3, 8 * 64), torch.float16)[0].to(dev)
    q, k, v = (packed[:, a:b].unflatten(1, (-1, 64)) for a, b in ((0, 256), (256, 384), (384, 512)))
    outs, caches = [], []
    for dense in (True, False):
        cache = to_device(want, dev)
        out = torch.zeros(3, 4, 64 if dense else 80, dtype=torch.float16, device=dev)
        args = [t.contiguous() if dense else t for t in (q, k, v)]
        ext.decode_attention_q4(args[0], cache, lens, out[..., :64], ext.decode_attention_q4_workspace(3, 4, cache), 0.125, *args[1:])
        assert not out[..., 64:].any()
        outs.append(out[..., :64].clone())
        caches.append(cache)
    assert torch.equal(*outs) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*caches))


def test_decode_refusals_on_the_device(ext, hip_device):
    dev = hip_device
    cache = ext.kv_q4_cache(2, 2, 64, 64)
    q, lens, ws = torch.zeros(2, 4, 64, dtype=torch.float16, device=dev), _index([1, 1], dev), ext.decode_attention_q4_workspace(2, 4, cache)
    out, new = torch.empty_like(q), torch.zeros(2, 2, 64, dtype=torch.float16, device=dev)
    bad = cache._replace(k_meta=cache.k_meta[:, :, :32])
    for args in ((q[:1], cache, lens, out, ws), (q, cache, lens, out[:1], ws), (q, cache, lens[:1], out, ws), (q, cache, lens.int(), out, ws),
                 (q, bad, lens, out, ws), (q, cache._replace(v_codes=cache.v_codes.cpu()), lens, out, ws), (q[:, :3], cache, lens, out[:, :3], ws),
                 (q, cache, lens, out, ws[:0]), (q, cache, lens, out, ws.double()), (q.float(), cache, lens, out, ws), (q, cache, lens, out.bfloat16(), ws)):
        with pytest.raises(RuntimeError):
            ext.decode_attention_q4(*args, 0.125)
    for fresh in ((new, None), (None, new), (new[:1], new), (new, new.bfloat16()), (new, new[:, :1])):
        with pytest.raises(RuntimeError):
            ext.decode_attention_q4(q, cache, lens, out, ws, 0.125, *fresh)
    with pytest.raises(RuntimeError, match='overlap'):
        ext.kv_q4_read(cache, starts([4, 4], dev), lens, new[:1].expand(8, -1, -1), torch.empty(8, 2, 64, dtype=torch.float16, device=dev))
    with pytest.raises(RuntimeError):
        ext.kv_q4_append(new, new[:1], starts([1, 1], dev), lens, cache)


def test_decode_streams_and_graph(ext, hip_device):
    """Two streams with a workspace each, and a captured call replayed while lens advances and eager calls with another
    workspace run between: each the bits of the eager call."""
    dev, rng = hip_device, np.random.default_rng(11)
    lens = [900, 40, 1100]
    sets = []
    for _ in range(2):
        cache = to_device(_filled(rng, 3, 2, 1216, 64, lens), dev)
        q, k, v = (rounded(rng, (3, h, 64), torch.float16)[0].to(dev) for h in (4, 2, 2))
        sets.append([q, cache, _index(lens, dev), torch.zeros_like(q), ext.decode_attention_q4_workspace(3, 4, cache), 0.125, k, v])
    want = []
    for s in sets:
        ext.decode_attention_q4(*s)
        want.append(s[3].clone())
        s[3].zero_()
    torch.cuda.synchronize()
    for s in sets:
        with torch.cuda.stream(torch.cuda.Stream()):
            ext.decode_attention_q4(*s)
    torch.cuda.synchronize()
    assert all(torch.equal(s[3], w) for s, w in zip(sets, want))
    one = sets[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.decode_attention_q4(*one)
    other_ws = ext.decode_attention_q4_workspace(3, 4, one[1])
    for turn in range(4):
        one[2].copy_(_index([x + turn for x in lens], dev))
        one[6].add_(1)
        graph.replay()
        got = one[3].clone()
        eager = list(one)
        eager[3], eager[4] = torch.zeros_like(one[3]), other_ws
        ext.decode_attention_q4(*eager)
        torch.cuda.synchronize()
        assert torch.equal(got, eager[3])


def test_far_cache_rows(ext, hip_device):
    """A sequence whose rows lie more than 2^32 bytes behind the first one's, of codes, and as many elements of steps:
    written, read and attended to."""
    dev, rng = hip_device, np.random.default_rng(13)
    n, max_len = 9, 1 << 23  # 9 x 2^23 rows x 64 bytes of codes
    cache = ext.kv_q4_cache(n, 1, max_len, 128)
    k, _ = rounded(rng, (100, 1, 128), torch.float16)
    v, _ = rounded(rng, (100, 1, 128), torch.float16)
    cu, pos = starts([0] * 8 + [100], dev), _index([0] * 8 + [max_len - 100], dev)
    ext.kv_q4_append(k.to(dev), v.to(dev), cu, pos, cache)
    k_got, v_got = torch.empty(100, 1, 128, dtype=torch.float16, device=dev), torch.empty(100, 1, 128, dtype=torch.float16, device=dev)
    ext.kv_q4_read(cache, cu, pos, k_got, v_got)
    want = serving.empty_cache(1, 1, 128, 128)
    for i in range(100):
        serving.write_row(want, 0, i, k[i].float().numpy(), v[i].float().numpy())
    kw, vw = serving.read_rows(want, 0, range(100))
    assert np.array_equal(k_got.cpu().numpy(), kw) and np.array_equal(v_got.cpu().numpy(), vw)
    ext.kv_q4_append(k.to(dev), v.to(dev), cu, _index([0] * 9, dev), cache)
    q, q64 = rounded(rng, (n, 2, 128), torch.float16)
    out = torch.full((n, 2, 128), float('nan'), dtype=torch.float16, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index([0] * 8 + [100], dev), out, ext.decode_attention_q4_workspace(n, 2, cache), 0.088)
    got = out.double().cpu().numpy()
    assert not got[:8].any()
    _check_decode(got[8:], q64[8:], want, [100], 0.088, torch.float16)


@pytest.mark.parametrize('kind, dim, heads, kv_heads', [('fp16', 64, 4, 4), ('bf16', 128, 8, 2)])
def test_prompt_then_tokens(ext, hip_device, kind, dim, heads, kv_heads):
    """The operators as a server runs them: the prompts of three clips through prompt_attention and into the cache; the
    second half of one prompt later, over the values that the cache holds for its first half; then 5 tokens each, one
    captured step replayed while lens advances on the device."""
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(14)
    scale, nq = dim ** -0.5, [30, 4, 61]
    cache, want = ext.kv_q4_cache(3, kv_heads, 96, dim), serving.empty_cache(3, kv_heads, 96, dim)
    q, q64 = rounded(rng, (95, heads, dim), dtype)
    k, k64 = rounded(rng, (95, kv_heads, dim), dtype)
    v, v64 = rounded(rng, (95, kv_heads, dim), dtype)
    out, cu, zero = torch.empty(95, heads, dim, dtype=dtype, device=dev), starts(nq, dev), _index([0, 0, 0], dev)
    ext.prompt_attention(q.to(dev), k.to(dev), v.to(dev), out, cu, cu, scale)
    check_prompts(out.double().cpu().numpy(), q64, k64, v64, nq, nq, scale, True, dtype)
    ext.kv_q4_append(k.to(dev), v.to(dev), cu, zero, cache)
    at = 0
    for s, length in enumerate(nq):
        for i in range(length):
            serving.write_row(want, s, i, k[at + i].float().numpy(), v[at + i].float().numpy())
        at += length
    assert same_bits(cache, want)
    # the last clip's prompt goes on: 20 more tokens over the 61 in the cache
    more = [rounded(rng, (20, h, dim), dtype) for h in (heads, kv_heads, kv_heads)]
    held = [torch.empty(81, kv_heads, dim, dtype=dtype, device=dev) for _ in range(2)]
    ext.kv_q4_read(cache, starts([0, 0, 61], dev), zero, held[0][:61], held[1][:61])
    for h, (t, _) in zip(held, more[1:]):
        h[61:] = t.to(dev)
    out = torch.empty(20, heads, dim, dtype=dtype, device=dev)
    ext.prompt_attention(more[0][0].to(dev), *held, out, starts([20], dev), starts([81], dev), scale)
    check_prompts(out.double().cpu().numpy(), more[0][1], *(h.double().cpu().numpy() for h in held), [20], [81], scale, True, dtype)
    ext.kv_q4_append(more[1][0].to(dev), more[2][0].to(dev), starts([0, 0, 20], dev), _index([0, 0, 61], dev), cache)
    for i in range(20):
        serving.write_row(want, 2, 61 + i, more[1][0][i].float().numpy(), more[2][0][i].float().numpy())
    lens, ws = _index([30, 4, 81], dev), ext.decode_attention_q4_workspace(3, heads, cache)
    bufs = [torch.zeros(3, h, dim, dtype=dtype, device=dev) for h in (heads, kv_heads, kv_heads)]
    out = torch.empty(3, heads, dim, dtype=dtype, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.decode_attention_q4(bufs[0], cache, lens, out, ws, scale, bufs[1], bufs[2])
        lens.add_(1)
    for token in range(5):
        new = [rounded(rng, tuple(b.shape), dtype) for b in bufs]
        for b, (t, _) in zip(bufs, new):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        now = [x + token for x in (30, 4, 81)]
        for s in range(3):
            serving.write_row(want, s, now[s], new[1][0][s].float().numpy(), new[2][0][s].float().numpy())
        assert same_bits(cache, want) and lens.tolist() == [x + 1 for x in now]
        _check_decode(out.double().cpu().numpy(), new[0][1], want, [x + 1 for x in now], scale, dtype)


@pytest.mark.parametrize('kind', ['fp16', 'bf16'])
def test_compiled_binding_and_ctypes(ext, hip_device, kind):
    """Every op through the compiled binding alone (a call that it leaves to ctypes fails here) and through ctypes alone:
    the same bits, on a stream of its own each."""
    from flash_whisper_amd.ext import WhisperExt

    assert ext._bind is not None
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(15)
    q, k, v = (rounded(rng, (40, h, 64), dtype)[0].to(dev) for h in (4, 2, 2))
    cu, pos, one = starts([7, 33], dev), _index([3, 0], dev), _index([20, 33], dev)
    results = []
    for compiled in (True, False):
        e = WhisperExt()
        if compiled:
            e._call = None
        else:
            e._bind = None
        with torch.cuda.stream(torch.cuda.Stream()):
            cache = e.kv_q4_cache(2, 2, 64, 64)
            ws = e.decode_attention_q4_workspace(2, 4, cache)
            outs = [torch.zeros_like(t) for t in (q, k, v)] + [torch.zeros(2, 4, 64, dtype=dtype, device=dev) for _ in range(2)]
            e.prompt_attention(q, k, v, outs[0], cu, cu, 0.125)
            e.prompt_attention(q, k, v, outs[0], cu, cu, 0.125, causal=False)
            e.kv_q4_append(k, v, cu, pos, cache)
            e.kv_q4_read(cache, cu, pos, outs[1], outs[2])
            e.decode_attention_q4(q[:2], cache, pos, outs[3], ws, 0.125)
            e.decode_attention_q4(q[:2], cache, one, outs[4], ws, 0.125, k[:2], v[:2])
        torch.cuda.synchronize()
        results.append(outs + list(cache))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize('n', [300, 5000])
def test_many_sequences(ext, hip_device, n):
    """More sequences than one, two or 64 rounds of looking for them: rows in and out, attention over caches of one chunk
    and of several, prompts, each against the same done in calls of at most 50 sequences."""
    dev, rng = hip_device, np.random.default_rng(n)
    lengths = rng.integers(0, 4, n)
    lengths[[3, n // 2, n - 1]] = 40, 0, 90
    total = int(lengths.sum())
    q, k, v = (rounded(rng, (total, h, 64), torch.float16)[0].to(dev) for h in (2, 1, 1))
    cu, zero = starts(lengths, dev), torch.zeros(n, dtype=torch.int64, device=dev)
    small, large = ext.kv_q4_cache(n, 1, 96, 64), ext.kv_q4_cache(n, 1, 2080, 64)
    outs = [torch.full((total, 2, 64), 7.0, dtype=torch.float16, device=dev) for _ in range(2)]
    decoded = [torch.full((n, 2, 64), 7.0, dtype=torch.float16, device=dev) for _ in range(3)]
    q1, lens = rounded(rng, (n, 2, 64), torch.float16)[0].to(dev), torch.tensor(lengths, device=dev)
    ext.prompt_attention(q, k, v, outs[0], cu, cu, 0.125)
    for out, cache in zip(decoded, (small, large)):
        ext.kv_q4_append(k, v, cu, zero, cache)
        ext.decode_attention_q4(q1, cache, lens, out, ext.decode_attention_q4_workspace(n, 2, cache), 0.125)
    back = [torch.zeros_like(k), torch.zeros_like(v)]
    ext.kv_q4_read(large, cu, zero, *back)
    for a in range(0, n, 50):
        b, at = min(a + 50, n), cu[a:a + 51] - cu[a]
        rows = slice(int(cu[a]), int(cu[b]))
        ext.prompt_attention(q[rows], k[rows], v[rows], outs[1][rows], at, at, 0.125)
        part = ext.kv_q4_cache(b - a, 1, 96, 64)
        ext.kv_q4_append(k[rows], v[rows], at, zero[a:b], part)
        assert all(torch.equal(x[a:b], y) for x, y in zip(small, part))
        held = [torch.zeros_like(k[rows]), torch.zeros_like(k[rows])]
        ext.kv_q4_read(part, at, zero[a:b], *held)
        assert all(torch.equal(x[rows], y) for x, y in zip(back, held))
        ext.decode_attention_q4(q1[a:b], part, lens[a:b], decoded[2][a:b], ext.decode_attention_q4_workspace(b - a, 2, part), 0.125)
    assert torch.equal(*outs)
    assert torch.equal(decoded[0], decoded[2]) and (decoded[1].float() - decoded[2].float()).abs().max() <= 2 ** -7


@pytest.mark.parametrize('kind, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('scale', [0.0, -0.125, 1.0])
def test_decode_scales(ext, hip_device, scale, kind, dim):
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(19)
    lens = [70, 3]
    want = _filled(rng, 2, 1, 96, dim, lens)
    q, q64 = rounded(rng, (2, 2, dim), dtype)
    cache, out = to_device(want, dev), torch.empty(2, 2, dim, dtype=dtype, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index(lens, dev), out, ext.decode_attention_q4_workspace(2, 2, cache), scale)
    _check_decode(out.double().cpu().numpy(), q64, want, lens, scale, dtype)


@pytest.mark.parametrize('max_len', [512, 4128])
def test_decode_no_numbers(ext, hip_device, max_len):
    """A query that is no number makes its own head NaN; a row of such keys every head that reads it; a value in such a
    row its dims; the other sequence stays as it is."""
    dev, rng = hip_device, np.random.default_rng(20)
    lens = [max_len - 10, 300]
    cache = to_device(_filled(rng, 2, 2, max_len, 64, lens), dev)
    q, at = rounded(rng, (2, 4, 64), torch.float16)[0].to(dev), _index(lens, dev)
    ws, want = ext.decode_attention_q4_workspace(2, 4, cache), torch.empty(2, 4, 64, dtype=torch.float16, device=dev)
    ext.decode_attention_q4(q, cache, at, want, ws, 0.125)
    bad, got = q.clone(), torch.empty_like(want)
    bad[0, 1, 5] = float('nan')
    ext.decode_attention_q4(bad, cache, at, got, ws, 0.125)
    assert got[0, 1].isnan().all()
    got[0, 1] = want[0, 1]
    assert torch.equal(got, want)
    k = torch.zeros(1, 2, 64, dtype=torch.float16, device=dev)
    v = k.clone()
    k[0, 0, 3], v[0, 1, 40] = float('inf'), float('nan')  # dims 0 .. 31 of head 0's key, 32 .. 63 of head 1's value
    ext.kv_q4_append(k, v, starts([1, 0], dev), _index([150, 0], dev), cache)
    ext.decode_attention_q4(q, cache, at, got, ws, 0.125)
    assert got[0, :2].isnan().all() and got[0, 2:, 32:].isnan().all() and got[0, 2:, :32].isfinite().all()
    assert torch.equal(got[1], want[1])


def _spread(n, high, few):
    """n lengths, most of them short, every one of `few` among them."""
    lens = [int(x) for x in np.random.default_rng(n).integers(0, high, n)]
    for i, x in enumerate(few):
        lens[(i * 37 + 5) % n] = x
    return lens


# Long caches are shared out in chunks. Few items: chunks by the lengths (one sequence, short and long; lengths at
# multiples of a chunk; two to four rounds of 64 sequences); many items: chunks of one size; more sequences than are
# looked through. The fresh row is at the end of a chunk, and the first of a new one.
@pytest.mark.parametrize('fresh', [False, True])
@pytest.mark.parametrize('kind, dim, heads, kv_heads, max_len, lens', [
    ('fp16', 64, 4, 2, 16384, [3000]), ('fp16', 128, 2, 1, 16384, [511]), ('bf16', 128, 8, 1, 16384, [16384]), ('fp16', 64, 2, 2, 131072, [40000]),
    ('bf16', 64, 17, 1, 8192, [8192, -1, 0, 512, 511, 513, 4096]), ('fp16', 64, 1, 1, 2080, _spread(70, 60, [2080, 2047, 0, 512])),
    ('fp16', 64, 2, 1, 2080, _spread(256, 20, [2080, 1024, 1023, 0, -1])), ('bf16', 64, 1, 1, 2080, _spread(270, 20, [2080, 2048, 2047, 0, -1])),
    ('fp16', 64, 20, 20, 2560, _spread(26, 60, [2560, 896, 895, 0, 1792, -1])), ('bf16', 128, 128, 32, 2560, _spread(16, 60, [2559, 896, 897, 0]))])
def test_decode_shared_out(ext, hip_device, kind, dim, heads, kv_heads, max_len, lens, fresh):
    dev, dtype, rng = hip_device, TYPES[kind], np.random.default_rng(max_len + len(lens))
    n = len(lens)
    want = _filled(rng, n, kv_heads, max_len, dim, lens)
    cache = to_device(want, dev)
    q, q64 = rounded(rng, (n, heads, dim), dtype)
    k, v = (rounded(rng, (n, kv_heads, dim), dtype)[0] for _ in range(2))
    out = torch.full((n, heads, dim), float('nan'), dtype=dtype, device=dev)
    ws = torch.full_like(ext.decode_attention_q4_workspace(n, heads, cache), float('nan'))
    ext.decode_attention_q4(q.to(dev), cache, _index(lens, dev), out, ws, dim ** -0.5, *((k.to(dev), v.to(dev)) if fresh else ()))
    rows = [min(x, max_len - 1) for x in lens]
    for s, row in enumerate(rows):
        if fresh and row >= 0:
            serving.write_row(want, s, row, k[s].float().numpy(), v[s].float().numpy())
    assert same_bits(cache, want)
    _check_decode(out.double().cpu().numpy(), q64, want, [r + 1 if r >= 0 else 0 for r in rows] if fresh else lens, dim ** -0.5, dtype)


@pytest.mark.parametrize('n, heads, kv_heads, max_len', [(8, 8, 8, 1024), (8, 8, 8, 1056), (9, 8, 8, 1056), (1, 20, 4, 2048), (1, 20, 4, 2080)])
def test_decode_sides_of_one_chunk(ext, hip_device, n, heads, kv_heads, max_len):
    """Heads of 128: caches that are one chunk, and those next to them that are shared out."""
    dev, rng = hip_device, np.random.default_rng(max_len + n)
    lens = [max_len - 3, 512, 513, 511, 0, 1024, 100, 1, 900][:n]
    want = _filled(rng, n, kv_heads, max_len, 128, lens)
    cache = to_device(want, dev)
    q, q64 = rounded(rng, (n, heads, 128), torch.float16)
    out = torch.full((n, heads, 128), float('nan'), dtype=torch.float16, device=dev)
    ext.decode_attention_q4(q.to(dev), cache, _index(lens, dev), out, ext.decode_attention_q4_workspace(n, heads, cache), 128 ** -0.5)
    _check_decode(out.double().cpu().numpy(), q64, want, lens, 128 ** -0.5, torch.float16)
