"""Single-token attention over a cache in pages at the limits of its types, of its plan and of what a group may hold."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def _ext():
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def _i64(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int64, device=dev)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('below', [9, 15, 20.9, 23.4, 24.6, 27.4])
@pytest.mark.parametrize('rows, members, group', [(32, 1, 1), (1000, 1, 3), (5000, 1, 2), (1504, 3, 4), (1504, 9, 8), (4096, 10, 30)])
def test_small_weights(hip_device, dtype, dim, below, rows, members, group):
    """A key of large weight and value 0 among 31 that weigh 2^-below of it, tile by tile: the output is what the small ones
    sum up to. A block a sequence, pieces, groups of up to 16, 64 and 128 columns a run."""
    dtype, page, large, value = TYPES[dtype], 32, 16.0, 4096.0
    pages, scale = -(-rows // page), below * np.log(2) / large
    k = torch.zeros(pages, 1, page, dim, dtype=dtype, device=hip_device)
    v = torch.full((pages, 1, page // 8, dim, 8), value, dtype=dtype, device=hip_device)
    k[:, :, 5, 0], v[:, :, 0, :, 5] = large, 0.0
    q = torch.zeros(members, group, dim, dtype=dtype, device=hip_device)
    q[..., 0] = 1.0
    from flash_whisper_amd.ext import KvPages

    ext, cache, out = _ext(), KvPages(k, v), torch.full_like(q, 9.0)
    table = torch.arange(pages, dtype=torch.int32, device=hip_device).expand(members, pages).contiguous()
    ws = ext.decode_attention_paged_workspace(members, group, cache, pages, 1)
    ext.decode_attention_paged(q, cache, table, _i64([rows] * members, hip_device), out, ws, scale,
                               _i64([0, members], hip_device), _i64([rows], hip_device))
    # sinks and small keys of a sequence (rows may end inside a tile, behind its sink)
    sinks = -(-rows // page)
    w = np.exp2(-below) * (rows - sinks)
    want = w * value / (sinks + w)
    # The output rounded; each weight rounded for the product and for the sum (u each, of what it adds to the output: the small
    # ones' sum is the output itself); scores of size below x ln 2 and their exponentials in fp32; fp32 sums; fp16 weights
    # below 2^-22 of the maximum are off by at most 2^-33 of it (the type's smallest step, halved, the weights 2^8 times as
    # large), and outputs there by 2^-25.
    u = torch.finfo(dtype).eps / 2
    tol = want * (3 * u + 2.0 ** -15 * below * np.log(2) + 2.0 ** -19 + rows * 2.0 ** -24) + 2.0 ** -25
    if dtype == torch.float16:
        tol += rows * 2.0 ** -33 * value / sinks
    err = np.abs(out.double().cpu().numpy() - want).max()
    assert err <= tol, f'{err:.3e} of {want:.3e}, {err / tol:.2f}'


def test_sum_of_subnormal_weights(hip_device):
    """Values of 1 and weights that fp16 holds without a leading one (2^-23 of each wave's first key): what they add to the sum of
    the weights (one instruction) and to the values (another) is the same, so the output is 1. 8 sequences, a piece each of
    2^21 rows of one page; its four waves have 2^19 keys each, which sum up to a sixteenth of the largest."""
    from flash_whisper_amd.ext import KvPages

    ext, n, heads, page, rows = _ext(), 8, 64, 256, 1 << 21
    k = torch.zeros(2, heads, page, 64, dtype=torch.float16, device=hip_device)
    k[1, :, :128:32, 0] = 16.0  # a key of each wave's first tile
    table = torch.zeros(n, rows // page, dtype=torch.int32, device=hip_device)
    table[:, 0] = 1
    q = torch.zeros(n, heads, 64, dtype=torch.float16, device=hip_device)
    q[..., 0] = 1.0
    cache, out = KvPages(k, torch.ones(2, heads, page // 8, 64, 8, dtype=torch.float16, device=hip_device)), torch.full_like(q, 9.0)
    ws = ext.decode_attention_paged_workspace(n, heads, cache, rows // page)
    ext.decode_attention_paged(q, cache, table, _i64([rows] * n, hip_device), out, ws, 23 * np.log(2) / 16)
    # per wave and lane 2^14 tiles of 4 additions each to a sum between 2^8 and 2^9, half a step of it (2^-16) each; the
    # values' sums the same; the output rounded
    assert (out.float() - 1).abs().max().item() <= 2 * 2 ** 16 * 2.0 ** -16 / 2 ** 8 + 2.0 ** -11


@pytest.mark.parametrize('groups, shared, rest, idle', [
    ([5], [1500], 0, [0]), ([5], [1500], 40, [0, 1, 3]), ([3, 40], [1300, 1411], 70, [0, 3, 4, 5]), ([2, 62], [1200, 1333], 9, [0, *range(2, 63)]),
    ([30, 40], [1300, 1280], 90, [0, 30, 31]),                                 # the plan of a launch
    ([1100, 3], [70, 64], 20, [*range(700), 1100]), ([1] * 300 + [800], [0] * 300 + [50], 20, [*range(300, 500)])])  # its arrays in memory
@pytest.mark.parametrize('group', [1, 20])
def test_idle_first(hip_device, groups, shared, rest, idle, group):
    """Idle sequences in front of a group whose tables list nothing, or pages of others: the live ones share their own."""
    from test_gpu_paged_attention import Scene, _rest

    n = sum(groups)
    if n > 100:
        group = 1 + group // 8  # (the oracle's time)
    scene = Scene(41, groups, shared, _rest(41, n, 0, rest), 16, 1, group, 64, 'bf16', spare_width=70, idle=idle)
    for entry in (-1, 2 ** 31 - 1, 0):
        scene.table[idle] = entry
        out = scene.run(hip_device)
        scene.check(out)
        assert not out[idle].any()


@pytest.mark.parametrize('where', ['behind', 'before', 'between'])
@pytest.mark.parametrize('groups, shared, rest, count', [
    ([5], [1500], 40, 5), ([5, 5], [1500, 1460], 0, 10), ([3, 20], [1280, 1411], 70, 23), ([3, 20], [1280, 1411], 70, 64),
    ([3, 20], [1280, 1411], 70, 65), ([30, 40], [1300, 1280], 90, 70), ([2, 64], [1200, 1333], 9, 3000)])
@pytest.mark.parametrize('group', [1, 9])
def test_empty_groups(hip_device, groups, shared, rest, count, where, group):
    """As many groups as sequences and more, all but a few empty: the rows of those are still read once, from the first
    sequence's table (whole pages of them are in no other table here), and the results are those without groups."""
    from test_gpu_paged_attention import Scene, _rest

    n, page = sum(groups), 16
    scene = Scene(42, groups, shared, _rest(42, n, 0, rest), page, 1, group, 64, 'fp16', spare_width=90)
    scene.check(scene.run(hip_device, groups=False))
    spare, cu, to = count - len(groups), scene.cu.tolist(), scene.shared.tolist()
    at = {'behind': len(groups), 'before': 0, 'between': 1}[where]
    scene.cu = np.array(cu[:at + 1] + [cu[at]] * spare + cu[at + 1:])
    scene.shared = np.array(to[:at] + [999] * spare + to[at:])
    scene.check(scene.run(hip_device))
    table = scene.table.copy()
    for a, b, rows in zip(cu, cu[1:], to):
        least = min(rows, *scene.lens[a:b])
        all_alike = (scene.lens[a:b] == least).all()
        scene.table[a + 1:b, :(least if all_alike else least // 32 * 32) // page] = -1
    out, scene.table = scene.run(hip_device), table
    scene.check(out)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('size', [10, 14, 18, 20, 23, 24, 24.5, 25, 25.7, 26, 26.2, 26.5, 26.8, 26.95])
@pytest.mark.parametrize('rows, members, group', [(1000, 1, 3), (5000, 1, 2), (1504, 9, 8), (4096, 10, 30)])
def test_scores_up_to_their_limit(hip_device, dtype, size, rows, members, group):
    """Scores near 2^size in size, up to 2^27, of either sign, that grow or fall by one step of fp32 from tile to tile, by fewer
    log2 units than they can be off when they are rounded: the weights of keys that do not yet move the maximum stay in the type,
    and the waves' and pieces' results are relative to what they say."""
    from flash_whisper_amd.ext import KvPages

    ext, dtype, page, dim, rng = _ext(), TYPES[dtype], 32, 64, np.random.default_rng(rows)
    tiles = -(-rows // page)
    up = np.arange(tiles) * (120 if size < 24 else 7) // tiles
    v = torch.from_numpy(rng.standard_normal((tiles, 1, page // 8, dim, 8))).to(dtype)
    v64 = v.double().numpy().transpose(0, 2, 4, 1, 3).reshape(-1, dim)[:rows]
    q = torch.zeros(members, group, dim, dtype=dtype, device=hip_device)
    q[..., 0], q[..., 1] = 1.0, 2.0 ** -8
    table = torch.arange(tiles, dtype=torch.int32, device=hip_device).expand(members, tiles).contiguous()
    for sign, step in ((1, 1), (1, -1), (-1, 1), (-1, -1)):
        k = torch.zeros(tiles, 1, page, dim, dtype=dtype, device=hip_device)
        k[..., 0], k[..., 1] = 2.0 ** 15, torch.from_numpy(step * up).to(hip_device)[:, None, None]
        scale = float(np.float32(sign * 2.0 ** (size - 15) * np.log(2)))
        cache, out = KvPages(k, v.to(hip_device)), torch.full_like(q, 9.0)
        ws = ext.decode_attention_paged_workspace(members, group, cache, tiles, 1)
        ext.decode_attention_paged(q, cache, table, _i64([rows] * members, hip_device), out, ws, scale, _i64([0, members], hip_device),
                                   _i64([rows], hip_device))
        s = scale * (step * np.repeat(up, page)[:rows] * 2.0 ** -8)  # beside what all have in common
        w = np.exp(s - s.max())
        w /= w.sum()
        # Dot products are exact here, and so is the product with scale log2(e) before the maximum is taken off; that factor is
        # off by 2^-23, of the differences alone. Beside it: output and weights rounded (u; 2 u), exponentials and sums in fp32,
        # fp16 weights below 2^-22 of the largest.
        u = torch.finfo(dtype).eps / 2
        want, spread = w @ v64, w @ np.abs(v64)
        tol = u * np.abs(want) + (2 * u + 2.0 ** -19 + 2.0 ** -23 * np.ptp(s) + rows * 2.0 ** -24) * spread \
            + rows * 2.0 ** -33 * np.abs(v64).max() + 2.0 ** -25
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= tol).all(), f'{np.nanmax(err):.3e}, {np.isnan(err).sum()} NaN, worst ratio {np.nanmax(err / tol):.2f}, {sign} {step}'
