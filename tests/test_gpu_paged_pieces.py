"""Single-token attention over a cache in pages where pieces of work are long: the ring of a wide piece at its steady state, and
table entries fetched again, 64 tiles on, in wide and narrow pieces. How long pieces are is worked out here from the same rules,
and asserted, so that a change of those does not leave the loops untested."""

import numpy as np
import pytest
import torch

from serving_tools import check_attention
from test_gpu_paged_attention import Scene, _rest

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}
TILE, COLS = 32, 16


def pieces(heads, kv_heads, cu, shared, lens, groups):
    """(columns, tiles) of the pieces of the groups of more than one sequence, and of the sequences, where tables are cut up."""
    n, group = len(lens), heads // kv_heads
    columns = -(-n // groups) * group if groups else 0
    cols = 128 if columns > 256 else 64 if groups and n * group > COLS else COLS
    want = max(1, (256 if 64 < columns <= 256 else 512) // kv_heads)
    rows, members = [0] * n, []
    for a, b, most in zip(cu, cu[1:], shared):
        live = lens[a:b]
        have = min(most, min(live)) if b - a > 1 else 0
        have = have if have == max(live, default=0) else have // TILE * TILE
        rows[a:b] = [have] * (b - a)
        members.append((have, (b - a) * group))
    runs = [(have, min(cols, c - i)) for have, c in members if have for i in range(0, c, cols)]
    own = [(max(x - r, 0), min(COLS, group - i)) for x, r in zip(lens, rows) for i in range(0, group, COLS)]
    chunk = (int(sum(x for x, _ in runs + own) * 1.0001 / want) // 128 + 1) * 128
    cut = lambda x: [-(-(-(-x // -(-x // chunk))) // TILE)] * -(-x // chunk) if x else []
    return [(c, t) for x, c in runs for t in cut(x)], [(c, t) for x, c in own for t in cut(x)]


class Long:
    """Sequences (or groups of them with one table) over a pool of pages, most of them listed many times. The pages of the tiles
    `hot` are in no other place and have the keys of the largest weight, as has page 0, which is in no table; those of `bad` are
    entries that are no page. Rows behind the last one hold NaN."""

    def __init__(self, dev, members, rows, hot, bad, page, kv_heads, group, dim, dtype):
        gen = torch.Generator(device=dev).manual_seed(7)
        self.dev, self.page, self.dim, self.kv_heads, self.members, self.rows = dev, page, dim, kv_heads, members, rows
        n, width, rng = len(members), -(-rows // page) + 1100 // page, np.random.default_rng(rows)
        table = rng.integers(1, 20, (n, width))
        hot = sorted({32 * t // page + i for t in hot for i in range(max(1, TILE // page)) if 32 * t + page * i < rows})
        pages = 20 + n * (len(hot) + 1)
        table[:, hot] = 20 + np.arange(n * len(hot)).reshape(n, -1)
        last = -(-rows // page) - 1
        if last not in hot:
            table[:, last] = pages - n + np.arange(n)
        for i, t in enumerate(bad):
            table[:, 32 * t // page] = (-1, pages, 2 ** 31 - 1)[i % 3]
        normal = lambda *shape: torch.randn(shape, generator=gen, device=dev)
        k, v = normal(pages, kv_heads, page, dim), normal(pages, kv_heads, page // 8, dim, 8)
        k[0, ..., 0] = k[20:20 + n * len(hot), ..., 0] = 4.0 * dim ** 0.5
        if rows % page:
            behind = torch.arange(page, device=dev) >= rows % page
            ends = torch.from_numpy(table[:, last]).to(dev)
            k[ends] = k[ends].masked_fill(behind[:, None], float('nan'))
            v[ends] = v[ends].masked_fill(behind.view(page // 8, 1, 8), float('nan'))
        self.k, self.v = k.to(TYPES[dtype]), v.to(TYPES[dtype])
        self.table = torch.from_numpy(np.repeat(table, members, 0).astype(np.int32)).to(dev)
        q = normal(sum(members), kv_heads * group, dim)
        q[..., 0] = 2.0
        self.q, self.scale = q.to(TYPES[dtype]), dim ** -0.5

    def run(self, groups):
        from flash_whisper_amd.ext import KvPages, load_ext

        ext, cache, out = load_ext(), KvPages(self.k, self.v), torch.full_like(self.q, 9.0)
        i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=self.dev)
        n, heads, _ = self.q.shape
        extra = (i64([0, *np.cumsum(self.members)]), i64([self.rows] * len(self.members))) if groups else ()
        ws = ext.decode_attention_paged_workspace(n, heads, cache, self.table.size(1), len(self.members) if groups else 0)
        ws.fill_(float('nan'))
        ext.decode_attention_paged(self.q, cache, self.table, i64([self.rows] * n), out, ws, self.scale, *extra)
        return out

    def check(self, out):
        """Against float64, as oracle.serving.attend defines it; the sequences of a table at once."""
        at, row = 0, torch.arange(self.rows, device=self.dev)
        for members in self.members:
            where = self.table[at].long()[row // self.page]
            mine = row[(where >= 0) & (where < len(self.k))]
            where = where[(where >= 0) & (where < len(self.k))]
            k = self.k[where, :, mine % self.page].double().permute(1, 2, 0).contiguous()
            v = self.v[where, :, mine % self.page // 8, :, mine % 8].double().transpose(0, 1).contiguous()
            q = self.q[at:at + members].double().view(members, self.kv_heads, -1, self.dim).permute(1, 0, 2, 3).flatten(1, 2)
            w = torch.softmax(q @ k * self.scale, -1)
            back = lambda x: x.view(self.kv_heads, members, -1, *x.shape[2:]).transpose(0, 1).flatten(1, 2).cpu().numpy()
            size = (q.abs() @ k.abs()).amax(-1) * self.scale
            got = out[at:at + members].double().cpu().numpy()
            check_attention(got, back(w @ v), back(w @ v.abs()), back(size), v.abs().max().item(), len(mine), self.q.dtype)
            at += members


@pytest.mark.parametrize('dtype, dim', [('fp16', 64), ('fp16', 128), ('bf16', 64), ('bf16', 128)])
@pytest.mark.parametrize('page', [16, 64])
@pytest.mark.parametrize('tiles', [3, 4, 5, 63, 64, 65, 66, 67, 129, 130])
def test_wide(hip_device, dtype, dim, page, tiles):
    """8 groups of 3 x 8 columns over 64 key/value heads: a piece of 24 columns and all rows each."""
    rows = TILE * tiles - 5
    hot = [t for t in (0, 2, 62, 63, 64, 65, 126, 127, 128, 129) if t < tiles]
    scene = Long(hip_device, [3] * 8, rows, hot, [t for t in (68, 72, 110) if t < tiles - 4], page, 64, 8, dim, dtype)
    assert pieces(512, 64, range(0, 25, 3), [rows] * 8, [rows] * 24, 8) == ([(24, tiles)] * 8, [])
    scene.check(scene.run(True))


@pytest.mark.parametrize('dtype, dim', [('fp16', 128), ('bf16', 64)])
@pytest.mark.parametrize('page', [16, 64])
@pytest.mark.parametrize('tiles', [5, 64, 66, 130])
def test_widest(hip_device, dtype, dim, page, tiles):
    """3 groups of 17 x 16 columns: runs of 128, 128 and 16, of which the last is no wide one."""
    rows = TILE * tiles - 5
    hot = [t for t in (1, 62, 63, 64, 65, 128) if t < tiles]
    scene = Long(hip_device, [17] * 3, rows, hot, [t for t in (70, 100) if t < tiles - 4], page, 64, 16, dim, dtype)
    assert pieces(1024, 64, range(0, 52, 17), [rows] * 3, [rows] * 51, 3) == ([(128, tiles), (128, tiles), (16, tiles)] * 3, [])
    scene.check(scene.run(True))


@pytest.mark.parametrize('dtype, dim', [('fp16', 64), ('fp16', 128), ('bf16', 64), ('bf16', 128)])
@pytest.mark.parametrize('page', [16, 64])
@pytest.mark.parametrize('n, tiles, group', [(8, 63, 1), (8, 64, 1), (8, 65, 5), (8, 66, 1), (8, 129, 2), (66, 65, 1), (66, 129, 1)])
def test_narrow(hip_device, dtype, dim, page, n, tiles, group):
    """A piece a sequence, `tiles` tiles for each of its four waves; the plan by waves and by a launch."""
    rows = TILE * 4 * tiles - 5
    hot = [t for t in (1, 4 * 63 + 1, 4 * 64, 4 * 64 + 3, 4 * 65 + 2, 4 * 127, 4 * 128 + 1) if t < 4 * tiles]
    scene = Long(hip_device, [1] * n, rows, hot, [t for t in (4 * 64 + 10, 4 * 66 + 1) if t < 4 * tiles - 8], page, 64, group, dim, dtype)
    assert pieces(64 * group, 64, [0], [], [rows] * n, 0) == ([], [(group, 4 * tiles)] * n)
    scene.check(scene.run(False))


@pytest.mark.parametrize('n', [63, 64, 65])
@pytest.mark.parametrize('last', [1, 2, 5, 40, 0])
def test_last_lane(hip_device, n, last):
    """As many sequences as a wave's plan takes, one fewer and one more, in groups that end with the last one: of a sequence, of
    several, of all but a few, of all (0)."""
    last = last or n
    groups = [g for g in (n - last - (n - last) // 3, (n - last) // 3, last) if g]
    shared = [[1300, 1111, 1290][i % 3] for i in range(len(groups))]
    scene = Scene(61, groups, shared, _rest(61, n, 0, 150), 16, 2, 3, 64, 'bf16', spare_width=5, idle=[n - 2] if last > 2 else [])
    scene.check(scene.run(hip_device))
    scene.check(scene.run(hip_device, groups=False))
