"""Single-token attention over a cache in pages, with and without groups that share rows, against the float64 oracle."""

import numpy as np
import pytest
import torch

from oracle import pages as oracle
from serving_tools import check_attention, rounded

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def _ext():
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def _rest(seed, n, low, high):
    return [int(x) for x in np.random.default_rng(seed).integers(low, high + 1, n)]


class Scene:
    """Groups of sequences whose first rows are the same pages; the rest of each is its own, the page in which the shared
    rows end copied. Rows behind a sequence's length and spare pages hold NaN."""

    def __init__(self, seed, groups, shared, rest, page, kv_heads, group, dim, dtype, spare_width=2, idle=()):
        rng = np.random.default_rng(seed)
        self.dtype, self.page, self.kv_heads, self.dim, self.heads = TYPES[dtype], page, kv_heads, dim, kv_heads * group
        lens, tables, copies, at = [], [], [], 0
        for g, members in enumerate(groups):
            whole = shared[g] // page
            base = list(range(at, at + whole))
            at += whole
            for m in range(members):
                n = shared[g] + rest[len(lens)]
                more = -(-n // page) - whole
                if shared[g] % page and m:
                    copies.append((tables[len(lens) - m][whole], at))
                tables.append(base + list(range(at, at + max(more, 1))))
                lens.append(n)
                at += max(more, 1)
        width = max(len(t) for t in tables) + spare_width
        order = rng.permutation(at)
        self.table = np.full((len(lens), width), -1, np.int32)
        for s, t in enumerate(tables):
            self.table[s, :len(t)] = order[t]
        level = rng.standard_normal((2, kv_heads, dim))
        self.k, k64 = rounded(rng, (at, kv_heads, page, dim), self.dtype)
        self.v, v64 = rounded(rng, (at, kv_heads, page // 8, dim, 8), self.dtype)
        self.k = (self.k + torch.from_numpy(level[0])[None, :, None]).to(self.dtype)
        self.v = (self.v + torch.from_numpy(level[1])[None, :, None, :, None]).to(self.dtype)
        for a, b in copies:
            self.k[order[b]], self.v[order[b]] = self.k[order[a]].clone(), self.v[order[a]].clone()
        # what no sequence sees
        seen = np.zeros((at, page), bool)
        for s, n in enumerate(lens):
            rows = np.arange(n)
            seen[self.table[s, rows // page], rows % page] = True
        hidden = torch.from_numpy(~seen)
        self.k.masked_fill_(hidden[:, None, :, None], float('nan'))
        self.v.masked_fill_(hidden.view(at, 1, page // 8, 1, 8), float('nan'))
        self.q, self.q64 = rounded(rng, (len(lens), self.heads, dim), self.dtype)
        self.lens = np.array(lens)
        for s in idle:
            self.lens[s] = -1
        self.cu, self.shared = np.r_[0, np.cumsum(groups)], np.array(shared)

    def run(self, dev, groups=True, scale=None, q=None, out=None, ws=None, capture=False):
        from flash_whisper_amd.ext import KvPages

        ext, n = _ext(), len(self.lens)
        cache = KvPages(self.k.to(dev), self.v.to(dev))
        q = self.q.to(dev) if q is None else q
        out = torch.full_like(q, 9.0) if out is None else out
        i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=dev)
        table = torch.from_numpy(self.table).to(dev)
        ws = ext.decode_attention_paged_workspace(n, self.heads, cache, self.table.shape[1], len(self.shared) if groups else 0) if ws is None else ws
        ws.fill_(float('nan'))
        extra = (i64(self.cu), i64(self.shared)) if groups else ()
        ext.decode_attention_paged(q, cache, table, i64(self.lens), out, ws, self.dim ** -0.5 if scale is None else scale, *extra)
        return out

    def check(self, out, scale=None):
        got = out.double().cpu().numpy()
        k, v = self.k.double().numpy(), self.v.double().numpy()
        scale = self.dim ** -0.5 if scale is None else scale
        for s, (want, spread, size, keys, vmax) in enumerate(oracle.attend(self.q64, k, v, self.table, self.lens, scale)):
            check_attention(got[s][None], want, spread, size, vmax, keys, self.dtype)
            if keys == 0:
                assert not got[s].any()


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('page', [16, 32, 128])
@pytest.mark.parametrize('kv_heads, group, lens', [
    (3, 1, [1]), (2, 1, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 200]), (1, 5, [100, 3]), (2, 16, [77, 300]), (1, 20, [5, 400]),
    (1, 48, [33])])
def test_alone(hip_device, dtype, dim, page, kv_heads, group, lens):
    """Short tables: a block a sequence, no groups."""
    scene = Scene(7, [1] * len(lens), [0] * len(lens), lens, page, kv_heads, group, dim, dtype)
    scene.check(scene.run(hip_device, groups=False))


@pytest.mark.parametrize('dtype, dim', [('fp16', 64), ('bf16', 128)])
@pytest.mark.parametrize('page', [16, 32, 64, 256])
@pytest.mark.parametrize('kv_heads, group, lens', [
    (1, 1, [5000]), (2, 4, [0, 1, 31, 32, 33, 1100, 4097, 127, 128, 129]), (1, 20, [3000, 7]), (1, 35, [1500])])
def test_alone_long(hip_device, dtype, dim, page, kv_heads, group, lens):
    """Long tables, cut into pieces by the lengths there are."""
    scene = Scene(8, [1] * len(lens), [0] * len(lens), lens, page, kv_heads, group, dim, dtype, spare_width=1100 // page + 1)
    scene.check(scene.run(hip_device, groups=False))


@pytest.mark.parametrize('dtype, dim', [('fp16', 128), ('bf16', 64)])
@pytest.mark.parametrize('n, most, width', [(70, 1900, 2048), (70, 1900, 2064), (40, 900, 1024), (6, 700, 768), (6, 740, 784), (6, 1000, 1024)])
def test_alone_sides_of_the_rules(hip_device, dtype, dim, n, most, width):
    """Tables on either side of what is taken whole: of many sequences, of few, of heads of both sizes."""
    lens = [most, *_rest(n, n - 1, 0, most)]
    scene = Scene(24, [1] * n, [0] * n, lens, 16, 2, 2, dim, dtype, spare_width=width // 16 - -(-most // 16))
    assert scene.table.shape[1] * 16 == width
    scene.check(scene.run(hip_device, groups=False))


@pytest.mark.parametrize('dtype, dim', [('fp16', 64), ('fp16', 128), ('bf16', 64), ('bf16', 128)])
@pytest.mark.parametrize('page', [16, 64])
@pytest.mark.parametrize('groups, shared, rest, kv_heads, group', [
    ([5], [1500], 0, 3, 1),                        # beams over audio: all rows are shared
    ([5, 5], [1500, 1490], 0, 2, 1),
    ([5], [224], 150, 3, 1),                       # short: a block a sequence
    ([2, 1, 3], [1300, 0, 1111], 300, 2, 4),       # columns of 8 and 12
    ([20], [1216], 60, 1, 4),                      # 80 columns in several runs
    ([7, 9], [2000, 31], 500, 1, 20),              # 20 heads a key/value head; less than a tile shared
    ([40], [1100], 3, 1, 1),                       # more than 32 sequences
    ([1, 1, 3], [1200, 0, 33], 1200, 2, 2),
    ([20], [1500], 0, 1, 16),                      # 320 columns: 128 in a run, the last one partial
    ([3, 30], [1300, 1411], 70, 1, 20),
    ([2, 2, 2], [1290, 1300, 1400], 200, 2, 32)])  # 64 columns: all of a run
def test_groups(hip_device, dtype, dim, page, groups, shared, rest, kv_heads, group):
    """Groups of every make, and the same sequences without them: both within the bound."""
    n = sum(groups)
    scene = Scene(9, groups, shared, _rest(n, n, 0, rest), page, kv_heads, group, dim, dtype, spare_width=1100 // page)
    scene.check(scene.run(hip_device))
    scene.check(scene.run(hip_device, groups=False))


@pytest.mark.parametrize('shared, rest', [([1500], 0), ([1500], 40), ([64], 1500)])
@pytest.mark.parametrize('idle', [(0,), (2, 4), (0, 1, 2, 3, 4)])
def test_idle_members(hip_device, shared, rest, idle):
    """Idle sequences of a group get zeros, the others what they get without them; also where the first one is idle."""
    scene = Scene(10, [5], shared, _rest(1, 5, 0, rest), 32, 2, 3, 64, 'fp16', spare_width=40, idle=idle)
    out = scene.run(hip_device)
    scene.check(out)
    assert not out[list(idle)].any()


def test_shared_past_the_lengths(hip_device):
    """More rows named as shared than the shortest sequence has, or any: those that all have are shared."""
    scene = Scene(11, [3, 2], [1500, 1200], [0, 100, 700, 0, 0], 32, 2, 2, 64, 'fp16')
    scene.lens[0] = 1407
    for shared in ([1500, 1200], [1500, 5000], [1450, 2 ** 62], [-5, 7], [2 ** 62, -2 ** 62]):
        scene.shared = np.array(shared)
        scene.check(scene.run(hip_device))
    scene.lens[1] = 0  # a sequence without rows: nothing is shared
    scene.check(scene.run(hip_device))


def test_odd_starts(hip_device):
    """Sequences outside the groups share nothing; starts past the sequences are clamped, ones that descend make no groups."""
    scene = Scene(12, [1, 3, 2, 1], [0, 1300, 1250, 0], [1400, 5, 90, 200, 7, 8, 3], 64, 2, 2, 128, 'bf16')
    for cu, shared in (([1, 4, 6], [1300, 1250]), ([1, 4], [1300]), ([4, 6, 99], [1250, 0]), ([0, 0, 0, 1, 4], [5, 5, 9999, 1300]),
                       ([4, 1, 6], [1300, 1250]), ([-3, 1, 4, 6, 7], [64, 1300, 1250, 0])):
        scene.cu, scene.shared = np.array(cu), np.array(shared)
        if cu == [4, 6, 99]:
            scene.shared = np.array([1250, 0])
        scene.check(scene.run(hip_device))


@pytest.mark.parametrize('page', [16, 32])
@pytest.mark.parametrize('spare', [1, 80])
def test_bad_pages(hip_device, page, spare):
    """Entries that are no page hide their rows: at the start, the middle, the end, in all of a sequence and in shared rows."""
    scene = Scene(13, [2, 1, 1, 1], [640, 0, 0, 0], [100, 50, 300, 40, 333], page, 2, 2, 64, 'fp16', spare_width=spare)
    t = scene.table
    t[0:2, 3] = -1
    t[0:2, 4] = 2 ** 31 - 1
    t[2, 0], t[2, 2 * 32 // page], t[4, 300 // page] = -5, len(scene.k), len(scene.k) + 7
    t[3] = -2 ** 31
    out = scene.run(hip_device)
    scene.check(out)
    assert not out[3].any()


@pytest.mark.parametrize('page, dim', [(16, 64), (16, 128), (64, 64), (64, 128)])
@pytest.mark.parametrize('group', [5, 70])
def test_bad_pages_of_many_columns(hip_device, page, dim, group):
    """Entries that are no page among shared rows that many columns see, at halves and ends of steps, and in the last one."""
    scene = Scene(20, [5, 1], [1500, 0], [0, 0, 0, 0, 0, 700], page, 1, group, dim, 'bf16')
    t = scene.table
    for j in (0, 1, 2, 3, 5, 8, 13, 1499 // page):
        if j <= 1499 // page:
            t[:5, j] = (-1, len(scene.k), 2 ** 31 - 1)[j % 3]
    scene.check(scene.run(hip_device))
    t[:5] = -1
    out = scene.run(hip_device)
    scene.check(out)
    assert not out[:5].any()


def test_groups_of_one(hip_device):
    """As many groups as sequences: taken as none, whatever they say."""
    scene = Scene(21, [1] * 6, [0] * 6, [1300, 5, 0, 900, 33, 64], 32, 2, 2, 64, 'fp16', spare_width=20)
    for cu, shared in ((np.arange(7), [900] * 6), ([0, 6, 6, 6, 6, 6, 6], [0] * 6)):
        scene.cu, scene.shared = np.array(cu), np.array(shared)
        scene.check(scene.run(hip_device))


def test_seen_with_hidden_nan(hip_device):
    """(Every scene holds NaN behind the lengths.) Infinities there count as little."""
    for dtype in ('fp16', 'bf16'):
        scene = Scene(14, [3], [1100], [1, 9, 70], 16, 2, 1, 64, dtype)
        scene.k[torch.isnan(scene.k)] = float('-inf')
        scene.v[torch.isnan(scene.v)] = float('inf')
        scene.check(scene.run(hip_device))


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('scale', [0.0, -0.125, 3.0, 1e-30])
def test_scales(hip_device, dtype, scale):
    scene = Scene(15, [4], [1200], [3, 60, 0, 900], 32, 2, 2, 64, dtype)
    scene.check(scene.run(hip_device, scale=scale), scale=scale)
    scene.check(scene.run(hip_device, scale=scale, groups=False), scale=scale)


def test_large_scores(hip_device):
    """Scores that pass the running maximum by far, tile by tile, and one key that takes all the weight."""
    scene = Scene(16, [2], [2048], [100, 900], 32, 1, 2, 64, 'fp16')
    scene.k *= torch.linspace(0.1, 12, len(scene.k)).view(-1, 1, 1, 1).half()
    for scale in (0.125, -0.125, 1.0):
        scene.check(scene.run(hip_device, scale=scale), scale=scale)


def test_strided_rows(hip_device):
    """Queries and outputs inside larger tensors; what lies beside them stays."""
    scene = Scene(17, [3, 1], [1216, 0], [5, 40, 0, 1300], 32, 2, 3, 64, 'fp16')
    n, heads, dim = scene.q.shape
    q = torch.full((heads, n + 1, dim + 8), 5.0, dtype=torch.float16, device=hip_device)
    out = torch.full((n, heads + 2, dim), 5.0, dtype=torch.float16, device=hip_device)
    view = q.transpose(0, 1)[:n, :, 8:]
    view.copy_(scene.q)
    scene.check(scene.run(hip_device, q=view, out=out[:, 1:-1]))
    assert (out[:, 0] == 5).all() and (out[:, -1] == 5).all()


def test_many_sequences(hip_device):
    """More sequences than the plan's block has threads, short, long, idle, in groups of all sizes."""
    rng = np.random.default_rng(18)
    groups = [1] * 300 + [2] * 100 + [40, 70, 130] + [3] * 200
    shared = [0 if g == 1 else int(rng.integers(0, 90)) for g in groups]
    n = sum(groups)
    scene = Scene(18, groups, shared, _rest(18, n, 0, 60), 16, 1, 2, 64, 'fp16', spare_width=70, idle=[5, 301, 500])
    scene.check(scene.run(hip_device))
    scene.check(scene.run(hip_device, groups=False))


@pytest.mark.parametrize('groups, shared', [([1500], [65]), ([2, 1400], [40, 70]), ([1] * 100 + [1300] + [1] * 50, [0] * 100 + [33] + [0] * 50)])
def test_many_sequences_few_groups(hip_device, groups, shared):
    n = sum(groups)
    scene = Scene(22, groups, shared, _rest(22, n, 0, 40), 16, 1, 1, 64, 'bf16', spare_width=70, idle=[3, 1000])
    scene.check(scene.run(hip_device))


@pytest.mark.parametrize('spare', [0, 70])
def test_lengths_past_the_table(hip_device, spare):
    """A sequence longer than its table has the table's rows; the smallest length is idle."""
    scene = Scene(23, [3], [128], [64, 128, 32], 32, 2, 2, 64, 'fp16', spare_width=spare)
    scene.table[scene.table < 0] = 0
    scene.k, scene.v = torch.nan_to_num(scene.k), torch.nan_to_num(scene.v)
    scene.lens = np.array([2 ** 63 - 1, 2 ** 31 + 5, -2 ** 63])
    scene.shared = np.array([128])
    out = scene.run(hip_device)
    scene.check(out)
    assert not out[2].any()


def test_far_pages(hip_device):
    """Pages past 2^31 elements of an array."""
    from flash_whisper_amd.ext import KvPages

    ext, heads, dim, page = _ext(), 8, 128, 256
    n_pages = 2 ** 31 // (heads * dim * page) + 40
    cache = ext.kv_pages(n_pages, heads, page, dim, torch.bfloat16)
    scene = Scene(19, [2], [1300], [40, 500], page, heads, 2, dim, 'bf16', spare_width=1)
    far = n_pages - 1 - np.arange(len(scene.k))
    cache.k[far.tolist()], cache.v[far.tolist()] = scene.k.to(hip_device), scene.v.to(hip_device)
    table = torch.tensor(np.where(scene.table >= 0, n_pages - 1 - scene.table, -1).astype(np.int32), device=hip_device)
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    out = torch.empty_like(scene.q, device=hip_device)
    ws = ext.decode_attention_paged_workspace(2, 16, cache, table.size(1), 1)
    ext.decode_attention_paged(scene.q.to(hip_device), KvPages(*cache), table, i64(scene.lens), out, ws, dim ** -0.5, i64(scene.cu), i64(scene.shared))
    scene.check(out)
