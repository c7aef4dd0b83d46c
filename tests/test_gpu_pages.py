"""Page tables from lengths, and rows written to their slots, against the oracle, bit by bit."""

import numpy as np
import pytest
import torch

from oracle import pages as oracle

pytestmark = pytest.mark.gpu


def _ext():
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def _scene(rng, n, page, most, new, gone, spare, width=None, idle=0.1):
    """Sequences with pages: pos, cu, table, held, own, stack, count, as NumPy."""
    pos = rng.integers(0, most + 1, n)
    held = -(-pos // page)
    more = np.where(rng.random(n) < 0.5, 1, rng.integers(0, new + 1, n))
    ended = rng.random(n) < gone
    pos = np.where(ended, rng.integers(0, pos + 1), pos)
    more = np.where(ended & (rng.random(n) < 0.5), 0, more)
    pos = np.where(rng.random(n) < idle, -1, pos)
    own = rng.integers(0, held + 1)
    width = width or int(max(held.max(), (-(-(pos + more) // page)).max())) + 2
    held = np.minimum(held, width)
    pages = int(held.sum()) + spare
    order = rng.permutation(pages).astype(np.int32)
    table, at = np.full((n, width), -7, np.int32), 0
    for s in range(n):
        table[s, :held[s]] = order[at:at + held[s]]
        at += held[s]
    stack = np.full(pages, -9, np.int32)
    stack[:spare] = order[at:at + spare]
    return pos, np.r_[0, np.cumsum(more)], table, held, own, stack, spare


def _run_map(dev, scene, page, rows=None, with_own=True, in_place=False, calls=1):
    pos, cu, table, held, own, stack, spare = scene
    rows = int(cu[-1]) if rows is None else rows
    i64 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int64, device=dev)
    t_table, t_stack = torch.tensor(table, device=dev), torch.tensor(stack, device=dev)
    t_held, count, slots = i64(held), i64([spare, -5]), torch.full((rows,), -77, dtype=torch.int64, device=dev)
    held_out, count_out = (None, None) if in_place else (torch.full_like(t_held, -3), torch.full_like(count, -3))
    for _ in range(calls):
        _ext().kv_page_map(i64(pos), i64(cu), t_table, t_held, t_stack, count, slots, page, i64(own) if with_own else None,
                           held_out, count_out)
    want = oracle.page_map(pos, cu, table, held, own if with_own else None, stack, spare, rows, page)
    assert np.array_equal(t_table.cpu(), want[0])
    assert (t_held if in_place else held_out).tolist() == want[1]
    assert t_stack.tolist() == want[2]
    assert (count if in_place else count_out).tolist() == want[3]
    assert slots.tolist() == [-77 if x is None else x for x in want[4]]


@pytest.mark.parametrize('page', [16, 32, 64, 128, 256])
@pytest.mark.parametrize('in_place', [False, True])
@pytest.mark.parametrize('n, most, new, gone, spare', [
    (1, 0, 1, 0.0, 3), (1, 500, 3000, 0.0, 400), (7, 40, 1, 0.0, 0), (64, 400, 1, 0.1, 70), (64, 400, 50, 0.5, 10), (300, 900, 40, 0.3, 900),
    (1023, 200, 3, 0.2, 500), (1024, 200, 3, 0.2, 500), (1025, 200, 3, 0.2, 500), (2500, 100, 60, 0.4, 20000), (5, 30000, 9000, 0.4, 3000)])
def test_map(hip_device, page, n, most, new, gone, spare, in_place):
    """Requests that come, go on, are cut back, end and idle; stacks with pages for all, some and none; one launch and two."""
    rng = np.random.default_rng(page * 1000 + n)
    _run_map(hip_device, _scene(rng, n, page, most, new, gone, spare), page, in_place=in_place)


@pytest.mark.parametrize('n, calls', [(40, 3), (1024, 1)])
def test_map_many_rows_take_what_came_back(hip_device, n, calls):
    """Few free pages but many that come back in the same call, and go to rows of many blocks."""
    rng = np.random.default_rng(n)
    pos, cu, table, held, own, stack, spare = _scene(rng, n, 16, 3000, 400, 0.6, 5, idle=0.0)
    own[:] = 0
    _run_map(hip_device, (pos, cu, table, held, own, stack, spare), 16, calls=calls)


@pytest.mark.parametrize('n', [3, 1500])
def test_map_forms(hip_device, n):
    """In place, without `own`, repeated with the same inputs, tables too narrow, rows behind the last sequence."""
    rng = np.random.default_rng(n)
    for kwargs, width in ((dict(in_place=True), None), (dict(with_own=False), None), (dict(calls=3), None), ({}, 4)):
        _run_map(hip_device, _scene(rng, n, 16, 100, 30, 0.3, 2 * n, width=width), 16, **kwargs)
    scene = _scene(rng, n, 16, 100, 30, 0.3, 2 * n)
    _run_map(hip_device, scene, 16, rows=int(scene[1][-1]) + 9)
    scene[1][-1] += 12  # starts past the rows are clamped to them
    _run_map(hip_device, scene, 16, rows=int(scene[1][-1]) - 12)


def test_map_empty(hip_device):
    """No new rows at all, no stack; positions past every table."""
    _run_map(hip_device, (np.array([33, 0]), np.array([0, 0, 0]), np.zeros((2, 4), np.int32), np.array([3, 0]), np.array([0, 0]),
                          np.zeros(0, np.int32), 0), 16)
    scene = (np.array([2 ** 40, 5]), np.array([0, 2, 3]), np.arange(8, dtype=np.int32).reshape(2, 4), np.array([4, 1]),
             np.array([0, 0]), np.zeros(3, np.int32), 0)
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    table, slots, count = torch.tensor(scene[2], device=hip_device), i64([9, 9, 9]), i64([0, 0])
    held = i64([4, 1])
    _ext().kv_page_map(i64([2 ** 40, 5]), i64([0, 2, 3]), table, held, torch.zeros(3, dtype=torch.int32, device=hip_device), count, slots, 16)
    assert held.tolist() == [4, 1] and slots.tolist() == [-1, -1, 4 * 16 + 5] and count.tolist() == [0, 2 ** 36 + 1 - 4]


@pytest.mark.parametrize('in_place', [False, True])
def test_map_most_rows(hip_device, in_place):
    """As many packed rows as a call may have, 2^31 - 256: what the launch has threads for passes 2^31."""
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    rows, last = 2 ** 31 - 256, 300
    table = torch.zeros((2, 24), dtype=torch.int32, device=hip_device)
    stack = torch.arange(44, dtype=torch.int32, device=hip_device)
    held, count, slots = i64(0, 0), i64(44, 0), torch.full((rows,), -77, dtype=torch.int64, device=hip_device)
    outs = () if in_place else (torch.zeros_like(held), torch.zeros_like(count))
    _ext().kv_page_map(i64(0, 5), i64(0, rows - last, rows), table, held, stack, count, slots, 16, None, *outs)
    held, count = outs or (held, count)
    assert held.tolist() == [24, 20] and count.tolist() == [0, (rows - last + 15) // 16 - 24]
    assert table[0].tolist() == list(range(43, 19, -1)) and table[1, :20].tolist() == list(range(19, -1, -1))
    assert slots[:384].tolist() == [16 * (43 - r // 16) + r % 16 for r in range(384)]
    assert slots[-last:].tolist() == [16 * (19 - r // 16) + r % 16 for r in range(5, 5 + last)]
    low, high = torch.aminmax(slots[384:-last])
    assert low.item() == high.item() == -1


def test_map_takes_what_came_back(hip_device):
    """Pages that one sequence gives back go to another in the same call."""
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    table = torch.tensor([[5, 6, 7, 0], [1, 0, 0, 0]], dtype=torch.int32, device=hip_device)
    held, count, slots = i64(3, 1), i64(0, 0), i64(*[9] * 33)
    stack = torch.full((8,), -1, dtype=torch.int32, device=hip_device)
    _ext().kv_page_map(i64(0, 16), i64(0, 0, 33), table, held, stack, count, slots, 16, i64(1, 0))
    assert held.tolist() == [0, 3] and count.tolist() == [0, 1] and table[1].tolist() == [1, 7, 6, 0]
    assert slots.tolist() == [7 * 16 + i for i in range(16)] + [6 * 16 + i for i in range(16)] + [-1]


def _rows(rng, shape, dtype, dev):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype).to(dev)


def _bits(t):
    return t.cpu().view(torch.int16).numpy()


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('heads, dim, page', [(1, 64, 16), (20, 64, 32), (8, 128, 64), (3, 128, 256)])
@pytest.mark.parametrize('lengths', [[1], [8], [1] * 19, [7, 1, 0, 30, 2, 16], [5, 100, 64]])
def test_append(hip_device, dtype, heads, dim, page, lengths):
    """Rows in runs that begin and end anywhere, rows without a place, strided rows; what is not written stays."""
    rng = np.random.default_rng(heads * 1000 + dim + page + len(lengths))
    n_pages = sum(-(-(x + 40) // page) for x in lengths) + 2
    order, slots = list(rng.permutation(n_pages)), []
    for x in lengths:
        pos, mine = int(rng.integers(0, 40)), [order.pop() for _ in range(-(-(x + 40) // page))]
        slots += [int(mine[j // page]) * page + j % page for j in range(pos, pos + x)]
    slots = np.array(slots, np.int64)
    slots[rng.random(len(slots)) < 0.1] = rng.choice([-1, n_pages * page, -(2 ** 40), 2 ** 50])
    rows = len(slots)
    k = _rows(rng, (rows, 2 * heads, dim), dtype, hip_device)[:, heads:]
    v = _rows(rng, (heads, rows, dim), dtype, hip_device).transpose(0, 1)
    cache = _ext().kv_pages(n_pages, heads, page, dim, dtype)
    for t in cache:
        t.copy_(_rows(rng, t.shape, dtype, hip_device))
    want = oracle.append(_bits(cache.k), _bits(cache.v), _bits(k.contiguous()), _bits(v.contiguous()), slots.tolist())
    _ext().kv_page_append(k, v, torch.from_numpy(slots).to(hip_device), cache)
    assert np.array_equal(_bits(cache.k), want[0]) and np.array_equal(_bits(cache.v), want[1])


def test_append_any_order(hip_device):
    """Slots in any order: ascending across pages, backwards, runs that start inside a unit, each window of 8 rows apart."""
    rng = np.random.default_rng(3)
    ext, heads, dim, page, n_pages = _ext(), 2, 64, 16, 40
    size = page * n_pages
    orders = [np.arange(size), np.arange(size)[::-1].copy(), rng.permutation(size),
              np.concatenate([np.arange(s, min(s + 13, size)) for s in rng.permutation(np.arange(0, size, 13))]),
              (np.arange(size) + 5) % size, np.arange(0, size, 8), np.arange(3, 11)]
    for slots in orders:
        k, v = (_rows(rng, (len(slots), heads, dim), torch.float16, hip_device) for _ in range(2))
        cache = ext.kv_pages(n_pages, heads, page, dim)
        want = oracle.append(_bits(cache.k), _bits(cache.v), _bits(k), _bits(v), slots.tolist())
        ext.kv_page_append(k, v, torch.tensor(slots, device=hip_device), cache)
        assert np.array_equal(_bits(cache.k), want[0]) and np.array_equal(_bits(cache.v), want[1])


def test_append_far_rows(hip_device):
    """Pages past 2^31 elements of an array, and rows whose strides pass it."""
    ext, heads, dim, page = _ext(), 8, 128, 256
    n_pages = 2 ** 31 // (heads * dim * page) + 5
    cache = ext.kv_pages(n_pages, heads, page, dim, torch.bfloat16)
    rng = np.random.default_rng(5)
    slots = np.r_[np.arange((n_pages - 1) * page + 3, n_pages * page), 0, n_pages * page]
    k, v = (_rows(rng, (len(slots), heads, dim), torch.bfloat16, hip_device) for _ in range(2))
    ext.kv_page_append(k, v, torch.tensor(slots, device=hip_device), cache)
    assert torch.equal(cache.k[-1, :, 3:], k[:page - 3].transpose(0, 1)) and torch.equal(cache.k[0, :, 0], k[-2])
    got = cache.v[-1].permute(0, 1, 3, 2).reshape(heads, page, dim)
    assert torch.equal(got[:, 3:], v[:page - 3].transpose(0, 1)) and torch.equal(cache.v[0, :, 0, :, 0], v[-2])
    assert not cache.k[1:-1].any() and not cache.v[1:-1].any()


def test_map_below_own(hip_device):
    """A sequence that is cut back into pages of others, and whose `own` is lowered to what it then held, owns what it takes
    from there on: when it ends, every page but those of others is on the stack again."""
    i64 = lambda *x: torch.tensor(x, dtype=torch.int64, device=hip_device)
    table = torch.zeros(2, 8, dtype=torch.int32, device=hip_device)
    stack, count, held, own = torch.arange(12, dtype=torch.int32, device=hip_device), i64(12, 0), i64(0, 0), i64(0, 0)
    step = lambda pos, new: _ext().kv_page_map(i64(*pos), i64(0, new[0], sum(new)), table, held, stack, count,
                                               torch.empty(sum(new), dtype=torch.int64, device=hip_device), 16, own)
    step((0, -1), (80, 0))                                  # five pages of the first
    table[1, :5] = table[0, :5]                             # a fork that lists them, and goes on
    held[1] = own[1] = 5
    step((80, 80), (0, 30))
    assert held.tolist() == [5, 7] and count.tolist() == [5, 0]
    step((80, 40), (0, 0))                                  # cut back to 40 rows: three pages, all of the first's
    assert held.tolist() == [5, 3] and count.tolist() == [7, 0]
    torch.minimum(own, held, out=own)
    step((80, 48), (0, 20))                                 # two pages of its own
    assert held.tolist() == [5, 5] and count.tolist() == [5, 0] and not set(table[1, 3:5].tolist()) & set(table[0, :5].tolist())
    step((80, 0), (0, 0))
    assert held.tolist() == [5, 0] and count.tolist() == [7, 0]
    step((0, 0), (0, 0))
    assert held.tolist() == [0, 0] and count.tolist() == [12, 0] and sorted(stack.tolist()) == list(range(12))
