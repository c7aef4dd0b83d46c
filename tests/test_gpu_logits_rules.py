"""Rules on logits against the float64 oracle."""

import numpy as np
import pytest
import torch

from oracle import pages as oracle

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _ext():
    from flash_whisper_amd.ext import load_ext

    return load_ext()


def check(got, x, rules, dtype):
    """At most 5 roundings in fp32, of x / r or x r, f c, two differences and the bias, each 2^-24 of what has been summed up in
    size; then one to the type (half a step, fp16 below 2^-14: 2^-25)."""
    want, size = oracle.rules(x.double().cpu().numpy(), **rules)
    got = got.double().cpu().numpy()
    u, low = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    fp32 = 5 * 2.0 ** -24 * size
    assert np.array_equal(np.isneginf(got), np.isneginf(want)) and np.array_equal(np.isnan(got), np.isnan(want))
    some = np.isfinite(want)
    with np.errstate(invalid='ignore'):
        err = np.abs(got - want)[some]
    tol = ((u * (np.abs(want) + fp32) if dtype != torch.float32 else 0) + fp32 + low)[some]
    assert (err <= tol).all(), f'{err.max():.3e}, {(err / tol).max():.2f}'


def make(rng, rows, vocab, dtype, history=0, biased=0, sets=0, prompt=True, penalties=('repetition', 'presence', 'frequency')):
    """Logits and rules as NumPy; ids at both ends of the vocabulary, some outside it, many twice."""
    x = torch.from_numpy((3 * rng.standard_normal((rows, vocab))).astype(np.float32)).to(dtype)
    rules = {}
    ids = lambda n: np.concatenate([rng.integers(0, vocab, n), rng.integers(0, min(vocab, 9), n), [vocab - 1, 0, -1, vocab, 2 ** 40, -2 ** 40]])
    if history:
        lengths = rng.integers(0, history + 1, rows)
        lengths[0] = history
        rules.update(cu=np.r_[0, np.cumsum(lengths)])
        rules.update(tokens=rng.permutation(np.resize(ids(history * rows), lengths.sum())))
        if prompt:
            rules.update(prompt=rng.integers(-1, lengths + 2))
        if 'repetition' in penalties:
            rules.update(repetition=rng.uniform(0.5, 2, rows).astype(np.float32))
        if 'presence' in penalties:
            rules.update(presence=rng.uniform(-1, 2, rows).astype(np.float32))
        if 'frequency' in penalties:
            rules.update(frequency=rng.uniform(-0.2, 0.5, rows).astype(np.float32))
    if biased:
        lengths = rng.integers(0, biased + 1, rows)
        lengths[-1] = biased
        rules.update(cu_bias=np.r_[0, np.cumsum(lengths)], bias_ids=rng.permutation(np.resize(ids(biased * rows), lengths.sum())),
                     bias=rng.uniform(-9, 9, lengths.sum()).astype(np.float32))
    if sets:
        masks = rng.integers(-2 ** 31, 2 ** 31, (sets, (vocab + 31) // 32)).astype(np.int32)
        masks[0] = 0  # allows nothing
        rules.update(masks=masks, mask_of=rng.integers(-1, sets + 1, rows))
    return x, rules


def run(dev, x, rules, out=None, **more):
    t = {k: torch.from_numpy(np.ascontiguousarray(v)).to(dev) for k, v in rules.items()}
    x = x.to(dev) if not x.is_cuda else x
    out = torch.full_like(x, 7.0) if out is None else out
    _ext().logits_rules(x, out, **t)
    return out


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab', [(1, 1), (3, 7), (2, 31), (5, 33), (1, 2047), (2, 2049), (1, 51866), (4, 51865), (9, 4097), (120, 40001)])
def test_all_rules(hip_device, dtype, rows, vocab):
    rng = np.random.default_rng(rows * 100000 + vocab)
    x, rules = make(rng, rows, vocab, dtype, history=60, biased=25, sets=3)
    check(run(hip_device, x, rules), x, rules, dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kwargs', [{}, dict(history=1), dict(history=5000), dict(history=50, prompt=False), dict(biased=1), dict(biased=700),
                                    dict(sets=1), dict(sets=6), dict(history=50, penalties=('repetition',)),
                                    dict(history=50, penalties=('presence',), sets=2), dict(history=50, penalties=('frequency',), biased=9),
                                    dict(history=50, penalties=())])
def test_each_rule(hip_device, dtype, kwargs):
    rng = np.random.default_rng(len(str(kwargs)))
    x, rules = make(rng, 6, 5003, dtype, **kwargs)
    check(run(hip_device, x, rules), x, rules, dtype)


@pytest.mark.parametrize('dtype', TYPES)
def test_long_lists(hip_device, dtype):
    """Histories and lists too long for a cell of both: counts of 32767 and more, places past 65535; beside them short ones."""
    rng = np.random.default_rng(21)
    vocab, lengths, listed = 9001, [32767, 32768, 90000, 0, 10], [65535, 65536, 3, 70000, 0]
    x, _ = make(rng, 5, vocab, dtype)
    tokens = rng.integers(0, vocab, sum(lengths))
    tokens[:32767] = 17                           # one token alone: the largest count that a cell holds
    tokens[32767 + 32768:32767 + 32768 + 60000] = 4096
    rules = dict(tokens=tokens, cu=np.r_[0, np.cumsum(lengths)], prompt=np.array([0, 5, 100, 0, 3]),
                 repetition=rng.uniform(0.5, 2, 5).astype(np.float32), presence=rng.uniform(-1, 2, 5).astype(np.float32),
                 frequency=rng.uniform(-1e-3, 1e-3, 5).astype(np.float32), bias_ids=rng.integers(-5, vocab + 5, sum(listed)),
                 bias=rng.uniform(-9, 9, sum(listed)).astype(np.float32), cu_bias=np.r_[0, np.cumsum(listed)])
    check(run(hip_device, x, rules), x, rules, dtype)
    check(run(hip_device, x, {k: v for k, v in rules.items() if 'bias' not in k}), x, {k: v for k, v in rules.items() if 'bias' not in k}, dtype)
    check(run(hip_device, x, {k: v for k, v in rules.items() if 'bias' in k}), x, {k: v for k, v in rules.items() if 'bias' in k}, dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, history', [(3, 20001, 300), (3, 20001, 3000), (90, 100001, 2500)])
def test_slices(hip_device, dtype, rows, vocab, history):
    """Slices of each size, the last of a row partial."""
    rng = np.random.default_rng(rows + history)
    x, rules = make(rng, rows, vocab, dtype, history=history, biased=40, sets=2)
    check(run(hip_device, x, rules), x, rules, dtype)


def test_mask_forms(hip_device):
    """One set for all rows, a set for each row, more sets and words than needed."""
    rng = np.random.default_rng(4)
    x, _ = make(rng, 5, 1000, torch.float16)
    for sets, words in ((1, 32), (5, 32), (8, 40)):
        masks = rng.integers(-2 ** 31, 2 ** 31, (sets, words)).astype(np.int32)
        check(run(hip_device, x, {'masks': masks}), x, {'masks': masks}, torch.float16)


@pytest.mark.parametrize('dtype', TYPES)
def test_in_place_and_strided(hip_device, dtype):
    """out may be logits itself; rows may lie apart at any element, and what lies between them stays."""
    rng = np.random.default_rng(6)
    x, rules = make(rng, 4, 4099, dtype, history=40, biased=5, sets=2)
    a = x.to(hip_device)
    run(hip_device, a, rules, out=a)
    check(a, x, rules, dtype)
    wide, target = (torch.full((4, 4107), 3.0, dtype=dtype, device=hip_device) for _ in range(2))
    wide[:, 3:-5] = x.to(hip_device)
    run(hip_device, wide[:, 3:-5], rules, out=target[:, 1:-7])
    check(target[:, 1:-7], x, rules, dtype)
    assert (target[:, 0] == 3).all() and (target[:, -7:] == 3).all()


def test_numbers_that_are_none(hip_device):
    """NaN and infinite logits: as the formulas have them; a hidden token is -infinity whatever it was."""
    x = torch.tensor([[float('nan'), float('inf'), float('-inf'), 1.0, float('nan'), float('inf'), -0.0, 60000.0]])
    rules = dict(tokens=np.array([0, 1, 2, 7]), cu=np.array([0, 4]), repetition=np.array([0.5], np.float32), bias_ids=np.array([3, 6]),
                 bias=np.array([float('-inf'), 2.0], np.float32), cu_bias=np.array([0, 2]), masks=np.array([[0xCF - 256]], np.int32))
    for dtype in TYPES:
        got = run(hip_device, x.to(dtype), rules)[0].float().tolist()
        inf = float('inf')
        assert np.isnan(got[0]) and got[1] == inf and got[2] == -inf and got[3] == -inf and got[4] == -inf and got[5] == -inf and got[6] == 2.0
        assert got[7] == (inf if dtype == torch.float16 else x.to(dtype)[0, 7].item() * 2)


def test_counts_do_not_depend_on_order(hip_device):
    """The same history in any order gives the same bits; of a repeated bias the last place counts."""
    rng = np.random.default_rng(8)
    x, rules = make(rng, 3, 3001, torch.float32, history=4000)
    rules.update(prompt=np.zeros(3, np.int64))
    first = run(hip_device, x, rules)
    for r in range(3):
        a, b = rules['cu'][r:r + 2]
        rules['tokens'][a:b] = rng.permutation(rules['tokens'][a:b])
    assert torch.equal(first, run(hip_device, x, rules))
    biased = dict(bias_ids=np.full(500, 7), bias=np.arange(500).astype(np.float32), cu_bias=np.array([0, 500, 500, 500]))
    got = run(hip_device, x, biased).cpu()
    assert got[0, 7] == x[0, 7] + 499 and torch.equal(got[1:], x[1:])


def test_far_rows(hip_device):
    """Logits past 2^31 elements."""
    vocab, rows = 60001, 2 ** 31 // 60001 + 3
    x = torch.zeros(rows, vocab, dtype=torch.float16, device=hip_device)
    x[-1] = 4
    masks = np.full((2, (vocab + 31) // 32), -1, np.int32)
    masks[1, 0] = 5
    of = np.full(rows, -1)
    of[-1] = 1
    out = run(hip_device, x, dict(masks=masks, mask_of=of), out=x)
    assert not out[:-1].any() and out[-1, 32:].eq(4).all() and out[-1, 0] == 4 and out[-1, 1] == float('-inf') and out[-1, 2] == 4


def test_no_rows(hip_device):
    x = torch.zeros(0, 50, dtype=torch.float16, device=hip_device)
    _ext().logits_rules(x, x.clone())
