"""A batch of answers to shared prompts, as cases that can be timed and checked one by one.

A server that decodes several answers to one clip or prompt at once (beams, samples, questions to one text) keeps keys
and values in pages, so that the rows all answers share are held once. A step of it needs: pages for the new rows and the
places those go to, found from the requests' lengths; the rows written there; the attention of one new token a sequence,
which reads shared rows once for all; and the rules on the logits: penalties for repeated tokens, biases, the mask of a
grammar. Head counts and lengths are those of whisper-large-v3-turbo (20 heads of 64, 448 positions, 1500 audio frames,
51866 tokens) and, for other language models, grouped heads of 128, long prefixes and other vocabularies.

Kinds:
  map     page tables brought up to the sequences' lengths from a stack of free pages, and the slots of the new rows
  append  rows of k and v written to their slots
  attend  one query a sequence over lens[s] rows in pages; the sequences of a group share their first rows
  rules   logits under penalties, biases and masks

Pages of P rows (h kv heads, D dims):
  k [pages, h, P, D]        row-major
  v [pages, h, P/8, D, 8]   8 rows of a dim together: row t, dim d at [t / 8, d, t % 8]
Slot x is row x % P of page x / P; a negative one is no place. A sequence's row j is row j % P of page table[s, j / P].

Map: sequence s has rows pos[s] .. of cu[s + 1] - cu[s] new rows, and wants the pages of all rows up to its last. Pages it
holds beyond that and owns (from entry own[s] on) go back onto the stack, in the order of sequences and entries; then pages
are taken from the top, in the same order, while there are any. pos < 0: an idle sequence, left as it is, without slots.
Rules, in this order: a token of the row's history: x / r for x > 0, x r else; minus frequency times its count
among the generated tokens, minus presence where that is not 0; plus its bias (of a repeated id the last); -inf where the
mask's bit is 0.
"""

import random

import torch

own = False

DEV = 'cuda'
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}


def listed():
    return [
        # 64 sequences of a step, a token each
        {'name': 'map_step', 'kind': 'map', 'n': 64, 'new': 1, 'past': 400, 'page': 16, 'gone': 0.03, 'spare': 1.0, 'mix': 1},
        # a round of a large server: prompts of very different lengths come in, tokens go on, requests end
        {'name': 'map_prompts', 'kind': 'map', 'n': 600, 'new': 4000, 'past': 8000, 'page': 32, 'gone': 0.2, 'spare': 0.9,
         'mix': 2},
        # the next token of 8 clips with 5 beams each
        {'name': 'append_token', 'kind': 'append', 'n': 40, 'new': 1, 'past': 400, 'page': 16, 'kv_heads': 20, 'dim': 64,
         'type': 'fp16', 'mix': 3},
        # ragged prompts
        {'name': 'append_prompts', 'kind': 'append', 'n': 12, 'new': 8000, 'past': 500, 'page': 64, 'kv_heads': 8,
         'dim': 128, 'type': 'bf16', 'mix': 4},
        # self attention of one clip's 5 beams: the prompt's rows are shared
        {'name': 'attend_beams', 'kind': 'attend', 'groups': '5', 'shared': 224, 'rest': 150, 'rest_min': 150, 'page': 16,
         'width': 28, 'heads': 20, 'kv_heads': 20, 'dim': 64, 'type': 'fp16', 'mix': 5},
        # cross attention of 8 clips with 5 beams each: all rows are shared
        {'name': 'attend_audio', 'kind': 'attend', 'groups': '5,5,5,5,5,5,5,5', 'shared': 1500, 'rest': 0, 'rest_min': 0, 'page': 32,
         'width': 47, 'heads': 20, 'kv_heads': 20, 'dim': 64, 'type': 'fp16', 'mix': 6},
        # 64 answers to one long text
        {'name': 'attend_samples', 'kind': 'attend', 'groups': '64', 'shared': 8000, 'rest': 1000, 'rest_min': 1, 'page': 32,
         'width': 288, 'heads': 32, 'kv_heads': 8, 'dim': 128, 'type': 'bf16', 'mix': 7},
        # questions to three very long texts, and sequences that share nothing
        {'name': 'attend_texts', 'kind': 'attend', 'groups': '4,1,7,1,1,3', 'shared': 50000, 'rest': 5000, 'rest_min': 100,
         'page': 64, 'width': 1024, 'heads': 64, 'kv_heads': 8, 'dim': 128, 'type': 'fp16', 'mix': 8},
        # one clip's next token: history and the suppressed tokens
        {'name': 'rules_token', 'kind': 'rules', 'rows': 1, 'vocab': 51866, 'type': 'fp16', 'history': 224, 'biased': 0, 'sets': 1,
         'penalties': True, 'mix': 9},
        # 8 clips with 5 beams each, some words favoured, one of a few grammar states each
        {'name': 'rules_beams', 'kind': 'rules', 'rows': 40, 'vocab': 51866, 'type': 'fp16', 'history': 448, 'biased': 100,
         'sets': 6, 'penalties': True, 'mix': 10},
        # a large batch with long histories
        {'name': 'rules_batch', 'kind': 'rules', 'rows': 256, 'vocab': 100003, 'type': 'fp32', 'history': 9000, 'biased': 300,
         'sets': 256, 'penalties': True, 'mix': 11},
    ]


def _log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(['map', 'append', 'attend', 'attend', 'attend', 'rules', 'rules'])
    case = {'kind': kind, 'mix': rng.randrange(1 << 20)}
    page = rng.choice([16, 32, 64, 128])
    if kind == 'map':
        n, new = _log_int(rng, 1, 800), rng.choice([1, _log_int(rng, 1, 4000)])
        return {**case, 'n': n, 'new': min(new, max(1, 200000 // n)), 'past': _log_int(rng, 1, 8000), 'page': page,
                'gone': rng.choice([0.0, 0.1, 0.4]), 'spare': rng.choice([0.5, 1.0, 1.0])}
    if kind == 'rules':
        vocab = rng.choice([_log_int(rng, 100, 100000), 51865, 51866, 32000])
        rows = _log_int(rng, 1, max(1, min(256, 12000000 // vocab)))
        return {**case, 'rows': rows, 'vocab': vocab, 'type': rng.choice(['fp16', 'bf16', 'fp32']),
                'history': rng.choice([0, _log_int(rng, 1, 9000)]), 'biased': rng.choice([0, _log_int(rng, 1, 300)]),
                'sets': rng.choice([0, 1, rows, rng.randrange(1, rows + 1)]), 'penalties': rng.random() < 0.8}
    dim, kv_heads = rng.choice([64, 128]), rng.choice([1, 2, 4, 5, 8, 20])
    case.update(page=page, kv_heads=kv_heads, dim=dim, type=rng.choice(['fp16', 'bf16']))
    if kind == 'append':
        new = rng.choice([1, _log_int(rng, 1, 8000)])
        return {**case, 'n': _log_int(rng, 1, max(1, min(256, 16000 // new))), 'new': new, 'past': _log_int(rng, 1, 2000),
                'kv_heads': min(kv_heads, 8)}
    shared, rest = rng.choice([0, _log_int(rng, 1, 40000)]), _log_int(rng, 1, 8000)
    # at most 80 Mi elements of K over all sequences
    most = max(1, (80 << 20) // ((shared + rest) * kv_heads * dim))
    left, groups = _log_int(rng, 1, min(most, 128)), []
    while left:
        groups.append(rng.randrange(1, left + 1) if rng.random() < 0.7 else 1)
        left -= groups[-1]
    return {**case, 'groups': ','.join(map(str, groups)), 'shared': shared, 'rest': rest, 'rest_min': _log_int(rng, 1, rest),
            'width': (shared + rest) // page + rng.randrange(1, 20), 'heads': kv_heads * rng.choice([1, 1, 2, 4, 5, 8, 16])}


# ---- inputs ---------------------------------------------------------------------------------


def _lengths(rng, n, high, low):
    """n lengths between low and high, spread over their logarithm, the longest among them."""
    some = [high] + [_log_int(rng, max(low, 1), max(high, 1)) if high else 0 for _ in range(n - 1)]
    rng.shuffle(some)
    return some


def _ints(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _starts(lengths):
    cu = [0]
    for x in lengths:
        cu.append(cu[-1] + x)
    return cu


def _normal(gen, shape, kind):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(kind)


def _level(gen, shape, heads, kind):
    """Keys and values: a level of its own for each head dim, as projections with a bias have, plus noise. `heads`
    has the sizes of shape along the axes of head and dim, 1 elsewhere."""
    level = torch.randn(heads, generator=gen, device=DEV)
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).add_(level).to(kind)


def _map_plan(case):
    """Lengths and pages of a map case, as lists: pos, new, held, own, width, pages."""
    rng, page = random.Random(case['mix']), case['page']
    pos = _lengths(rng, case['n'], case['past'], 1)
    new = [1 if rng.random() < 0.7 else x for x in _lengths(rng, case['n'], case['new'], 1)]
    held, mine = [-(-p // page) for p in pos], []
    for s in range(case['n']):
        if rng.random() < case['gone']:  # ended, rolled back, or idle
            how = rng.randrange(3)
            pos[s], new[s] = (0, 0) if how == 0 else (rng.randrange(pos[s] + 1), new[s]) if how == 1 else (-1, new[s])
        mine.append(rng.choice([0, 0, rng.randrange(held[s] + 1)]))
    want = [-(-(p + x) // page) if p >= 0 else h for p, x, h in zip(pos, new, held)]
    takes = sum(max(0, w - h) for w, h in zip(want, held))
    free = int(takes * case['spare']) + (10 if case['spare'] == 1 else 0)
    return pos, new, held, mine, max(max(want), max(held)) + 3, free


def _map_state(case, seed):
    pos, new, held, mine, width, free = _map_plan(case)
    gen = torch.Generator().manual_seed(seed)
    pages = sum(held) + free
    order = torch.randperm(pages, generator=gen, dtype=torch.int32)
    table = torch.zeros(case['n'], width, dtype=torch.int32)
    at = 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    stack = torch.zeros(pages, dtype=torch.int32)
    stack[:free] = order[at:]
    cu = _starts(new)
    return {'pos': _ints(pos), 'cu': _ints(cu), 'held': _ints(held), 'own': _ints(mine), 'table': table.to(DEV),
            'free': stack.to(DEV), 'count': _ints([free, 0]), 'slots': torch.full((cu[-1],), -1, dtype=torch.int64, device=DEV),
            'held_out': _ints(held), 'count_out': _ints([0, 0]), 'page': case['page']}


def _append_plan(case):
    """pos, new and the pages there are."""
    rng = random.Random(case['mix'])
    new = _lengths(rng, case['n'], case['new'], 1)
    pos = [rng.randrange(case['past'] + 1) for _ in new]
    return pos, new, sum(-(-(p + x) // case['page']) for p, x in zip(pos, new))


def _pages(gen, case, pages, make):
    kind, h, p, d = TYPES[case['type']], case['kv_heads'], case['page'], case['dim']
    return make(gen, (pages, h, p, d), (1, h, 1, d), kind), make(gen, (pages, h, p // 8, d, 8), (1, h, 1, d, 1), kind)


def _append_state(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    pos, new, pages = _append_plan(case)
    kind, page = TYPES[case['type']], case['page']
    order, slots, at = torch.randperm(pages, generator=gen, device=DEV), [], 0
    for p, x in zip(pos, new):
        row = torch.arange(p, p + x, device=DEV)
        slots.append(order[at + row // page] * page + row % page)
        at += -(-(p + x) // page)
    slots = torch.cat(slots)
    slots[torch.rand(slots.shape, generator=gen, device=DEV) < 0.001] = -1  # rows that got no page
    shape = (sum(new), case['kv_heads'], case['dim'])
    cache = _pages(gen, case, pages, lambda g, full, heads, dtype: torch.zeros(full, dtype=dtype, device=DEV))
    return {'k': _level(gen, shape, shape[1:], kind), 'v': _level(gen, shape, shape[1:], kind), 'slots': slots, 'cache': cache}


def _attend_plan(case):
    """For each group its members and its shared rows, for each sequence its rows."""
    rng, groups = random.Random(case['mix']), [int(x) for x in case['groups'].split(',')]
    shared = _lengths(rng, len(groups), case['shared'], case['shared'] // 4)
    shared = [x if n > 1 else 0 for x, n in zip(shared, groups)]
    each = [x for x, n in zip(shared, groups) for _ in range(n)]
    rest = _lengths(rng, len(each), case['rest'], case['rest_min'])
    return groups, shared, [a + b for a, b in zip(each, rest)]


def _attend_state(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, page, (groups, shared, lens) = TYPES[case['type']], case['page'], _attend_plan(case)
    n, own_pages, at = len(lens), [], 0
    table, s = torch.zeros(n, case['width'], dtype=torch.int32), 0
    for rows, members in zip(shared, groups):
        # shared rows that end inside the last page of every member leave it shared, else each has its own copy
        whole = -(-rows // page) if all(x == rows for x in lens[s:s + members]) else rows // page
        table[s:s + members, :whole] = torch.arange(at, at + whole, dtype=torch.int32)
        at += whole
        for i in range(s, s + members):
            more = -(-lens[i] // page) - whole
            table[i, whole:whole + more] = torch.arange(at, at + more, dtype=torch.int32)
            if rows % page and more > 0:
                own_pages.append((s, i, whole))
            at += more
        s += members
    k, v = _pages(gen, case, at, _level)
    order = torch.randperm(at, generator=gen, device=DEV)
    table = order[table.to(DEV).long()].to(torch.int32)
    for first, i, j in own_pages:  # the shared rows of a page that is filled up by each member for itself
        if i > first:
            k[table[i, j]] = k[table[first, j]]
            v[table[i, j]] = v[table[first, j]]
    q = _normal(gen, (n, case['heads'], case['dim']), kind)
    return {'q': q, 'cache': (k, v), 'table': table, 'lens': _ints(lens), 'out': torch.empty_like(q),
            'cu': _ints(_starts(groups)), 'shared': _ints(shared), 'scale': case['dim'] ** -0.5}


def _history_lengths(case):
    rng = random.Random(case['mix'])
    return [x if case['history'] else 0 for x in _lengths(rng, case['rows'], case['history'], case['history'] // 4)]


def _rules_state(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows, vocab, kind = case['rows'], case['vocab'], TYPES[case['type']]
    s = {'x': _normal(gen, (rows, vocab), torch.float32).mul_(3).to(kind), 'history': bool(case['history']),
         'biased': bool(case['biased']), 'sets': bool(case['sets']), 'penalties': case['penalties']}
    s['out'] = torch.empty_like(s['x'])
    lengths = _history_lengths(case)
    # some tokens are far more frequent than others
    often = torch.rand(sum(lengths), generator=gen, device=DEV).pow_(4)
    s.update(tokens=(often * vocab).long().clamp_(max=vocab - 1), cu=_ints(_starts(lengths)),
             prompt=_ints([x // 3 for x in lengths]))
    even = lambda low, high: low + (high - low) * torch.rand(rows, generator=gen, device=DEV)  # noqa: E731
    s.update(repetition=even(0.8, 1.5), presence=even(0.0, 1.0), frequency=even(0.0, 0.3))
    s.update(bias_ids=torch.randint(vocab, (rows * case['biased'],), generator=gen, device=DEV),
             bias=even(0, 1).repeat_interleave(case['biased'], output_size=rows * case['biased']).mul_(7).sub_(3),
             cu_bias=_ints([i * case['biased'] for i in range(rows + 1)]))
    words = (vocab + 31) // 32
    masks = torch.randint(-2**31, 2**31, (2, case['sets'], words), generator=gen, device=DEV)
    s['masks'] = (masks[0] | masks[1]).to(torch.int32)  # three of four tokens may come
    s['mask_of'] = torch.randint(-1 if case['sets'] > 1 else 0, max(case['sets'], 1), (rows,), generator=gen, device=DEV)
    return s


def prepare(case, seed):
    make = {'map': _map_state, 'append': _append_state, 'attend': _attend_state, 'rules': _rules_state}[case['kind']]
    return {'kind': case['kind'], **make(case, seed)}


# ---- the plain form ---------------------------------------------------------------------------


def _plain_map(s):
    pos, cu, held, mine, page = s['pos'], s['cu'], s['held'], s['own'], s['page']
    table, free, width = s['table'], s['free'].clone(), s['table'].size(1)
    rows = pos + cu.diff()
    need = torch.where(pos < 0, held, (rows + page - 1) // page)
    want = need.clamp(max=width)
    entry = torch.arange(width, device=DEV)[None]
    # back onto the stack
    low = torch.maximum(want, mine)
    back = (held - low).clamp(min=0)
    place = s['count'][0] + (back.cumsum(0) - back)[:, None] + entry - low[:, None]
    given = (entry >= low[:, None]) & (entry < held[:, None])
    stack = torch.cat([free, free.new_zeros(1)])
    stack[torch.where(given, place, free.numel())] = torch.where(given, table, 0)
    top = s['count'][0] + back.sum()
    # and off it
    take = (want - held).clamp(min=0)
    rank = (take.cumsum(0) - take)[:, None] + entry - held[:, None]
    taken = (entry >= held[:, None]) & (entry < want[:, None]) & (rank < top)
    table = torch.where(taken, stack[(top - 1 - rank).clamp(min=0, max=free.numel() - 1)], table)
    got = taken.sum(1)
    now = torch.where(want > held, held + got, want)
    missing = (need - want).clamp(min=0).sum() + (take - got).sum()
    # the slots of the rows
    row = torch.arange(s['slots'].numel(), device=DEV)
    seq = torch.bucketize(row, cu[1:], right=True)
    at = pos[seq] + row - cu[seq]
    page_of = table[seq, (at // page).clamp(min=0, max=width - 1)].long()
    slots = torch.where((pos[seq] >= 0) & (at // page < now[seq]), page_of * page + at % page, -1)
    s['table'].copy_(table)
    return {'table': s['table'], 'held': now, 'stack': stack[:-1], 'count': torch.stack([top - got.sum(), missing]), 'slots': slots}


def _plain_append(s):
    k, v, slots = s['k'], s['v'], s['slots']
    (ck, cv), page = s['cache'], s['cache'][0].size(2)
    # rows without a place repeat the first one that has one, or leave slot 0 as it is
    has = slots >= 0
    rows = torch.where(has, torch.arange(slots.numel(), device=DEV), has.int().argmax())
    any_, at = has.any(), slots[rows].clamp(min=0)
    k_at, v_at = (at // page, slice(None), at % page), (at // page, slice(None), at % page // 8, slice(None), at % 8)
    ck[k_at] = torch.where(any_, k[rows], ck[k_at])
    cv[v_at] = torch.where(any_, v[rows], cv[v_at])
    return ck, cv


def _plain_attend(s):
    q, (k, v), lens = s['q'], s['cache'], s['lens']
    (n, heads, dim), (_, kv_heads, page, _) = q.shape, k.shape
    table = s['table'].long()
    kp = k[table].transpose(1, 2).reshape(n, kv_heads, -1, dim).float()
    vp = v[table].permute(0, 2, 1, 3, 5, 4).reshape(n, kv_heads, -1, dim).float()
    scores = (q.float() * s['scale']).view(n, kv_heads, heads // kv_heads, dim) @ kp.transpose(2, 3).contiguous()
    seen = torch.arange(kp.size(2), device=DEV) < lens[:, None, None, None]
    scores.masked_fill_(~seen, float('-inf'))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == float('-inf'), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return ((p @ vp) / torch.where(total == 0, 1.0, total)).view(n, heads, dim).to(q.dtype)


def _plain_rules(s):
    x = s['x'].float()
    rows, vocab = x.shape
    if s['history'] and s['penalties']:
        place = torch.arange(s['tokens'].numel(), device=DEV)
        row = torch.bucketize(place, s['cu'][1:], right=True)
        count = torch.zeros(2, rows * vocab, dtype=torch.int32, device=DEV)
        key = row * vocab + s['tokens']
        fresh = place - s['cu'][row] >= s['prompt'][row]
        count[0].index_add_(0, key, torch.ones_like(key, dtype=torch.int32))
        count[1].index_add_(0, key, fresh.int())
        count = count.view(2, rows, vocab)
        r = s['repetition'][:, None]
        x = torch.where(count[0] > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - s['frequency'][:, None] * count[1] - s['presence'][:, None] * (count[1] > 0)
    if s['biased']:
        place = torch.arange(s['bias_ids'].numel(), device=DEV)
        row = torch.bucketize(place, s['cu_bias'][1:], right=True)
        last = torch.full((rows * vocab,), -1, dtype=torch.int64, device=DEV)
        last.scatter_reduce_(0, row * vocab + s['bias_ids'], place, 'amax')
        last = last.view(rows, vocab)
        x = x + torch.where(last >= 0, s['bias'][last.clamp(min=0)], 0.0)
    if s['sets']:
        bits = torch.arange(vocab, device=DEV)
        words = s['masks'][s['mask_of'].clamp(min=0)][:, bits // 32]
        may = ((words >> (bits % 32).int()) & 1).bool() | (s['mask_of'] < 0)[:, None]
        x = torch.where(may, x, float('-inf'))
    return x.to(s['x'].dtype)


def _own(s):
    from flash_whisper_amd.ext import KvPages, load_ext

    ext = load_ext()
    if s['kind'] == 'map':
        ext.kv_page_map(s['pos'], s['cu'], s['table'], s['held'], s['free'], s['count'], s['slots'], s['page'], s['own'],
                        s['held_out'], s['count_out'])
        return {'table': s['table'], 'held': s['held_out'], 'stack': s['free'], 'count': s['count_out'], 'slots': s['slots']}
    if s['kind'] == 'append':
        ext.kv_page_append(s['k'], s['v'], s['slots'], KvPages(*s['cache']))
        return s['cache']
    if s['kind'] == 'attend':
        cache = KvPages(*s['cache'])
        if 'ws' not in s:  # a decoding stream keeps its workspace
            s['ws'] = ext.decode_attention_paged_workspace(*s['q'].shape[:2], cache, s['table'].size(1), s['shared'].numel())
        ext.decode_attention_paged(s['q'], cache, s['table'], s['lens'], s['out'], s['ws'], s['scale'], s['cu'], s['shared'])
        return s['out']
    rules = {}
    if s['history'] and s['penalties']:
        rules.update({name: s[name] for name in ('tokens', 'cu', 'prompt', 'repetition', 'presence', 'frequency')})
    if s['biased']:
        rules.update({name: s[name] for name in ('bias_ids', 'bias', 'cu_bias')})
    if s['sets']:
        rules.update(masks=s['masks'], mask_of=s['mask_of'])
    ext.logits_rules(s['x'], s['out'], **rules)
    return s['out']


def run(s):
    if own:
        return _own(s)
    return {'map': _plain_map, 'append': _plain_append, 'attend': _plain_attend, 'rules': _plain_rules}[s['kind']](s)


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    if case['kind'] == 'map':
        pos, new, held, mine, _, free = _map_plan(case)
        want = [-(-(p + x) // case['page']) if p >= 0 else h for p, x, h in zip(pos, new, held)]
        moved = sum(max(0, h - max(w, m)) for w, h, m in zip(want, held, mine))
        moved += min(free + moved, sum(max(0, w - h) for w, h in zip(want, held)))
        # lengths in, held out, pages moved between table and stack, slots out with their pages
        return {'bytes': case['n'] * 5 * 8 + moved * 8 + sum(new) * 8 + sum(new) // case['page'] * 4, 'flops': sum(new) * 4}
    if case['kind'] == 'append':
        rows = sum(_append_plan(case)[1])
        return {'bytes': rows * (8 + 2 * 2 * 2 * case['kv_heads'] * case['dim']), 'flops': rows * case['kv_heads'] * 8}
    if case['kind'] == 'attend':
        groups, shared, lens = _attend_plan(case)
        each = [x for x, n in zip(shared, groups) for _ in range(n)]
        rows = sum(shared) + sum(a - b for a, b in zip(lens, each))
        return {'bytes': 4 * len(lens) * case['heads'] * case['dim'] + rows * case['kv_heads'] * case['dim'] * 4
                + -(-rows // case['page']) * 4, 'flops': 4 * case['dim'] * case['heads'] * sum(lens)}
    size, some = TYPES[case['type']].itemsize, case['rows'] * case['vocab']
    return {'bytes': 2 * size * some + (sum(_history_lengths(case)) * 8 if case['penalties'] else 0)
            + case['rows'] * case['biased'] * 12 + case['sets'] * ((case['vocab'] + 31) // 32) * 4, 'flops': 4 * some}


# ---- the definition in 64 bits --------------------------------------------------------------------


def _exact_map(s):
    """The sequences one after another, page by page."""
    pos, cu, held, mine, stack = (s[x].tolist() for x in ('pos', 'cu', 'held', 'own', 'free'))
    table, page, (count, _) = s['table'].tolist(), s['page'], s['count'].tolist()
    width, missing, slots = len(table[0]), 0, []
    rows = [p + b - a for p, a, b in zip(pos, cu, cu[1:])]
    for i, p in enumerate(pos):
        pages = -(-rows[i] // page)
        if p >= 0 and pages < held[i]:
            for j in range(max(pages, mine[i]), held[i]):
                stack[count] = table[i][j]
                count += 1
            held[i] = pages
    for i, p in enumerate(pos):
        for j in range(held[i], -(-rows[i] // page) if p >= 0 else 0):
            if j < width and count:
                count -= 1
                table[i][j] = stack[count]
                held[i] = j + 1
            else:
                missing += 1
        for row in range(p, rows[i]):
            slots.append(table[i][row // page] * page + row % page if p >= 0 and row // page < held[i] else -1)
    f = lambda x: torch.tensor(x, dtype=torch.float64, device=DEV)  # noqa: E731
    return {'table': f(table), 'held': f(held), 'stack': f(stack), 'count': f([count, missing]), 'slots': f(slots)}


def _exact_append(s):
    ck, cv = (x.double() for x in s['cache'])
    page = ck.size(2)
    for row, slot in enumerate(s['slots'].tolist()):
        if slot >= 0:
            ck[slot // page, :, slot % page] = s['k'][row].double()
            cv[slot // page, :, slot % page // 8, :, slot % 8] = s['v'][row].double()
    return ck, cv


def _exact_attend(s):
    q, (k, v) = s['q'], s['cache']
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    page, group = k.size(2), q.size(1) // k.size(1)
    for i, length in enumerate(s['lens'].tolist()):
        pages = s['table'][i, :-(-length // page)].long()
        for h in range(k.size(1)):
            kk = k[pages, h].reshape(-1, q.size(2))[:length].double()
            vv = v[pages, h].transpose(2, 3).reshape(-1, q.size(2))[:length].double()
            if length:
                score = q[i, h * group:(h + 1) * group].double() @ kk.T.contiguous() * s['scale']
                out[i, h * group:(h + 1) * group] = torch.softmax(score, -1) @ vv
    return out


def _exact_rules(s):
    x = s['x'].double()
    vocab = x.size(1)
    cu, cu_bias = s['cu'].tolist(), s['cu_bias'].tolist()
    for r in range(x.size(0)):
        if s['history'] and s['penalties']:
            tokens, prompt = s['tokens'][cu[r]:cu[r + 1]], s['prompt'][r].item()
            met = torch.unique(tokens)
            y = x[r, met]
            x[r, met] = torch.where(y > 0, y / s['repetition'][r].double(), y * s['repetition'][r].double())
            made, count = torch.unique(tokens[prompt:], return_counts=True)
            x[r, made] -= s['frequency'][r].double() * count + s['presence'][r].double()
        if s['biased']:
            ids, values = s['bias_ids'][cu_bias[r]:cu_bias[r + 1]].tolist(), s['bias'][cu_bias[r]:cu_bias[r + 1]].tolist()
            for i, b in dict(zip(ids, values)).items():
                x[r, i] += b
        of = s['mask_of'][r].item()
        if s['sets'] and of >= 0:
            bits = s['masks'][of][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32) & 1
            x[r, bits.flatten()[:vocab] == 0] = float('-inf')
    return x


def exact(case, seed):
    s = prepare(case, seed)
    return {'map': _exact_map, 'append': _exact_append, 'attend': _exact_attend, 'rules': _exact_rules}[case['kind']](s)
