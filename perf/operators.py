"""Attention over whole prompts and over a cache held in 4 bits, as cases that can be timed and checked one by one.

Serving many clips at once needs three steps next to the batch-1 path: the attention of the prompts of several
sequences (packed, each of its own length), writing keys and values into a cache of 4 bits a value, and the
attention of one new token a sequence over that cache. Head counts and lengths are those of whisper-large-v3-turbo (20
heads of 64, 448 positions, 1500 audio frames) and, for other language models, grouped heads of 128 and long caches.

Kinds:
  prompt  q [tokens, heads, dim] over k, v [tokens, kv_heads, dim], sequences delimited by cu_q and cu_k; causal
          ones see keys up to their own position counted from the end of the sequence
  cache   rows of k and v written into the cache and read back as the values that the cache holds for them
  decode  one query a sequence over lens[s] cached keys; with `fresh`, the new token's row is written at lens[s] first
          and read back after

The cache (n sequences, h kv heads, L rows, D dims; groups of 32 dims share a step and a low value, both fp16):
  k_codes uint8 [n, h, L, D/2]            element d of a row in byte d/2, even d in the low 4 bits
  k_meta  fp16  [n, h, L, D/32, 2]        step, low
  v_codes uint8 [n, h, L/8, D/4, 16]      row t, element d in byte 2 (t % 8) + (d % 4) / 2, even d in the low 4 bits
  v_meta  fp16  [n, h, L/8, D/32, 2, 8]   the steps of 8 rows, then their lows
Code c stands for fp16(low + step c); low = fp16(min), step = (max - min) / 15 in fp16 rounded towards zero (so that
no finite value reads back as an infinity), c = the nearest code, ties to even.
"""

import random

import torch

own = False

DEV = 'cuda'
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}
GROUP = 32


def listed():
    return [
        # the 4 prompt tokens of one clip: the smallest call, latency
        {'name': 'prompt_start', 'kind': 'prompt', 'n': 1, 'q': 4, 'q_min': 4, 'past': 0, 'keys': 0, 'heads': 20,
         'kv_heads': 20, 'dim': 64, 'type': 'fp16', 'causal': True, 'mix': 1},
        # 16 clips' prompts, each with up to 220 tokens of the text before
        {'name': 'prompt_text', 'kind': 'prompt', 'n': 16, 'q': 224, 'q_min': 4, 'past': 0, 'keys': 0, 'heads': 20,
         'kv_heads': 20, 'dim': 64, 'type': 'fp16', 'causal': True, 'mix': 2},
        # the same prompts over the 1500 audio frames of their clips
        {'name': 'prompt_audio', 'kind': 'prompt', 'n': 16, 'q': 224, 'q_min': 4, 'past': 0, 'keys': 1500, 'heads': 20,
         'kv_heads': 20, 'dim': 64, 'type': 'fp16', 'causal': False, 'mix': 2},
        # prompts of very different lengths, some the continuation of one that was run before
        {'name': 'prompt_packed', 'kind': 'prompt', 'n': 12, 'q': 4096, 'q_min': 1, 'past': 1000, 'keys': 0,
         'heads': 16, 'kv_heads': 4, 'dim': 64, 'type': 'fp16', 'causal': True, 'mix': 3},
        # one long prompt of a model with grouped heads
        {'name': 'prompt_long', 'kind': 'prompt', 'n': 1, 'q': 8192, 'q_min': 8192, 'past': 0, 'keys': 0, 'heads': 32,
         'kv_heads': 8, 'dim': 128, 'type': 'bf16', 'causal': True, 'mix': 4},
        # one token of each of 16 lanes
        {'name': 'cache_token', 'kind': 'cache', 'n': 16, 'q': 1, 'q_min': 1, 'max_len': 448, 'kv_heads': 20,
         'dim': 64, 'type': 'fp16', 'mix': 5},
        # the cross keys and values of 8 clips, one layer
        {'name': 'cache_audio', 'kind': 'cache', 'n': 8, 'q': 1500, 'q_min': 1500, 'max_len': 1504, 'kv_heads': 20,
         'dim': 64, 'type': 'fp16', 'mix': 6},
        # long ragged prompts
        {'name': 'cache_long', 'kind': 'cache', 'n': 6, 'q': 16000, 'q_min': 100, 'max_len': 16384, 'kv_heads': 8,
         'dim': 128, 'type': 'bf16', 'mix': 7},
        # self attention of one clip's next token
        {'name': 'decode_self', 'kind': 'decode', 'n': 1, 'len': 300, 'len_min': 300, 'max_len': 448, 'heads': 20,
         'kv_heads': 20, 'dim': 64, 'type': 'fp16', 'fresh': True, 'mix': 8},
        # cross attention of 16 lanes
        {'name': 'decode_audio', 'kind': 'decode', 'n': 16, 'len': 1500, 'len_min': 1500, 'max_len': 1504, 'heads': 20,
         'kv_heads': 20, 'dim': 64, 'type': 'fp16', 'fresh': False, 'mix': 9},
        # 64 sequences of very different lengths, grouped heads
        {'name': 'decode_batch', 'kind': 'decode', 'n': 64, 'len': 8000, 'len_min': 1, 'max_len': 8192, 'heads': 32,
         'kv_heads': 8, 'dim': 128, 'type': 'bf16', 'fresh': True, 'mix': 10},
        # one sequence with a long cache
        {'name': 'decode_long', 'kind': 'decode', 'n': 1, 'len': 131000, 'len_min': 131000, 'max_len': 131072,
         'heads': 64, 'kv_heads': 8, 'dim': 128, 'type': 'fp16', 'fresh': False, 'mix': 11},
    ]


def _log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(['prompt', 'prompt', 'cache', 'decode', 'decode'])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 20])
    group = rng.choice([1, 1, 2, 4, 5, 8, 16])
    case = {'kind': kind, 'kv_heads': kv_heads, 'dim': dim, 'type': rng.choice(['fp16', 'bf16']),
            'mix': rng.randrange(1 << 20)}
    if kind == 'prompt':
        # at most 128 Mi scores and 32 heads, so a drawn case stays below the long prompt
        q = _log_int(rng, 1, 4096)
        n = _log_int(rng, 1, max(1, min(64, 16384 // q)))
        past = rng.choice([0, 0, _log_int(rng, 1, 2048)])
        causal = rng.random() < 0.7
        keys = 0 if causal else _log_int(rng, 1, 4096)
        while n * q * (keys or q + past) > 128 << 20:
            n = n // 2 if n > 1 else n
            q = q if n > 1 else q * 3 // 4
        return {**case, 'n': n, 'q': q, 'q_min': _log_int(rng, 1, q), 'past': past if causal else 0, 'keys': keys,
                'heads': kv_heads * group if kv_heads * group <= 32 else kv_heads, 'causal': causal}
    if kind == 'cache':
        q = _log_int(rng, 1, 16000)
        n = _log_int(rng, 1, max(1, min(64, 96000 // q)))
        return {**case, 'n': n, 'q': q, 'q_min': _log_int(rng, 1, q), 'kv_heads': min(kv_heads, 8) if n * q > 20000 else kv_heads,
                'max_len': (q + rng.randrange(200)) // 32 * 32 + 32}
    length = _log_int(rng, 1, 130000)
    n = _log_int(rng, 1, max(1, min(64, 262144 // length)))
    return {**case, 'n': n, 'len': length, 'len_min': _log_int(rng, 1, length), 'max_len': length // 32 * 32 + 32,
            'kv_heads': min(kv_heads, 8) if n * length > 50000 else kv_heads,
            'heads': (min(kv_heads, 8) if n * length > 50000 else kv_heads) * group, 'fresh': rng.random() < 0.5}


# ---- inputs ---------------------------------------------------------------------------------


def _lengths(case, high, low):
    """n lengths between low and high, spread over their logarithm, the longest first or last by chance."""
    rng = random.Random(case['mix'])
    some = [high] + [_log_int(rng, low, high) for _ in range(case['n'] - 1)]
    rng.shuffle(some)
    return some


def _prompt_lengths(case):
    """Query and key counts of the sequences."""
    nq = _lengths(case, case['q'], case['q_min'])
    rng = random.Random(case['mix'] + 1)
    return nq, [case['keys'] or x + (rng.randrange(case['past'] + 1) if case['past'] else 0) for x in nq]


def _starts(lengths):
    cu = [0]
    for x in lengths:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int64, device=DEV)


def _normal(gen, shape, kind):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(kind)


def _keys(gen, shape, kind):
    """Keys and values: a level of its own for each head dim, as projections with a bias have, plus noise."""
    level = torch.randn(shape[-2:], generator=gen, device=DEV)
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).add_(level).to(kind)


def _empty_cache(n, heads, max_len, dim):
    zeros = lambda *shape, kind=torch.float16: torch.zeros(shape, dtype=kind, device=DEV)  # noqa: E731
    return (zeros(n, heads, max_len, dim // 2, kind=torch.uint8), zeros(n, heads, max_len, dim // GROUP, 2),
            zeros(n, heads, max_len // 8, dim // 4, 16, kind=torch.uint8),
            zeros(n, heads, max_len // 8, dim // GROUP, 2, 8))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, dim, n, kv_heads = TYPES[case['type']], case['dim'], case['n'], case['kv_heads']
    s = {'kind': case['kind'], 'scale': dim ** -0.5}
    if case['kind'] == 'prompt':
        nq, nk = _prompt_lengths(case)
        s.update(cu_q=_starts(nq), cu_k=_starts(nk), max_q=max(nq), max_k=max(nk), causal=case['causal'],
                 q=_normal(gen, (sum(nq), case['heads'], dim), kind), k=_keys(gen, (sum(nk), kv_heads, dim), kind),
                 v=_keys(gen, (sum(nk), kv_heads, dim), kind))
        s['out'] = torch.empty_like(s['q'])
    elif case['kind'] == 'cache':
        rows = _lengths(case, case['q'], case['q_min'])
        rng = random.Random(case['mix'] + 1)
        s.update(cu=_starts(rows), k=_keys(gen, (sum(rows), kv_heads, dim), kind),
                 v=_keys(gen, (sum(rows), kv_heads, dim), kind),
                 pos=torch.tensor([rng.randrange(case['max_len'] - x + 1) for x in rows], dtype=torch.int64, device=DEV),
                 cache=_empty_cache(n, kv_heads, case['max_len'], dim))
        s['k_out'], s['v_out'] = torch.empty_like(s['k']), torch.empty_like(s['v'])
    else:
        lens = _lengths(case, case['len'], case['len_min'])
        if case['fresh']:
            lens = [min(x, case['max_len'] - 1) for x in lens]
        s['cache'] = _empty_cache(n, kv_heads, case['max_len'], dim)
        for which in (0, 1):  # one head's rows at a time: the cache may be large
            for h in range(kv_heads):
                x = _keys(gen, (n, case['max_len'], 1, dim), kind)[:, :, 0]
                step, low, codes = _quantise(x)
                if which == 0:
                    s['cache'][0][:, h] = _bytes(codes)
                    s['cache'][1][:, h] = torch.stack([step, low], -1)
                else:
                    s['cache'][2][:, h] = _bytes(codes).view(n, -1, 8, dim // 4, 2).transpose(2, 3).reshape(n, -1, dim // 4, 16)
                    s['cache'][3][:, h] = torch.stack([step, low], -1).view(n, -1, 8, dim // GROUP, 2).permute(0, 1, 3, 4, 2)
        s.update(q=_normal(gen, (n, case['heads'], dim), kind), fresh=case['fresh'],
                 lens=torch.tensor(lens, dtype=torch.int64, device=DEV))
        if case['fresh']:
            s.update(k=_keys(gen, (n, kv_heads, dim), kind), v=_keys(gen, (n, kv_heads, dim), kind),
                     each=torch.arange(n + 1, dtype=torch.int64, device=DEV))
            s['k_out'], s['v_out'] = torch.empty_like(s['k']), torch.empty_like(s['v'])
        s['out'] = torch.empty_like(s['q'])
    return s


# ---- the plain form ---------------------------------------------------------------------------


def _half_down(x):
    """x >= 0 in fp16, rounded towards zero."""
    near = x.half()
    return torch.where(near.to(x.dtype) > x, (near.view(torch.int16) - 1).view(torch.float16), near)


def _quantise(x):
    """(step, low) fp16 [..., D/32] and codes uint8 [..., D] of rows x [..., D]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    high, low = g.amax(-1), g.amin(-1)
    step, low = _half_down((high - low) * (1 / 15)), low.half()
    divisor = torch.where(step > 0, step, 1.0).float()  # a group of one value: code 0
    codes = ((g - low.float().unsqueeze(-1)) / divisor.unsqueeze(-1)).round_().clamp_(0, 15)
    return step, low, codes.to(torch.uint8).flatten(-2)


def _bytes(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(data, step, low):
    """What codes [..., D/2 bytes] with their groups' steps and lows stand for: fp16 values, as fp32."""
    codes = torch.stack([data & 15, data >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    return (codes.mul_(step.float().unsqueeze(-1)).add_(low.float().unsqueeze(-1))).half().flatten(-2).float()


def _softmax_product(scores, seen, v):
    """Softmax over the keys that are seen (none: zero) times v; scores [..., rows, keys], v [..., keys, dim]."""
    scores.masked_fill_(~seen, float('-inf'))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == float('-inf'), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, 1.0, total)


def _row_of(cu, total):
    """For each packed row its sequence and its place in it."""
    row = torch.arange(total, device=DEV)
    seq = torch.bucketize(row, cu[1:], right=True)
    return seq, row - cu[seq]


def _plain_prompt(s):
    q, k, v, cu_q, cu_k = s['q'], s['k'], s['v'], s['cu_q'], s['cu_k']
    (_, heads, dim), kv_heads, n = q.shape, k.size(1), cu_q.numel() - 1
    i, j = torch.arange(s['max_q'], device=DEV), torch.arange(s['max_k'], device=DEV)
    nq, nk = cu_q.diff()[:, None], cu_k.diff()[:, None]
    qp = q[(cu_q[:-1, None] + i).clamp(max=q.size(0) - 1)].float()  # [n, rows, heads, dim]
    at = (cu_k[:-1, None] + j).clamp(max=k.size(0) - 1)
    kp, vp = k[at].float(), v[at].float()
    qp = qp.view(n, -1, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, -1, dim)
    kp = kp.permute(0, 2, 3, 1).reshape(n * kv_heads, dim, -1).contiguous()
    vp = vp.permute(0, 2, 1, 3).reshape(n * kv_heads, -1, dim).contiguous()
    seen = (j < nk)[:, None, :]
    if s['causal']:
        seen = seen & (j <= i[:, None] + (nk - nq)[:, :, None])
    scores = torch.bmm(qp * s['scale'], kp).view(n, kv_heads, heads // kv_heads, s['max_q'], s['max_k'])
    o = _softmax_product(scores, seen[:, None, None], vp.view(n, kv_heads, 1, -1, dim))
    seq, place = _row_of(cu_q, q.size(0))
    return o.flatten(1, 2)[seq, :, place].to(q.dtype)


def _plain_append(cache, k, v, seq, row):
    (step, low, codes), dim = _quantise(k), k.size(-1)
    cache[0][seq, :, row] = _bytes(codes)
    cache[1][seq, :, row] = torch.stack([step, low], -1)
    step, low, codes = _quantise(v)
    v_codes = cache[2].view(*cache[2].shape[:3], dim // 4, 8, 2)
    v_codes[seq, :, row // 8, :, row % 8] = _bytes(codes).unflatten(-1, (-1, 2))
    cache[3][seq, :, row // 8, :, :, row % 8] = torch.stack([step, low], -1)


def _plain_read(cache, seq, row, kind):
    dim = cache[0].size(-1) * 2
    meta = cache[1][seq, :, row]
    k = _values(cache[0][seq, :, row], meta[..., 0], meta[..., 1])
    data = cache[2].view(*cache[2].shape[:3], dim // 4, 8, 2)[seq, :, row // 8, :, row % 8].flatten(-2)
    meta = cache[3][seq, :, row // 8, :, :, row % 8]
    return k.to(kind), _values(data, meta[..., 0], meta[..., 1]).to(kind)


def _plain_cache(s):
    seq, place = _row_of(s['cu'], s['k'].size(0))
    row = s['pos'][seq] + place
    _plain_append(s['cache'], s['k'], s['v'], seq, row)
    return _plain_read(s['cache'], seq, row, s['k'].dtype)


def _plain_decode(s):
    q, cache, lens = s['q'], s['cache'], s['lens']
    (n, heads, dim), kv_heads = q.shape, cache[0].size(1)
    if s['fresh']:
        seq = torch.arange(n, device=DEV)
        _plain_append(cache, s['k'], s['v'], seq, lens)
        rows = _plain_read(cache, seq, lens, q.dtype)
        lens = lens + 1
    max_len = cache[0].size(2)
    k = _values(cache[0], cache[1][..., 0], cache[1][..., 1])
    data = cache[2].view(n, kv_heads, max_len // 8, dim // 4, 8, 2).transpose(3, 4).reshape(n, kv_heads, max_len, dim // 2)
    meta = cache[3].permute(0, 1, 2, 5, 3, 4).reshape(n, kv_heads, max_len, dim // GROUP, 2)
    v = _values(data, meta[..., 0], meta[..., 1])
    scores = (q.float() * s['scale']).view(n, kv_heads, heads // kv_heads, dim) @ k.transpose(2, 3).contiguous()
    seen = torch.arange(max_len, device=DEV) < lens[:, None, None, None]
    o = _softmax_product(scores, seen, v).view(n, heads, dim).to(q.dtype)
    return (o, *rows) if s['fresh'] else o


def run(s):
    if own:
        from flash_whisper_amd.ext import load_ext

        ext = load_ext()
        if s['kind'] == 'prompt':
            ext.prompt_attention(s['q'], s['k'], s['v'], s['out'], s['cu_q'], s['cu_k'], s['scale'], s['causal'])
            return s['out']
        if s['kind'] == 'cache':
            ext.kv_q4_append(s['k'], s['v'], s['cu'], s['pos'], s['cache'])
            ext.kv_q4_read(s['cache'], s['cu'], s['pos'], s['k_out'], s['v_out'])
            return s['k_out'], s['v_out']
        if 'ws' not in s:  # a decoding stream keeps its workspace
            s['ws'] = ext.decode_attention_q4_workspace(s['q'].size(0), s['q'].size(1), s['cache'])
        if s['fresh']:
            ext.decode_attention_q4(s['q'], s['cache'], s['lens'], s['out'], s['ws'], s['scale'], s['k'], s['v'])
            ext.kv_q4_read(s['cache'], s['each'], s['lens'], s['k_out'], s['v_out'])
            return s['out'], s['k_out'], s['v_out']
        ext.decode_attention_q4(s['q'], s['cache'], s['lens'], s['out'], s['ws'], s['scale'])
        return s['out']
    return {'prompt': _plain_prompt, 'cache': _plain_cache, 'decode': _plain_decode}[s['kind']](s)


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    kv_heads, dim = case['kv_heads'], case['dim']
    held = kv_heads * (dim // 2 + dim // GROUP * 4)  # one cached row of K or of V
    if case['kind'] == 'prompt':
        nq, nk = _prompt_lengths(case)
        pairs = sum(a * b - (min(a, b) * (min(a, b) - 1) // 2 + max(0, a - b) * b if case['causal'] else 0)
                    for a, b in zip(nq, nk))
        return {'bytes': 2 * dim * (2 * sum(nq) * case['heads'] + 2 * sum(nk) * kv_heads),
                'flops': 4 * dim * pairs * case['heads']}
    if case['kind'] == 'cache':  # values in, cache out and in again, values out
        rows = sum(_lengths(case, case['q'], case['q_min']))
        return {'bytes': rows * 2 * (2 * 2 * dim * kv_heads + 2 * held), 'flops': rows * 2 * kv_heads * dim * 8}
    lens = [min(x, case['max_len'] - case['fresh']) for x in _lengths(case, case['len'], case['len_min'])]
    n, keys = case['n'], sum(lens) + case['n'] * case['fresh']
    # queries in and out, the cached rows; a fresh row in, written to the cache, and read back
    return {'bytes': 4 * n * case['heads'] * dim + 2 * keys * held + (n * 2 * (4 * kv_heads * dim + held) if case['fresh'] else 0),
            'flops': 4 * dim * keys * case['heads']}


# ---- the definition in 64 bits --------------------------------------------------------------------


def _attend64(q, k, v, scale, causal):
    """One sequence: q [rows, heads, dim], k and v [keys, kv_heads, dim], all float64."""
    out = torch.zeros_like(q)
    rows, keys, group = q.size(0), k.size(0), q.size(1) // k.size(1)
    if not keys:
        return out
    hidden = None
    if causal:
        hidden = torch.ones(rows, keys, dtype=torch.bool, device=DEV).triu(1 + keys - rows)
    for h in range(q.size(1)):
        s = q[:, h] @ k[:, h // group].T.contiguous() * scale
        if hidden is not None:
            s[hidden] = float('-inf')
        # rows without a key: softmax gives NaN there, the operator 0
        out[:, h] = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) @ v[:, h // group].contiguous()
    return out


def _held64(x):
    """The values that the cache holds for rows x [..., D]."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    low = g.min(-1, keepdim=True).values
    wide = (g.max(-1, keepdim=True).values - low) / 15
    last = torch.exp2((torch.frexp(wide).exponent - 1).clamp(min=-14).double() - 10)  # fp16's last place
    step = torch.floor(wide / last) * last
    low = low.to(torch.float16).double()
    code = torch.round((g - low) / torch.where(step == 0, torch.ones_like(step), step)).clamp(0, 15)
    code = torch.where(step == 0, torch.zeros_like(code), code)
    return (low + step * code).to(torch.float16).double().reshape(x.shape)


def _read64(cache, seq, head, rows):
    """K and V rows [0, rows) of one sequence and head, from the layout's definition."""
    k_codes, k_meta, v_codes, v_meta = (c[seq, head] for c in cache)
    t, d = torch.arange(rows, device=DEV)[:, None], torch.arange(2 * k_codes.size(-1), device=DEV)[None]
    shift = 4 * (d % 2)
    code = (k_codes[t, d // 2].long() >> shift) & 15
    k = k_meta[t, d // GROUP, 1].double() + k_meta[t, d // GROUP, 0].double() * code
    code = (v_codes[t // 8, d // 4, 2 * (t % 8) + (d % 4) // 2].long() >> shift) & 15
    v = v_meta[t // 8, d // GROUP, 1, t % 8].double() + v_meta[t // 8, d // GROUP, 0, t % 8].double() * code
    return k.to(torch.float16).double(), v.to(torch.float16).double()


def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] == 'prompt':
        out = torch.zeros(s['q'].shape, dtype=torch.float64, device=DEV)
        cq, ck = s['cu_q'].tolist(), s['cu_k'].tolist()
        for a, b, c, d in zip(cq, cq[1:], ck, ck[1:]):
            out[a:b] = _attend64(s['q'][a:b].double(), s['k'][c:d].double(), s['v'][c:d].double(), s['scale'], s['causal'])
        return out
    if case['kind'] == 'cache':
        return _held64(s['k']), _held64(s['v'])
    kv_heads, group = case['kv_heads'], case['heads'] // case['kv_heads']
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device=DEV)
    fresh = (_held64(s['k']), _held64(s['v'])) if case['fresh'] else None
    for seq, length in enumerate(s['lens'].tolist()):
        for h in range(kv_heads):
            k, v = _read64(s['cache'], seq, h, length)
            if fresh:
                k, v = torch.cat([k, fresh[0][seq, h][None]]), torch.cat([v, fresh[1][seq, h][None]])
            q = s['q'][seq, h * group:(h + 1) * group].double()[None]
            out[seq, h * group:(h + 1) * group] = _attend64(q, k[:, None], v[:, None], s['scale'], False)[0]
    return (out, *fresh) if fresh else out
