"""The attention over packed prompts and the 4-bit key/value cache from their definitions, in float64 (numpy)."""

import numpy as np

GROUP = 32


def attend(q, k, v, scale, causal):
    """One sequence: q [rows, heads, dim] over k, v [keys, kv_heads, dim]; query i sees the keys j <= i + keys - rows
    (causal) or all. Returns the output, and per element sum_j w_j |v_j| and, per row and head,
    max_j scale sum_d |q_d k_d| over the keys seen: what rounding errors of weights and scores are relative to."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    rows, heads, dim = q.shape
    keys, kv_heads, _ = k.shape
    out, spread, size = np.zeros_like(q), np.zeros_like(q), np.zeros((rows, heads))
    seen = np.ones((rows, keys), bool)
    if causal:
        seen = np.arange(keys)[None] <= np.arange(rows)[:, None] + keys - rows
    some = seen.any(1)
    for h in range(heads):
        kh, vh = k[:, h * kv_heads // heads], v[:, h * kv_heads // heads]
        if not some.any():
            continue
        with np.errstate(invalid='ignore', over='ignore'):
            s = np.where(seen, scale * (q[:, h] @ kh.T), -np.inf)[some]
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            # 0 x infinity where a key is not seen is nothing, not NaN
            finite = np.isfinite(vh)
            o = w @ np.where(finite, vh, 0.0)
            for j, d in np.argwhere(~finite):
                o[:, d] += np.where(seen[some][:, j], w[:, j] * vh[j, d], 0.0)
            out[some, h] = o
            spread[some, h] = w @ np.where(finite, np.abs(vh), 0.0)
            size[some, h] = np.where(seen, abs(scale) * (np.abs(q[:, h]) @ np.abs(kh).T), 0.0)[some].max(1)
    return out, spread, size


def half_down(x):
    """x >= 0 in fp16, rounded towards zero."""
    h = np.float16(x)
    return np.where(h.astype(x.dtype) > x, np.nextafter(h, np.float16(0)), h).astype(np.float16)


def quantise(x):
    """(step, low) fp16 [..., dim / 32] and codes uint8 [..., dim] of rows x [..., dim]."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(invalid='ignore', over='ignore', divide='ignore'):
        finite = (np.abs(g) < 65520).all(-1)  # what fp16 rounds to a number
        low32, high = g.min(-1), g.max(-1)
        step = np.where(finite, half_down(np.where(finite, (high - low32) * np.float32(1 / 15), 0)), np.float16(np.nan))
        low = np.float16(low32)
        s64, l64 = step.astype(np.float64)[..., None], low.astype(np.float64)[..., None]
        codes = np.rint((g.astype(np.float64) - l64) / np.where(s64 > 0, s64, np.inf))
    codes = np.where(np.isfinite(codes), codes, 0).clip(0, 15)
    return step.astype(np.float16), low, codes.astype(np.uint8).reshape(x.shape)


def values(step, low, codes):
    """What the codes stand for: fp16(low + step c), rounded once."""
    c = codes.astype(np.float64).reshape(*step.shape, GROUP)
    with np.errstate(invalid='ignore'):
        x = low.astype(np.float64)[..., None] + step.astype(np.float64)[..., None] * c
    return x.astype(np.float16).reshape(codes.shape)


def empty_cache(n, heads, max_len, dim, fill=0):
    """The cache's arrays, every byte `fill`."""
    b = lambda *shape: np.full((n, heads) + shape, fill, np.uint8)
    return (b(max_len, dim // 2), b(max_len, dim // GROUP, 4).view(np.float16).reshape(n, heads, max_len, dim // GROUP, 2),
            b(max_len // 8, dim // 4, 16),
            b(max_len // 8, dim // GROUP, 32).view(np.float16).reshape(n, heads, max_len // 8, dim // GROUP, 2, 8))


def write_row(cache, seq, row, k, v):
    """k, v [heads, dim] into one row of a sequence."""
    k_codes, k_meta, v_codes, v_meta = cache
    step, low, c = quantise(k)
    k_codes[seq, :, row] = c[:, 0::2] | c[:, 1::2] << 4
    k_meta[seq, :, row, :, 0], k_meta[seq, :, row, :, 1] = step, low
    step, low, c = quantise(v)
    for d in range(v.shape[1]):
        at = (seq, slice(None), row // 8, d // 4, 2 * (row % 8) + (d % 4) // 2)
        keep = v_codes[at] & (0xF0 if d % 2 == 0 else 0x0F)
        v_codes[at] = keep | c[:, d] << (4 * (d % 2))
    v_meta[seq, :, row // 8, :, 0, row % 8], v_meta[seq, :, row // 8, :, 1, row % 8] = step, low


def read_rows(cache, seq, rows):
    """The values of `rows` (indices) of a sequence: k, v fp16 [rows, heads, dim]."""
    k_codes, k_meta, v_codes, v_meta = (np.asarray(c)[seq] for c in cache)
    t, dim = np.asarray(rows, int)[:, None], 2 * k_codes.shape[-1]
    d = np.arange(dim)[None]
    k = (k_codes[:, t, d // 2] >> (4 * (d % 2))) & 15
    v = (v_codes[:, t // 8, d // 4, 2 * (t % 8) + (d % 4) // 2] >> (4 * (d % 2))) & 15
    g = np.arange(dim // GROUP)[None]
    k = values(k_meta[:, t, g, 0], k_meta[:, t, g, 1], k)
    v = values(v_meta[:, t // 8, g, 0, t % 8], v_meta[:, t // 8, g, 1, t % 8], v)
    return k.transpose(1, 0, 2), v.transpose(1, 0, 2)
