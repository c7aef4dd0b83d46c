"""A key/value cache in pages and the rules on logits from their definitions (numpy; float64 where numbers are computed)."""

import numpy as np

from . import serving


def page_map(pos, cu, table, held, own, stack, count, rows, page):
    """The sequences one after another, page by page; `rows`: packed rows there are. Returns table, held, stack, [pages on
    the stack, pages missing], slots (None where a row is in no sequence)."""
    table, held, stack = np.array(table), [int(x) for x in held], [int(x) for x in stack]
    n, width = table.shape
    count, missing, slots = int(count), 0, [None] * rows
    cu = [min(max(int(x), 0), rows) for x in cu]
    last = [int(p) + b - a for p, a, b in zip(pos, cu, cu[1:])]
    for s in range(n):
        pages = -(-last[s] // page)
        if pos[s] >= 0 and pages < held[s]:
            for j in range(max(pages, 0 if own is None else int(own[s])), held[s]):
                stack[count] = int(table[s, j])
                count += 1
            held[s] = pages
    for s in range(n):
        for j in range(held[s], -(-last[s] // page) if pos[s] >= 0 else 0):
            if j < width and count:
                count -= 1
                table[s, j] = stack[count]
                held[s] = j + 1
            else:
                missing += 1
        for i in range(cu[s + 1] - cu[s]):
            row = int(pos[s]) + i
            there = pos[s] >= 0 and row // page < held[s]
            slots[cu[s] + i] = int(table[s, row // page]) * page + row % page if there else -1
    return table, held, stack, [count, missing], slots


def append(k_pages, v_pages, k, v, slots):
    """Rows k, v [rows, heads, dim] into copies of the pages."""
    k_pages, v_pages = k_pages.copy(), v_pages.copy()
    page = k_pages.shape[2]
    for r, slot in enumerate(slots):
        if 0 <= slot < k_pages.shape[0] * page:
            k_pages[slot // page, :, slot % page] = k[r]
            v_pages[slot // page, :, slot % page // 8, :, slot % 8] = v[r]
    return k_pages, v_pages


def rows_of(k_pages, v_pages, table, n):
    """The first n rows of a sequence: k, v [rows, heads, dim], without those of pages that there are not."""
    page, rows = k_pages.shape[2], np.arange(n)
    at = table[rows // page]
    rows = rows[(at >= 0) & (at < len(k_pages))]
    at = table[rows // page]
    return k_pages[at, :, rows % page], v_pages[at, :, rows % page // 8, :, rows % 8]


def attend(q, k_pages, v_pages, table, lens, scale):
    """For each sequence of q [n, heads, dim]: what serving.attend returns, its keys and the largest |v|."""
    for s in range(len(q)):
        n = min(max(int(lens[s]), 0), table.shape[1] * k_pages.shape[2])
        k, v = rows_of(k_pages, v_pages, table[s], n)
        yield (*serving.attend(q[s][None], k, v, scale, False), len(k), np.abs(v[np.isfinite(v)]).max(initial=0))


def rules(x, tokens=None, cu=None, prompt=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None,
          cu_bias=None, masks=None, mask_of=None):
    """The logits x [rows, vocab] (float64) under the rules, and what their fp32 roundings are relative to."""
    x = np.array(x, np.float64)
    size = np.abs(x)
    rows, vocab = x.shape
    for r in range(rows):
        if tokens is not None:
            mine = tokens[cu[r]:cu[r + 1]]
            new = mine[(0 if prompt is None else max(int(prompt[r]), 0)):]
            met = np.unique(mine[(mine >= 0) & (mine < vocab)])
            rep = 1.0 if repetition is None else float(repetition[r])
            y = x[r, met]
            x[r, met] = np.where(y > 0, y / rep, y * rep)
            size[r, met] += np.abs(x[r, met])
            made, count = np.unique(new[(new >= 0) & (new < vocab)], return_counts=True)
            f = 0.0 if frequency is None else float(frequency[r])
            p = 0.0 if presence is None else float(presence[r])
            x[r, made] -= f * count + p
            size[r, made] += abs(f) * count + abs(p)
        if bias_ids is not None:
            for i, b in {int(i): float(b) for i, b in zip(bias_ids[cu_bias[r]:cu_bias[r + 1]], bias[cu_bias[r]:cu_bias[r + 1]])}.items():
                if 0 <= i < vocab:
                    x[r, i] += b
                    size[r, i] += abs(b)
        if masks is not None:
            of = int(mask_of[r]) if mask_of is not None else 0 if len(masks) == 1 else r
            if 0 <= of < len(masks):
                bits = masks[of].view(np.uint32)[np.arange(vocab) // 32] >> (np.arange(vocab) % 32).astype(np.uint32)
                x[r, bits & 1 == 0] = -np.inf
    return x, size
