"""TEST INFRASTRUCTURE ONLY: a decode worker's step from its definition, in numpy
and 64 bits. The product never imports it."""
from __future__ import annotations

import numpy as np

INT32_MAX = 2 ** 31 - 1


def tables(pages, starts, cached, new, block_size, max_blocks, max_tokens):
    """(block_tables, seq_lens, token_starts, slots, positions) of a step, request by request."""
    batch = len(cached)
    new = [1] * batch if new is None else [int(n) for n in new]
    table = np.full((batch, max_blocks), -1, np.int64)
    lens = np.full(batch, -1, np.int64)
    first = np.zeros(batch + 1, np.int64)
    slots, positions = np.full(max_tokens, -1, np.int64), np.full(max_tokens, -1, np.int64)
    at = 0
    for b in range(batch):
        c, n, lo, hi = int(cached[b]), new[b], int(starts[b]), int(starts[b + 1])
        listed = 0 <= lo <= hi <= len(pages)
        mine = [int(x) for x in pages[lo:hi]] if listed else []
        table[b, :min(len(mine), max_blocks)] = mine[:max_blocks]
        rows = max(n, 0)
        need = -(-(c + n) // block_size) if c + n > 0 else 0
        ok = listed and c >= 0 and n >= 0 and c + n <= INT32_MAX and need <= min(len(mine), max_blocks) and at + rows <= max_tokens
        first[b] = min(at, INT32_MAX)
        if ok:
            lens[b] = c + n
            for i in range(rows):
                page, off = mine[(c + i) // block_size], (c + i) % block_size
                positions[at + i] = c + i
                slots[at + i] = page * block_size + off if page >= 0 and page * block_size + off <= INT32_MAX else -1
        at += rows
    first[batch] = min(at, INT32_MAX)
    return tuple(x.astype(np.int32) for x in (table, lens, first, slots, positions))


def norm_rope(x, weight, eps, line, rotary, pairs):
    """Heads x[heads][dim] of one token, normed (weight None: not) and turned by
    line[rotary] (cosines, then sines); and the sum of the magnitudes that went
    into each result, for error bounds."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    out, size = x.copy(), np.abs(x)
    n = rotary // 2
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + n)
        c, s = float(line[i]), float(line[n + i])
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a], size[..., b] = abs(x[..., a] * c) + abs(x[..., b] * s), abs(x[..., b] * c) + abs(x[..., a] * s)
    return out, size
