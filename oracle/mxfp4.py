"""TEST INFRASTRUCTURE ONLY: MXFP4 pages from their definition, in numpy and 64
bits. The product never imports it.

A value is an E2M1 code times the power of two its group of 32 dims shares
(E8M0, 255 = NaN). Addresses are written out per element from the page layout:
codes of a head in a block of 16 tokens as [quarter of the dims][token][dim/8
bytes] for K and [quad of tokens][column of dim/16 dims][token][dim/32 bytes]
for V, scales as [group of 32 dims][token].
"""
from __future__ import annotations

import numpy as np

TOKENS, GROUP = 16, 32
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def quantise(x):
    """(codes, scales) of rows x[..., dim]: one code and one E8M0 byte an element / group."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    finite = np.isfinite(g).all(-1)
    top = np.abs(np.where(finite[..., None], g, 0.0)).max(-1)
    # frexp: top = m * 2^e with m in [0.5, 1), so floor(log2 top) = e - 1
    e = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127)
    scales = np.where(finite, np.clip(e + 127, 0, 254), 255).astype(np.uint8)
    y = np.abs(np.where(finite[..., None], g, 0.0)) * np.exp2(127.0 - scales.astype(np.float64))[..., None]
    far = np.abs(y[..., None] - E2M1)  # exact: differences of few-bit numbers
    best = far.min(-1, keepdims=True)
    tie = far == best
    even = np.array([i % 2 == 0 for i in range(8)])
    codes = np.where((tie & even).any(-1), (tie & even).argmax(-1), tie.argmax(-1)).astype(np.uint8)
    codes |= (np.signbit(g) << 3).astype(np.uint8)
    return codes.reshape(x.shape), scales


def values(codes, scales):
    """The doubles that codes [..., dim] and scales [..., dim/32] stand for."""
    v = np.where(codes & 8, -E2M1[codes & 7], E2M1[codes & 7])
    g = v.reshape(*v.shape[:-1], -1, GROUP)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (g * s[..., None]).reshape(codes.shape)


def half_bytes(heads, dim):
    return TOKENS * heads * dim // 2


def code_at(slots, heads, dim, is_value):
    """Byte of the pool that holds the code of each slot, head and dim."""
    s = np.asarray(slots, np.int64)[:, None, None]
    h = np.arange(heads, dtype=np.int64)[None, :, None]
    d = np.arange(dim, dtype=np.int64)[None, None, :]
    block, t = s // TOKENS, s % TOKENS
    base = block * half_bytes(heads, dim) + h * (TOKENS * dim // 2)
    if is_value:
        wide = dim // 16
        return base + ((t // 4 * 16 + d // wide) * 4 + t % 4) * (dim // 32) + d % wide // 2
    wide = dim // 4
    return base + (d // wide * TOKENS + t) * (dim // 8) + d % wide // 2


def scale_at(slots, heads, dim):
    s = np.asarray(slots, np.int64)[:, None, None]
    h = np.arange(heads, dtype=np.int64)[None, :, None]
    g = np.arange(dim // GROUP, dtype=np.int64)[None, None, :]
    return s // TOKENS * (half_bytes(heads, dim) // 16) + (h * (dim // GROUP) + g) * TOKENS + s % TOKENS


def put(pool, scales, slots, codes, sc, is_value):
    """Stores rows' codes [n][heads][dim] and scales into a pool, in place."""
    n, heads, dim = codes.shape
    at = code_at(slots, heads, dim, is_value)
    low, high = codes[..., 0::2], codes[..., 1::2]
    pool[at[..., 0::2]] = low | high << 4
    scales[scale_at(slots, heads, dim)] = sc


def get(pool, scales, slots, heads, dim, is_value):
    """Rows of slots as doubles [n][heads][dim]."""
    raw = pool[code_at(slots, heads, dim, is_value)]
    codes = np.where(np.arange(dim) % 2 == 1, raw >> 4, raw & 15).astype(np.uint8)
    return values(codes, scales[scale_at(slots, heads, dim)])


def decode(q, pools, tables, seq_lens, heads):
    """Attention of one query token per sequence in 64 bits: (out, spread, size,
    reach), each [batch][q_heads][dim] (reach without dim). spread = sum w |v -
    out| and size = sum w |v| with w the softmax weights, reach the largest sum
    |q k| / sqrt(dim): what error bounds are made of. q [batch][q_heads][dim];
    pools (k, v, k_scales, v_scales). A zero length gives zeros."""
    batch, q_heads, dim = q.shape
    group = q_heads // heads
    out, spread, size = (np.zeros((batch, q_heads, dim)) for _ in range(3))
    reach = np.zeros((batch, q_heads))
    k_pool, v_pool, k_scales, v_scales = pools
    for b in range(batch):
        n = int(seq_lens[b])
        if n == 0:
            continue
        t = np.arange(n)
        slots = np.asarray(tables[b], np.int64)[t // TOKENS] * TOKENS + t % TOKENS
        k = get(k_pool, k_scales, slots, heads, dim, False)
        v = get(v_pool, v_scales, slots, heads, dim, True)
        for h in range(q_heads):
            qh, kh, vh = q[b, h].astype(np.float64), k[:, h // group], v[:, h // group]
            s = kh @ qh / np.sqrt(dim)
            p = np.exp(s - s.max())
            w = p / p.sum()
            out[b, h] = w @ vh
            spread[b, h] = w @ np.abs(vh - out[b, h])
            size[b, h] = w @ np.abs(vh)
            reach[b, h] = (np.abs(kh) @ np.abs(qh)).max() / np.sqrt(dim)
    return out, spread, size, reach
