"""TEST INFRASTRUCTURE ONLY: attention of prompts in 64 bits: what pbe_prompt_attention and
pbe_paged_prompt_attention compute, from its definition.

Query i of a sequence's n queries, of `length` keys, sees keys 0 .. length - n + i.
"""
import numpy as np


def attend(q, k, v):
    """q [n][q_heads][dim], k and v [length][kv_heads][dim] of one sequence, in 64
    bits. Returns the outputs [n][q_heads][dim] and, for the bounds of a test, of each
    output sum w |v - o| and sum w |v| (w the softmax weights), and of each row
    [n][q_heads] the largest sum |q k| / sqrt(dim) of a key that it sees. A row that
    sees nothing is zeros; keys and values that a row does not see do not count,
    whatever they hold."""
    n, q_heads, dim = q.shape
    length, kv_heads, _ = k.shape
    group = q_heads // kv_heads
    out, spread, size = (np.zeros(q.shape) for _ in range(3))
    reach = np.zeros((n, q_heads))
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(n):
            seen = length - n + i + 1
            if seen <= 0:
                continue
            for h in range(q_heads):
                kk, vv = k[:seen, h // group], v[:seen, h // group]
                s = kk @ q[i, h] / np.sqrt(dim)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[i, h] = w @ vv
                spread[i, h] = w @ np.abs(vv - out[i, h])
                size[i, h] = w @ np.abs(vv)
                reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(dim)
    return out, spread, size, reach
