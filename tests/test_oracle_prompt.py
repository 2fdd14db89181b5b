"""The oracles of the prompt readers and the page movers: attention against torch in 64
bits, and what must hold of any fork or compaction."""
import numpy as np
import pytest
import torch

from oracle import pages as O
from oracle import prompt as A


@pytest.mark.parametrize("n,length,heads,group", [(1, 1, 1, 1), (5, 5, 2, 3), (3, 20, 1, 7), (17, 33, 2, 1)])
def test_attention_is_torchs(n, length, heads, group):
    rng = np.random.default_rng(n)
    q, k, v = (rng.standard_normal(s) for s in ((n, heads * group, 64), (length, heads, 64), (length, heads, 64)))
    t = lambda x, r: torch.from_numpy(x).transpose(0, 1).repeat_interleave(r, 0)  # noqa: E731
    mask = torch.arange(length)[None] <= torch.arange(n)[:, None] + length - n
    want = torch.nn.functional.scaled_dot_product_attention(t(q, 1), t(k, group), t(v, group), mask).transpose(0, 1).numpy()
    np.testing.assert_allclose(A.attend(q, k, v)[0], want, rtol=1e-12, atol=1e-12)


def test_rows_that_see_nothing_and_keys_that_nobody_sees():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal(s) for s in ((6, 1, 8), (4, 1, 8), (4, 1, 8)))
    k[3] = v[3] = np.nan          # seen by the last query only
    out = A.attend(q, k, v)[0]
    assert (out[:2] == 0).all() and np.isfinite(out[2:5]).all() and np.isnan(out[5]).all()


@pytest.mark.parametrize("seed", range(6))
def test_forks_share_whole_pages_only_and_take_what_nobody_holds(seed):
    rng = np.random.default_rng(seed)
    n_pages, block, width, stride = 60, 4, 9, 3
    lens = rng.integers(0, 25, 5)
    order, tables = list(rng.permutation(n_pages)), np.full((5, width), -1, np.int32)
    for i, n in enumerate(lens):
        tables[i, : -(-n // block)] = [order.pop() * stride for _ in range(-(-n // block))]
    parents, new = rng.integers(-1, 5, 8), rng.integers(0, 9, 8)
    reserved = rng.random(n_pages) < 0.2
    out, out_lens, counts, copies = O.fork(tables, lens, parents, new, n_pages, stride, block, reserved)
    held = {int(e) for p in set(parents[parents >= 0].tolist()) for e in tables[p] if e >= 0}
    written = []
    for i, p in enumerate(parents):
        if p < 0 or out_lens[i] < 0:
            assert (out[i] == -1).all()
            continue
        n, whole = int(lens[p]), int(lens[p]) // block
        assert out_lens[i] == n and (out[i] >= 0).sum() == -(-(n + int(new[i])) // block)
        np.testing.assert_array_equal(out[i, :whole], tables[p, :whole])
        written += [int(e) for e in out[i, whole:] if e >= 0]
    assert len(set(written)) == len(written)           # no page that two rows write to
    fresh = set(written) - held
    assert not any(reserved[e // stride] for e in fresh)
    assert all(b * stride in fresh and a * stride in held for a, b in copies)


@pytest.mark.parametrize("seed", range(6))
def test_compacted_pages_keep_their_contents(seed):
    rng = np.random.default_rng(seed)
    n_pages, stride = 40, 2
    tables = rng.integers(-1, n_pages, (4, 6)).astype(np.int32) * stride
    reserved = rng.random(n_pages) < 0.3
    out, moved, counts, moves = O.compact(tables, n_pages, stride, reserved)
    pages = np.arange(n_pages)
    for a, b in moves:
        pages[b] = a
    used = sorted({int(e) // stride for e in tables.ravel() if e >= 0})
    for old, new in zip(tables.ravel(), out.ravel()):
        assert new == old if old < 0 else pages[new // stride] == old // stride
    free = [p for p in range(n_pages) if not reserved[p]]
    movable = [p for p in used if not reserved[p]]
    assert sorted(moved[p] for p in movable) == free[: len(movable)] and all(moved[p] == p for p in used if reserved[p])
    assert counts.tolist() == [len(movable), len(moves)]
