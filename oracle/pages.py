"""TEST INFRASTRUCTURE ONLY: the page movers from their definition, one row and
one page after another. The product never imports it."""
import numpy as np


def _page(entry, n_pages, stride):
    return entry // stride if entry >= 0 and entry % stride == 0 and entry // stride < n_pages else -1


def fork(tables, lens, parents, new_lens, n_pages, stride, block, reserved=None):
    """(tables_out, lens_out, counts, copies): copies are (from, to) pages."""
    rows_in, width = tables.shape
    n = len(parents)
    blocks = lambda x: -(-x // block)  # noqa: E731
    good = []
    for i in range(n):
        p, more = int(parents[i]), 1 if new_lens is None else int(new_lens[i])
        ok = 0 <= p < rows_in and lens[p] >= 0 and more >= 0 and int(lens[p]) + more <= 2 ** 31 - 1 and blocks(int(lens[p]) + more) <= width
        good.append(ok)
    first = {}
    for i in range(n):
        if good[i]:
            first.setdefault(int(parents[i]), i)
    held = set() if reserved is None else set(np.flatnonzero(reserved).tolist())
    for p in first:
        held |= {_page(int(e), n_pages, stride) for e in tables[p, :blocks(int(lens[p]))]}
    free = [p for p in range(n_pages) if p not in held]
    out, out_lens, copies, wanted = np.full((n, width), -1, np.int32), np.zeros(n, np.int32), [], 0
    for i in range(n):
        p = int(parents[i])
        if p < 0:
            continue
        out_lens[i] = -1
        if not good[i]:
            continue
        length, more = int(lens[p]), 1 if new_lens is None else int(new_lens[i])
        kept = blocks(length)
        copy = length % block != 0 and first[p] != i
        if copy and _page(int(tables[p, kept - 1]), n_pages, stride) < 0:
            continue
        shared = kept - copy
        need = blocks(length + more) - shared
        at, wanted = wanted, wanted + need
        if need and wanted > len(free):
            continue
        out_lens[i] = length
        out[i, :shared] = tables[p, :shared]
        out[i, shared:shared + need] = [f * stride for f in free[at:wanted]]
        if copy:
            copies.append((_page(int(tables[p, kept - 1]), n_pages, stride), free[at]))
    return out, out_lens, np.array([wanted, len(free)]), copies


def compact(tables, n_pages, stride, reserved=None):
    """(tables_out, moved_to, counts, moves): moves are (from, to) pages."""
    taken = np.zeros(n_pages, bool) if reserved is None else np.asarray(reserved) != 0
    used = np.zeros(n_pages, bool)
    for e in tables.ravel():
        if _page(int(e), n_pages, stride) >= 0:
            used[_page(int(e), n_pages, stride)] = True
    total = int((used & ~taken).sum())
    front = np.flatnonzero(~taken)[:total].tolist()
    inside = set(front)
    leave = [p for p in range(n_pages) if used[p] and not taken[p] and p not in inside]
    empty = [p for p in front if not used[p]]
    moved = np.where(used, np.arange(n_pages), -1).astype(np.int32)
    for a, b in zip(leave, empty):
        moved[a] = b
    out = tables.copy()
    for at, e in np.ndenumerate(tables):
        p = _page(int(e), n_pages, stride)
        if p >= 0:
            out[at] = moved[p] * stride
    return out, moved, np.array([total, len(leave)]), list(zip(leave, empty))
