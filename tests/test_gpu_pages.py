"""pbe_fork_pages and pbe_compact_pages against their definition: tables, lengths,
counts and every byte of the pool."""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import pages as O
from tests.conftest import say
from tests.gpu_util import stream_ptr

pytestmark = pytest.mark.gpu


class Pool:
    """n_pages pages in planes of the given page sizes, the i-th cut into segments of
    `seg` pages, under random bytes."""

    def __init__(self, torch, n_pages, sizes=(4096,), seg=0, seed=0):
        self.torch, self.n, self.sizes = torch, n_pages, sizes
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        views, self.parts = [], []
        for size in sizes:
            step = seg or n_pages
            parts = [torch.randint(0, 256, (min(step, n_pages - i), size), generator=g, dtype=torch.uint8, device="cuda") for i in range(0, n_pages, step)]
            self.parts.append(parts)
            views.append((P.view_of([x.data_ptr() for x in parts], n_pages * size, step * size), size))
        self.planes = P.page_planes(views)

    def host(self):
        return [self.torch.cat(x).cpu().numpy() for x in self.parts]


def ints(torch, x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda") if x is not None else None


def ptr(t):
    return 0 if t is None else t.data_ptr()


def run_fork(torch, pool, tables, lens, parents, new_lens, stride, block, reserved, stream=None):
    rows, width = len(parents), tables.shape[1]
    dev = [ints(torch, x) for x in (tables, lens, parents, new_lens, reserved)]
    out, out_lens, counts = ints(torch, np.full((rows, width), 77)), ints(torch, [77] * rows), ints(torch, [77, 77])
    ws = torch.full((P.fork_pages_workspace_bytes(pool.n, len(lens), rows),), 0xff, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    P.fork_pages(pool.planes, pool.n, stride, block, ptr(dev[0]), ptr(dev[1]), len(lens), ptr(dev[2]), ptr(dev[3]), rows, width, ptr(dev[4]),
                 out.data_ptr(), out_lens.data_ptr(), counts.data_ptr(), ws.data_ptr(), ws.numel(), stream=stream_ptr(torch) if stream is None else stream)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in (out, out_lens, counts)]


def check_fork(torch, pool, tables, lens, parents, new_lens=None, stride=1, block=16, reserved=None):
    tables, lens = np.asarray(tables, np.int32), np.asarray(lens, np.int32)
    want = O.fork(tables, lens, parents, new_lens, pool.n, stride, block, reserved)
    pages = pool.host()
    for a, b in want[3]:
        for x in pages:
            x[b] = x[a]
    got = run_fork(torch, pool, tables, lens, parents, new_lens, stride, block, reserved)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    for g, w in zip(pool.host(), pages):
        np.testing.assert_array_equal(g, w)
    return want


def rows_of(rng, lens, n_pages, stride, width, block=16, spare=0):
    """Rows of pages of their own, out of shuffled ones, and the pages left."""
    order = list(rng.permutation(n_pages))
    rows = np.full((len(lens), width), -1, np.int32)
    for i, n in enumerate(lens):
        k = -(-n // block) + (spare if i % 2 else 0)
        rows[i, :k] = [order.pop() * stride for _ in range(k)]
    return rows, order


@pytest.mark.parametrize("sizes,seg,stride", [((4096,), 0, 1), ((1040,), 0, 56), ((16, 48), 11, 1), ((70000, 16400, 512, 512), 13, 4)])
def test_forks_ends_growth_and_moves_of_rows(torch_cuda, sizes, seg, stride):
    say(f"fork pages of {sizes} in segments of {seg}, stride {stride}")
    rng = np.random.default_rng(len(sizes) + stride)
    pool = Pool(torch_cuda, 150, sizes, seg, seed=stride)
    lens = [0, 1, 15, 16, 17, 160, 100, 33]
    rows, _ = rows_of(rng, lens, 150, stride, 14, spare=1)
    parents = [7, 1, 1, -1, 2, 5, 5, 5, 4, 1, 0, 3, 3, -5, 7]
    check_fork(torch_cuda, pool, rows, lens, parents, None, stride)
    check_fork(torch_cuda, pool, rows, lens, parents, [0] * 15, stride)
    check_fork(torch_cuda, pool, rows, lens, parents, list(rng.integers(0, 40, 15)), stride, reserved=rng.random(150) < 0.2)


def test_rows_that_do_not_fit_or_make_no_sense(torch_cuda):
    say("fork: bad rows")
    rng = np.random.default_rng(3)
    pool = Pool(torch_cuda, 40)
    lens = [20, 33, -1, 4 * 16, 16, 70]
    rows, _ = rows_of(rng, [20, 33, 0, 64, 16, 64], 40, 3, 4)
    rows[1, 1] = 10 ** 9                      # shared by its children, whatever it is
    rows[0, 1] = 41                           # not a multiple of the stride: no page to copy
    parents = [0, 0, 1, 1, 2, 3, 3, 4, 5, 6, 2 ** 31 - 1, -2 ** 31, 4]
    new = [1, 1, 0, 5, 1, 0, 1, -1, 0, 1, 1, 1, 2 ** 31 - 1]
    check_fork(torch_cuda, pool, rows, lens, parents, new, 3)


@pytest.mark.parametrize("room", [0, 1, 2, 3, 4, 5, 30])
def test_fresh_pages_run_out(torch_cuda, room):
    say(f"fork: {room} pages to take")
    rng = np.random.default_rng(room)
    lens = [17, 16, 40, 31]
    rows, left = rows_of(rng, lens, 39, 1, 6)
    reserved = np.ones(39, np.int32)
    reserved[left[:room]] = 0
    reserved[rows[rows >= 0]] = 0
    pool = Pool(torch_cuda, 39)
    want = check_fork(torch_cuda, pool, rows, lens, [0, 0, 1, 2, 3, 2, 2, 1, 3], [1, 1, 0, 20, 1, 1, 0, 1, 0], 1, reserved=reserved)
    assert want[2][1] == room


@pytest.mark.parametrize("seed", range(4))
def test_random_steps_of_many_requests(torch_cuda, seed):
    """Steps one after another, each on the last one's tables and grown lengths."""
    torch = torch_cuda
    say(f"fork: random steps, seed {seed}")
    rng = np.random.default_rng(seed)
    n_pages, block, stride = int(rng.integers(200, 3000)), int(rng.choice([1, 3, 16])), int(rng.choice([1, 2, 48]))
    pool = Pool(torch, n_pages, (64,), seed=seed)
    count = int(rng.integers(2, 60))
    width = max(4, n_pages // count)
    lens = [int(rng.integers(0, width * block // 3 + 1)) for _ in range(count)]
    rows, _ = rows_of(rng, lens, n_pages, stride, width, block)
    for _ in range(5):
        n = int(rng.integers(1, 2 * count))
        new = rng.integers(0, 2 * block + 1, n).astype(np.int32)
        rows, lens, _, _ = check_fork(torch, pool, rows, lens, rng.integers(-1, len(lens), n).astype(np.int32), new, stride, block)
        lens = np.where(lens >= 0, lens + new, -1)


def test_more_rows_than_the_plan_takes_at_once(torch_cuda):
    say("fork: 2500 rows, 1024 * 33 + 5 pages")
    rng = np.random.default_rng(9)
    n_pages = 1024 * 33 + 5
    pool = Pool(torch_cuda, n_pages, (16,))
    lens = [int(x) for x in rng.integers(0, 100, 1300)]
    rows, _ = rows_of(rng, lens, n_pages, 1, 9)
    check_fork(torch_cuda, pool, rows, lens, rng.integers(-1, 1300, 2500).astype(np.int32), None, 1, reserved=rng.random(n_pages) < 0.7)


def test_the_largest_pool(torch_cuda):
    say("fork and compact: 2^20 pages")
    rng = np.random.default_rng(10)
    n = 1 << 20
    pool = Pool(torch_cuda, n, (16,))
    lens = [1000, 37, 5]
    rows = np.full((3, 70), -1, np.int32)
    for i, k in enumerate((63, 3, 1)):
        rows[i, :k] = (n - 1 - rng.permutation(5000)[:k] * 3 - i) * 2
    check_fork(torch_cuda, pool, rows, lens, [0, 1, 0, 1, 2], None, 2)
    check_compact(torch_cuda, pool, rows, 2)


def check_compact(torch, pool, tables, stride=1, reserved=None, moved=True):
    tables = np.asarray(tables, np.int32)
    want = O.compact(tables, pool.n, stride, reserved)
    pages = pool.host()
    for a, b in want[3]:
        for x in pages:
            x[b] = x[a]
    dev = [ints(torch, x) for x in (tables, reserved)]
    out, to, counts = ints(torch, np.full(tables.shape, 77)), ints(torch, [77] * pool.n) if moved else None, ints(torch, [77, 77])
    ws = torch.full((P.compact_pages_workspace_bytes(pool.n),), 0xff, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    P.compact_pages(pool.planes, pool.n, stride, ptr(dev[0]), len(tables), tables.shape[1], ptr(dev[1]), out.data_ptr(), ptr(to), counts.data_ptr(),
                    ws.data_ptr(), ws.numel(), stream=stream_ptr(torch))
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out.cpu().numpy(), want[0])
    if moved:
        np.testing.assert_array_equal(to.cpu().numpy(), want[1])
    np.testing.assert_array_equal(counts.cpu().numpy(), want[2])
    for g, w in zip(pool.host(), pages):
        np.testing.assert_array_equal(g, w)
    return want


@pytest.mark.parametrize("sizes,seg,stride", [((4096,), 0, 1), ((1040,), 0, 56), ((16, 48), 11, 1), ((70000, 16400, 512, 512), 13, 4)])
@pytest.mark.parametrize("n_pages", [1, 63, 64, 65, 150, 1500])
def test_pages_move_to_the_front(torch_cuda, n_pages, sizes, seg, stride):
    if n_pages * sum(sizes) > 2 ** 26 or (seg and n_pages > 16 * seg):
        seg, sizes = 0, (sizes[-1], 16)
    say(f"compact {n_pages} pages of {sizes} in segments of {seg}, stride {stride}")
    rng = np.random.default_rng(n_pages + stride)
    pool = Pool(torch_cuda, n_pages, sizes, seg, seed=n_pages)
    for share, held in ((0.0, 0.0), (0.3, 0.0), (0.5, 0.3), (1.0, 0.1)):
        used = np.flatnonzero(rng.random(n_pages) < share)
        tables = np.full((5, max(1, n_pages)), -1, np.int32)
        for row in tables:                      # rows share pages
            k = int(rng.integers(0, len(used) + 1))
            row[:k] = rng.permutation(used)[:k] * stride
        tables[0, : len(used)] = used * stride
        reserved = (rng.random(n_pages) < held).astype(np.int32) if held else None
        check_compact(torch_cuda, pool, tables, stride, reserved, moved=share != 0.3)


def test_entries_that_name_no_page_stay_as_they_are(torch_cuda):
    say("compact: entries outside the pool")
    pool = Pool(torch_cuda, 20)
    check_compact(torch_cuda, pool, [[57, 3, -7, 60, 2 ** 31 - 1, -2 ** 31, 4, 30]], 3)


def test_compacted_pages_are_one_run(torch_cuda):
    say("compact: one run")
    rng = np.random.default_rng(4)
    pool = Pool(torch_cuda, 200)
    rows, _ = rows_of(rng, [160, 300, 47], 200, 1, 20)
    out, _, counts, _ = check_compact(torch_cuda, pool, rows)
    assert sorted(out[out >= 0]) == list(range(counts[0]))


def test_captured_moves_follow_what_changes_between_replays(torch_cuda):
    """A compaction behind a fork in one graph on a stream of its own, replayed in turn
    with another graph that shares the workspace."""
    torch = torch_cuda
    say("fork and compact in graphs that share a workspace")
    n, width, rows = 70, 8, 5
    ws = torch.full((max(P.fork_pages_workspace_bytes(n, rows, rows), P.compact_pages_workspace_bytes(n)),), 0xff, dtype=torch.uint8, device="cuda")
    side, runs = torch.cuda.Stream(), []
    for seed in range(2):
        rng = np.random.default_rng(seed)
        pool = Pool(torch, n, (4096, 528), 0, seed)
        lens = [int(x) for x in rng.integers(1, 60, rows)]
        tables, _ = rows_of(rng, lens, n, 3, width)
        dev = [ints(torch, x) for x in (tables, lens, range(rows))]
        mid, mid_lens, counts, last, moved = ints(torch, np.zeros((rows, width))), ints(torch, [0] * rows), ints(torch, [0, 0]), \
            ints(torch, np.zeros((rows, width))), ints(torch, [0] * n)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                P.fork_pages(pool.planes, n, 3, 16, ptr(dev[0]), ptr(dev[1]), rows, ptr(dev[2]), 0, rows, width, 0, mid.data_ptr(),
                             mid_lens.data_ptr(), counts.data_ptr(), ws.data_ptr(), ws.numel(), stream=side.cuda_stream)
                P.compact_pages(pool.planes, n, 3, mid.data_ptr(), rows, width, 0, last.data_ptr(), moved.data_ptr(), counts.data_ptr(), ws.data_ptr(),
                                ws.numel(), stream=side.cuda_stream)
        runs.append((g, pool, rng, tables, lens, dev, mid, mid_lens, last, moved, counts))
    for rep in range(4):
        for g, pool, rng, tables, lens, dev, mid, mid_lens, last, moved, counts in runs:
            parents = rng.integers(-1, rows, rows)
            dev[2].copy_(ints(torch, parents))
            want = O.fork(tables, np.asarray(lens), parents, None, n, 3, 16)
            packed = O.compact(want[0], n, 3)
            pages = pool.host()
            for moves in (want[3], packed[3]):
                for x in pages:
                    x[[b for _, b in moves]] = x[[a for a, _ in moves]]
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                g.replay()
            torch.cuda.synchronize()
            for got, x in zip((mid, mid_lens, last, moved, counts), (want[0], want[1], *packed[:3])):
                np.testing.assert_array_equal(got.cpu().numpy(), x)
            for got, x in zip(pool.host(), pages):
                np.testing.assert_array_equal(got, x)
