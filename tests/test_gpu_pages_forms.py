"""pbe_fork_pages and pbe_compact_pages at the ends of what they take, against their
definition."""
import numpy as np
import pytest

import pbe_handoff as P
from tests.conftest import say
from tests.test_gpu_pages import Pool, check_compact, check_fork, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows_in", [3583, 3584, 3585, 5000])
@pytest.mark.parametrize("rows_out", [700, 3000])
def test_forks_from_thousands_of_rows(torch_cuda, rows_in, rows_out):
    """Beyond 3,584 rows, first children are kept in the workspace. Parents are named up
    to some dozens of times, by children near and far; most last pages are not full."""
    say(f"fork: {rows_out} rows from {rows_in}")
    rng = np.random.default_rng(rows_in + rows_out)
    n_pages = 40000
    pool = Pool(torch_cuda, n_pages, (48,), seed=rows_in)
    lens = [int(x) for x in rng.integers(0, 80, rows_in)]
    rows, _ = rows_of(rng, lens, n_pages, 2, 8)
    parents = rng.integers(-1, rows_in, rows_out).astype(np.int32)
    few = rng.integers(0, rows_in, 30)
    often = rng.random(rows_out) < 0.4
    parents[often] = rng.choice(few, int(often.sum()))
    parents[[0, 1, -1]] = rows_in - 1, rows_in, rows_in - 1          # the last row; none such
    new = rng.integers(0, 40, rows_out).astype(np.int32)
    for more, reserved in ((None, None), (new, rng.random(n_pages) < 0.3), (new, rng.random(n_pages) < 0.95)):
        want = check_fork(torch_cuda, pool, rows, lens, parents, more, 2, reserved=reserved)
        assert len(want[3]) > 50


def test_as_many_planes_and_segments_as_a_call_takes(torch_cuda):
    say("fork and compact: 112 planes of two segments")
    rng = np.random.default_rng(1)
    pool = Pool(torch_cuda, 30, tuple(16 * (1 + i % 7) for i in range(112)), seg=15, seed=1)
    lens = [17, 40, 16, 3]
    rows, _ = rows_of(rng, lens, 30, 4, 6)
    check_fork(torch_cuda, pool, rows, lens, [0, 0, 1, 1, 2, 3, 3], None, 4)
    check_compact(torch_cuda, pool, rows, 4)


def test_the_largest_pages(torch_cuda):
    """Pages of 1 GiB in a pool of 9 GiB."""
    torch = torch_cuda
    say("fork and compact: pages of 1 GiB")
    size, n = 1 << 30, 9
    pool = torch.empty((n, size // 8), dtype=torch.int64, device="cuda")
    word = torch.arange(size // 8, device="cuda")
    for i in range(n):
        torch.add(word, i << 40, out=pool[i])
    planes = P.page_planes([(P.view_of([pool.data_ptr()], n * size, n * size), size)])
    ws = torch.full((4096,), 0xff, dtype=torch.uint8, device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    tables, lens, parents, out, out_lens, counts = ints(8, 5, -1), ints(20), ints(0, 0), ints(*[7] * 6), ints(7, 7), ints(7, 7)
    P.fork_pages(planes, n, 1, 16, tables.data_ptr(), lens.data_ptr(), 1, parents.data_ptr(), 0, 2, 3, 0, out.data_ptr(), out_lens.data_ptr(),
                 counts.data_ptr(), ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    assert out.tolist() == [8, 5, -1, 8, 0, -1] and counts.tolist() == [1, 7]
    last = ints(*[7] * 6)
    P.compact_pages(planes, n, 1, out.data_ptr(), 2, 3, 0, last.data_ptr(), 0, counts.data_ptr(), ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    # pages 0, 5 and 8 are in use: 0 stays, 5 moves to 1 and 8 to 2
    assert last.tolist() == [2, 1, -1, 2, 0, -1] and counts.tolist() == [3, 2]
    for page, holds in enumerate((5, 5, 8, 3, 4, 5, 6, 7, 8)):
        assert torch.equal(pool[page], word + (holds << 40)), page
