"""pbe_fork_pages where its plan takes other ways, against its definition."""
import numpy as np
import pytest

from tests.conftest import say
from tests.test_gpu_pages import Pool, check_fork, rows_of

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
