"""Sizes at the ends of what the prompt readers and page movers take, refused on the
host before any HIP call. No GPU needed."""
import pytest

import pbe_handoff as P
from tests.test_abi_prompt import FAKE, FORK, PAGES, ROWS

GB = 1 << 30


def refused(call, args, change, what):
    with pytest.raises(P.PbeError) as e:
        call(**{**args, **change})
    assert e.value.code == P.PBE_ERR_INVALID and what in str(e.value), (change, str(e.value))


@pytest.mark.parametrize("batch", [2 ** 31 - 255, 2 ** 31 - 64, 2 ** 31 - 1])
def test_batches_whose_last_sequences_a_wave_would_count_past(batch):
    """A wave looks at 64 sequences at a time, in 32-bit numbers."""
    far = {"batch": batch, "workspace": 0, "workspace_bytes": 0}
    refused(P.prompt_attention, ROWS, {**far, "q_starts": FAKE + 100 * GB, "k_starts": FAKE + 200 * GB}, "batch")
    refused(P.paged_prompt_attention, PAGES, {**far, "token_starts": FAKE + 100 * GB, "seq_lens": FAKE + 200 * GB, "tables": FAKE + 300 * GB, "max_blocks": 1},
            "batch")


@pytest.mark.parametrize("rows", [2 ** 31 - 1023, 2 ** 31 - 1])
def test_forks_of_more_rows_than_the_plan_counts(rows):
    """The plan takes 1,024 rows at a time, in 32-bit numbers."""
    apart = {n: FAKE + (i + 2) * 100 * GB for i, n in enumerate(("tables_in", "lens_in", "parents", "new_lens", "reserved", "tables_out", "lens_out", "counts",
                                                                "workspace"))}
    for change in (dict(rows_in=rows), dict(rows_out=rows)):
        refused(P.fork_pages, FORK, {**apart, **change, "max_blocks": 1, "workspace_bytes": 90 * GB}, "rows")
