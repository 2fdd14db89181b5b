"""Sizes at the ends of what pbe_paged_decode_mxfp4 takes: the host's arithmetic
here, the calls themselves on a GPU."""
import pytest

import pbe_handoff as P


@pytest.mark.parametrize("blocks", [2 ** 27, 2 ** 31 - 16, 2 ** 31 - 15, 2 ** 31 - 1])
def test_splits_of_the_widest_tables(blocks):
    """Long tables are cut for the chip, however wide they are."""
    most = P.decode_mxfp4_splits(1, 2, 2 ** 20)
    assert most > 1
    assert P.decode_mxfp4_splits(1, 2, blocks) == most
    assert P.decode_mxfp4_splits(40, 2, blocks) == P.decode_mxfp4_splits(40, 2, 2 ** 20) > 1


@pytest.mark.gpu
def test_a_sequence_in_the_widest_table(torch_cuda):
    from tests.conftest import say
    from tests.test_gpu_decode_mxfp4 import Case
    torch = torch_cuda
    say("decode mxfp4 with a table of 2^31 - 1 blocks")
    c = Case(torch, [900], 2, 3, 64, seed=1)
    wide = torch.full((2 ** 31 - 1,), -1, dtype=torch.int32, device="cuda")
    wide[: c.max_blocks] = c.tables_dev[0]
    c.max_blocks = len(wide)
    want = None
    for splits in (0, 1, 7):
        c.out.fill_(5.0)
        c.call(splits, tables=wide)
        want = c.check(want=want)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 16])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (1, 12, 128)])
def test_outputs_in_the_queries_place(torch_cuda, heads, group, dim, splits):
    from tests.conftest import say
    from tests.test_gpu_decode_mxfp4 import Case
    torch = torch_cuda
    say(f"decode mxfp4 in place H={heads}x{group} D={dim} splits={splits}")
    c = Case(torch, [0, 1, 40, 900, 2000], heads, group, dim, seed=2)
    c.call(splits)
    torch.cuda.synchronize()
    c.call(splits, out=c.q)
    torch.cuda.synchronize()
    assert torch.equal(c.q.view(torch.int16), c.out.view(torch.int16))
