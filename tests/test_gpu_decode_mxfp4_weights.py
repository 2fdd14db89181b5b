"""Weights of pbe_paged_decode_mxfp4 beyond BF16: probabilities enter the product
with the values as two BF16 parts, cut off, so within 2^-15 of themselves, and are
divided by the sum of the FP32 ones. Bound of an output o = sum w v: 2^-15 sum w
|v| for that, and for the rest what test_gpu_decode_mxfp4 derives: the scores'
error of sum w |v - o|, the FP32 sums' of sum w |v|, half a step of BF16 of o, and
what lies below FP32's smallest normal number. Where the values of a few tokens
cancel, that is far below the 2^-8 of their spread that one BF16 number leaves."""
import numpy as np
import pytest

from oracle import mxfp4 as M
from tests.conftest import say
from tests.test_gpu_decode_mxfp4 import Case

pytestmark = pytest.mark.gpu


def check(c, want=None):
    c.torch.cuda.synchronize()
    got = c.out.double().cpu().numpy()
    o, spread, size, reach = want or M.decode(c.q_host, c.views(), c.tables, c.lens, c.heads)
    n = np.array(c.lens)[:, None, None]
    e = (2 * (c.dim + 16) * 2.0 ** -24 * reach + 2.0 ** -20)[..., None]
    v_scales = c.views()[3]
    bound = 2.0 ** -8 * np.abs(o) + e * spread + (2.0 ** -15 + (n / 32 + 64) * 2.0 ** -23) * size
    bound += 2.0 ** -126 * (2 * n * 6 * 2.0 ** (float(v_scales[v_scales != 255].max()) - 127) + n + 1)
    off = np.abs(got - o) - bound
    assert off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))
    return o, spread, size, reach


@pytest.mark.parametrize("splits", [1, 8])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (4, 8, 128), (1, 12, 128), (2, 16, 64), (1, 1, 128)])
def test_weights_are_finer_than_bf16(torch_cuda, heads, group, dim, splits):
    say(f"decode mxfp4 weights H={heads}x{group} D={dim} splits={splits}")
    c = Case(torch_cuda, [2, 3, 4, 5, 2, 3, 17, 40, 300, 2000], heads, group, dim, seed=dim + group)
    c.call(splits)
    check(c)


@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (1, 12, 128)])
def test_values_that_cancel_leave_what_the_weights_say(torch_cuda, heads, group, dim):
    """Two tokens of opposite values: (w1 - w2) v, with w1 and w2 about equal."""
    say(f"decode mxfp4 weights of values that cancel H={heads}x{group} D={dim}")
    torch = torch_cuda
    c = Case(torch, [2] * 60, heads, group, dim, seed=dim)
    value = c.views()[1]
    for b in range(60):
        slot = int(c.tables[b, 0]) * 16
        one, two = (M.code_at([slot + t], heads, dim, True) for t in (0, 1))
        value[two] = value[one] ^ 0x88
        scales = c.views()[3]
        scales[M.scale_at([slot + 1], heads, dim)] = scales[M.scale_at([slot], heads, dim)]
    c.upload()
    c.q.copy_((c.q.double() / 16).to(torch.bfloat16))
    c.q_host = c.q.double().cpu().numpy()
    c.call(1)
    check(c)


@pytest.mark.parametrize("group", [9, 12, 16])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_sequences_of_many_query_heads(torch_cuda, dim, group):
    """More pieces than are joined four at a time."""
    say(f"decode mxfp4 5040 tokens H=1x{group} D={dim}")
    c = Case(torch_cuda, [5040, 20, 3000], 1, group, dim, seed=group)
    want = None
    for splits in (0, 64, 1):
        c.out.fill_(5.0)
        c.call(splits)
        want = check(c, want)
