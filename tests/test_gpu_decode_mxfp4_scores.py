"""Scores of pbe_paged_decode_mxfp4 whose terms differ by many powers of two:
queries with one dim far above the others. The bound is that of
test_gpu_decode_mxfp4 (products of BF16 numbers are exact in FP32, sums take a
rounding of 2^-24 per term); where the large dim meets zero codes, or keys as
small as it is large, the terms' magnitudes, and the bound with them, stay what
they are without it."""
import numpy as np
import pytest

from oracle import mxfp4 as M
from tests.conftest import say
from tests.test_gpu_decode_mxfp4 import T, Case

pytestmark = pytest.mark.gpu


def set_code(c, dim, code):
    """The code of one dim of every key."""
    pool = c.views()[0]
    at = M.code_at(np.arange(c.blocks * T), c.heads, c.dim, False)[..., dim].ravel()
    pool[at] = (pool[at] & 0x0F) | (code << 4) if dim % 2 else (pool[at] & 0xF0) | code


def key_scales(c):
    """The scale bytes of all keys' groups: [slots][heads][groups], and where they lie."""
    at = M.scale_at(np.arange(c.blocks * T), c.heads, c.dim)
    return at, c.views()[2]


def set_query(torch, c, dims, factor):
    c.q[..., dims] = (c.q[..., dims].double() * factor).to(torch.bfloat16)
    c.q_host = c.q.double().cpu().numpy()


LENS = [2, 3, 2, 17, 200, 2, 700]


@pytest.mark.parametrize("up", [14, 17, 20, 40, 100])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (1, 12, 128), (1, 9, 64)])
def test_a_large_query_dim_meets_zeros(torch_cuda, heads, group, dim, up):
    torch = torch_cuda
    say(f"decode mxfp4 scores: zeros at a dim 2^{up} above the others, H={heads}x{group} D={dim}")
    c = Case(torch, LENS, heads, group, dim, seed=up)
    set_code(c, dim - 3, 0)
    c.upload()
    set_query(torch, c, dim - 3, 2.0 ** up)
    for splits in (1, 8):
        c.call(splits)
        c.check()


@pytest.mark.parametrize("up", [14, 20, 60])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (1, 12, 128)])
def test_a_large_group_of_query_dims_meets_small_keys(torch_cuda, heads, group, dim, up):
    torch = torch_cuda
    say(f"decode mxfp4 scores: a group 2^{up} above the others, H={heads}x{group} D={dim}")
    c = Case(torch, LENS, heads, group, dim, seed=up + 1)
    at, scales = key_scales(c)
    first = at[..., 0]
    scales[first] = np.where(scales[first] == 255, 255, np.maximum(scales[first].astype(int) - up, 0))
    c.upload()
    set_query(torch, c, slice(0, 32), 2.0 ** up)
    for splits in (1, 8):
        c.call(splits)
        c.check()


@pytest.mark.parametrize("up", [8, 12, 16])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (1, 12, 128)])
def test_a_large_term_that_all_scores_share(torch_cuda, heads, group, dim, up):
    """It leaves the weights as they are, up to its rounding in the scores."""
    torch = torch_cuda
    say(f"decode mxfp4 scores: 2^{up} in all of them, H={heads}x{group} D={dim}")
    c = Case(torch, [2] * 40 + [5, 300], heads, group, dim, seed=up + 2)
    set_code(c, 5, 2)   # 1.0
    at, scales = key_scales(c)
    first = at[..., 0]
    scales[first] = np.where(scales[first] == 255, 255, 127)
    c.upload()
    c.q[..., 5] = 1.0
    set_query(torch, c, 5, 2.0 ** up)
    for splits in (1, 8):
        c.call(splits)
        c.check()


@pytest.mark.parametrize("up", [0, 30, 36, 60, 100])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (1, 12, 128)])
def test_equal_scores_of_any_size_give_the_mean(torch_cuda, heads, group, dim, up):
    """Every key is the same, so all weights are: the output is the values' mean, off
    by half a step of BF16 and (n / 32 + 64) roundings of 2^-23 of the sums."""
    torch = torch_cuda
    say(f"decode mxfp4 scores: equal ones of about 2^{up}, H={heads}x{group} D={dim}")
    c = Case(torch, [1, 2, 17, 100, 500, 900], heads, group, dim, seed=up + 3)
    for d in range(dim):
        set_code(c, d, 1 + d % 7)
    at, scales = key_scales(c)
    scales[at] = np.where(scales[at] == 255, 255, 127)
    c.upload()
    set_query(torch, c, slice(0, dim), 2.0 ** up)
    still = np.zeros_like(c.q_host)
    o, _, size, _ = M.decode(still, c.views(), c.tables, c.lens, heads)
    n = np.array(c.lens)[:, None, None]
    bound = 2.0 ** -8 * np.abs(o) + (n / 32 + 64) * 2.0 ** -23 * size
    for splits in (1, 8):
        c.out.fill_(5.0)
        c.call(splits)
        torch.cuda.synchronize()
        assert (np.abs(c.out.double().cpu().numpy() - o) <= bound).all()


BEYOND = [("first", lambda n: [0]), ("first tile", lambda n: range(0, 32)), ("first tiles of all waves", lambda n: range(0, 128)),
          ("all but the last", lambda n: range(0, n - 1)), ("every other block", lambda n: [t for t in range(n) if t // T % 2 == 0]),
          ("last", lambda n: [n - 1])]


def beyond(torch, lens, heads, group, dim, tokens, sign=8):
    """Queries and keys whose products pass FP32's range at some tokens, and are
    zero at that dim for the others: what the oracle says of these, but for the
    magnitudes of their scores."""
    c = Case(torch, lens, heads, group, dim, seed=dim + len(lens))
    set_code(c, 7, 0)
    pool, scales = c.views()[0], c.views()[2]
    for b, n in enumerate(lens):
        t = np.array([x for x in tokens(n) if x < n], np.int64)
        slots = c.tables[b, t // T].astype(np.int64) * T + t % T
        at = M.code_at(slots, heads, dim, False)[..., :32]
        pool[at] = 0
        pool[at[..., 7]] = (6 | sign) << 4   # 4 or -4, an odd dim: the high half
        scales[M.scale_at(slots, heads, dim)[..., 0]] = 252
    c.upload()
    c.q[..., 7] = 2.0 ** 20
    c.q_host = c.q.double().cpu().numpy()
    o, spread, size, _ = M.decode(c.q_host, c.views(), c.tables, lens, heads)
    q = c.q_host.copy()
    q[..., 7] = 0
    return c, (o, spread, size, M.decode(q, c.views(), c.tables, lens, heads)[3])


@pytest.mark.parametrize("which,tokens", BEYOND, ids=[w for w, _ in BEYOND])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (1, 12, 128)])
def test_scores_below_all_numbers_have_no_weight(torch_cuda, heads, group, dim, which, tokens):
    torch = torch_cuda
    say(f"decode mxfp4 scores: -infinity at {which}, H={heads}x{group} D={dim}")
    c, want = beyond(torch, [2, 33, 150, 700, 1100], heads, group, dim, tokens)
    for splits in (1, 2, 16):
        c.out.fill_(5.0)
        c.call(splits)
        c.check(want=want, skip=[b for b, n in enumerate(c.lens) if len(set(tokens(n)) & set(range(n))) == n])


def test_no_softmax_of_nothing_but_infinities(torch_cuda):
    torch = torch_cuda
    say("decode mxfp4 scores: all -infinity, or one +infinity")
    for sign, tokens in ((8, lambda n: range(n)), (0, lambda n: [n // 2]), (0, lambda n: range(n))):
        c, _ = beyond(torch, [1, 40, 700], 2, 6, 128, tokens, sign)
        for splits in (1, 8):
            c.out.fill_(5.0)
            c.call(splits)
            torch.cuda.synchronize()
            assert torch.isnan(c.out.float()).all()
    c, _ = beyond(torch, [0, 0], 2, 6, 128, lambda n: [])
    c.call(1)
    torch.cuda.synchronize()
    assert (c.out == 0).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_keys_of_two_to_the_128_count_as_infinities(torch_cuda, dim):
    """Scale byte 254 and code 6, which the page writer does not store."""
    torch = torch_cuda
    say(f"decode mxfp4 scores: a key of 6 x 2^127, D={dim}")
    c = Case(torch, [70], 1, 2, dim, seed=dim)
    slot = int(c.tables[0, 1]) * T + 4
    at = M.code_at([slot], 1, dim, False)[0, 0, :32]
    c.views()[0][at] = 0
    c.views()[0][at[9]] = 7 << 4
    c.views()[2][M.scale_at([slot], 1, dim)[0, 0, 0]] = 254
    c.upload()
    c.q[0, 0, 9], c.q[0, 1, 9] = 1.0, -1.0
    c.q_host = c.q.double().cpu().numpy()
    o, spread, size, reach = M.decode(c.q_host, c.views(), c.tables, c.lens, 1)
    c.views()[0][at[9]] = 0
    reach = M.decode(c.q_host, c.views(), c.tables, c.lens, 1)[3]
    c.call(1)
    torch.cuda.synchronize()
    assert torch.isnan(c.out[0, 0].float()).all()
    got, o, spread, size = c.out[0, 1].double().cpu().numpy(), o[0, 1], spread[0, 1], size[0, 1]
    e = 2 * (dim + 16) * 2.0 ** -24 * reach[0, 1] + 2.0 ** -20
    assert (np.abs(got - o) <= 2.0 ** -8 * np.abs(o) + e * spread + (2.0 ** -15 + 70 * 2.0 ** -23) * size).all()
