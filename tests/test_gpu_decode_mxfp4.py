"""pbe_paged_decode_mxfp4 against attention in 64 bits over the same pages.

Bound of an output o = sum w v (w the softmax weights): the probabilities are
rounded to BF16, each by at most 2^-8 of itself, and divided by the sum of the
rounded ones, which moves the mean by at most 2^-8 / (1 - 2^-8) sum w |v - o|.
In the same way an FP32 error e of a probability moves it by at most e sum w |v -
o|: e is the score's error, (dim + 16) roundings of 2^-24 of sum |q k| / sqrt(dim)
and as much again for the maximum's, the exponential's 2^-22 and the product's
with the maxima's scales. Sums of p v take a rounding per product of 32 tokens
and per piece, wave and join, below n / 32 + 64 of them, of 2^-23 each (the
products' own additions included), relative to sum w |v|. The output is rounded
to BF16, 2^-8 of itself. Below FP32's smallest normal number, 2^-126, a
probability, its BF16 rounding, its product with a value or the output may become
zero: with the largest probability 1, and so their sum at least 1, that moves the
output by at most 2^-126 for each token's probability and product (n times the
largest |v - o| <= 2 max |v|, and n) and for the output: 2^-126 (2 n max |v| + n +
1).
"""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import mxfp4 as M
from tests.conftest import say
from tests.gpu_util import stream_ptr

pytestmark = pytest.mark.gpu

T = 16


class Case:
    """A batch over shuffled pages (of a page-major arena's layer, or local
    pools). Behind the sequences' last tokens, and in the pages that none has,
    lie random codes under NaN scales; behind the last block of a table, ids
    that no pool has."""

    def __init__(self, torch, lens, heads, group, dim, layers=1, layer=0, seed=0, spread=1.0, spare=3, width=0):
        rng = np.random.default_rng(seed)
        self.torch, self.lens, self.heads, self.group, self.dim = torch, list(lens), heads, group, dim
        half = M.half_bytes(heads, dim)
        stride = 2 * layers if layers > 1 else 1
        blocks = [-(-n // T) for n in lens]
        n_pages = sum(blocks) + spare
        planes = 2 * layers * n_pages
        self.codes = rng.integers(0, 256, planes * half).astype(np.uint8)
        self.scales = np.full(planes * half // 16, 255, np.uint8)
        self.k_plane, self.v_plane = (2 * layer, 2 * layer + 1) if layers > 1 else (0, n_pages)
        self.blocks = planes - self.v_plane
        self.per = (half, half // 16)
        perm = rng.permutation(n_pages) * stride
        self.max_blocks = max(max(blocks), 1) + width
        self.tables = np.where(rng.random((len(lens), self.max_blocks)) < 0.5, -5, 2 ** 31 - 1).astype(np.int32)
        at = 0
        views = self.views()
        for b, (n, k) in enumerate(zip(lens, blocks)):
            self.tables[b, :k] = perm[at:at + k]
            at += k
            if n:
                t = np.arange(n)
                slots = self.tables[b, t // T].astype(np.int64) * T + t % T
                sc = M.scale_at(slots, heads, dim)
                for s in views[2:]:
                    s[sc] = np.clip(127 + np.rint(rng.standard_normal(sc.shape) * spread - 1), 0, 250)
        q = torch.tensor(rng.standard_normal((len(lens), heads * group, dim)) * 2, dtype=torch.float32).to(torch.bfloat16)
        self.q, self.q_host = q.cuda(), q.double().numpy()
        self.upload()

    def views(self):
        k, v = self.k_plane, self.v_plane
        return [self.codes[k * self.per[0]:], self.codes[v * self.per[0]:], self.scales[k * self.per[1]:], self.scales[v * self.per[1]:]]

    def upload(self):
        torch = self.torch
        self.dev = [torch.from_numpy(self.codes).cuda(), torch.from_numpy(self.scales).cuda()]
        self.tables_dev = torch.from_numpy(self.tables).cuda()
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.out = torch.full(self.q.shape, 5.0, dtype=torch.bfloat16, device="cuda")

    def workspace(self, splits):
        n = P.decode_mxfp4_workspace_bytes(len(self.lens), self.heads * self.group, self.dim, splits or 1024)
        return self.torch.full((max(n, 16),), 0xff, dtype=self.torch.uint8, device="cuda")  # NaN bytes

    def call(self, splits=0, workspace=None, stream=None, out=None, tables=None, lens=None):
        a, s = self.dev
        ws = self.workspace(splits) if workspace is None else workspace
        P.paged_decode_mxfp4(a.data_ptr() + self.k_plane * self.per[0], a.data_ptr() + self.v_plane * self.per[0], self.blocks * self.per[0],
                             s.data_ptr() + self.k_plane * self.per[1], s.data_ptr() + self.v_plane * self.per[1], self.blocks * self.per[1],
                             self.heads, self.dim, self.q.data_ptr(), (self.out if out is None else out).data_ptr(), len(self.lens),
                             self.heads * self.group, (self.tables_dev if tables is None else tables).data_ptr(),
                             (self.lens_dev if lens is None else lens).data_ptr(), self.max_blocks, splits, ws.data_ptr(), ws.numel(),
                             stream=stream_ptr(self.torch) if stream is None else stream)
        return ws

    def check(self, skip=(), out=None, want=None):
        self.torch.cuda.synchronize()
        got = (self.out if out is None else out).double().cpu().numpy()
        o, spread, size, reach = want or M.decode(self.q_host, self.views(), self.tables, [0 if b in skip else n for b, n in enumerate(self.lens)],
                                                  self.heads)
        n = np.array(self.lens)[:, None, None]
        e = (2 * (self.dim + 16) * 2.0 ** -24 * reach + 2.0 ** -20)[..., None]
        bound = 2.0 ** -8 * np.abs(o) + (2.0 ** -8 / (1 - 2.0 ** -8) + e) * spread + (n / 32 + 64) * 2.0 ** -23 * size
        v_scales = self.views()[3]
        bound += 2.0 ** -126 * (2 * n * 6 * 2.0 ** (float(v_scales[v_scales != 255].max()) - 127) + n + 1)
        keep = [b for b in range(len(self.lens)) if b not in skip]
        off = np.abs(got - o)[keep] - bound[keep]
        assert np.isfinite(got[keep]).all()
        assert off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))
        return o, spread, size, reach


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 129, 255, 256, 257, 1000]


@pytest.mark.parametrize("splits", [0, 1, 3, 64])
@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (4, 7, 128), (1, 1, 64), (3, 16, 128), (8, 4, 64), (1, 9, 128), (5, 2, 128)])
def test_batch_of_odd_lengths_matches_the_oracle(torch_cuda, heads, group, dim, splits):
    say(f"decode mxfp4 H={heads}x{group} D={dim} splits={splits}")
    c = Case(torch_cuda, LENS, heads, group, dim, seed=heads * 7 + group, width=2)
    c.call(splits)
    c.check()


@pytest.mark.parametrize("lens,splits", [([5040], 0), ([5040], 1), ([5040], 1024), ([1], 0), ([16], 1024), ([33, 9001], 0), ([2048] * 3, 5), ([7] * 70, 0),
                                         ([300, 4000, 12, 900] * 6, 0)])
@pytest.mark.parametrize("dim", [64, 128])
def test_few_and_many_sequences_in_an_arena_layer(torch_cuda, lens, splits, dim):
    say(f"decode mxfp4 {len(lens)} sequences up to {max(lens)} D={dim} splits={splits}")
    c = Case(torch_cuda, lens, 2, 6, dim, layers=3, layer=1, seed=len(lens))
    c.call(splits)
    c.check()


def test_unequal_scales_and_large_scores(torch_cuda):
    """Scales that differ by many powers of two from token to token: scores of
    hundreds, and values whose sums are carried by a few tokens."""
    say("decode mxfp4 unequal scales")
    c = Case(torch_cuda, [40, 700, 64], 2, 4, 128, seed=3, spread=4.0)
    for s in c.views()[2:]:
        s[s != 255] = np.minimum(s[s != 255], 135)
    c.upload()
    for splits in (1, 8):
        c.call(splits)
        c.check()


def test_smallest_scales_give_equal_weights(torch_cuda):
    """Scale byte 0 (2^-127): scores of zero and values below what BF16 shows."""
    torch = torch_cuda
    say("decode mxfp4 scale byte 0")
    c = Case(torch, [50], 1, 2, 64, seed=4)
    k, v = c.views()[2:]
    k[k != 255] = 0
    v[v != 255] = 127
    c.upload()
    c.call()
    c.check()


def test_bits_of_repeated_calls_and_of_whole_sequences(torch_cuda):
    """A batch gives the same bits on every call; a sequence read whole (one
    split) the same in any batch."""
    torch = torch_cuda
    say("decode mxfp4 bits in batches")
    c = Case(torch, [1000, 37, 640, 0, 999], 2, 6, 128, seed=6)
    whole = None
    for splits in (4, 40, 1):
        c.call(splits)
        torch.cuda.synchronize()
        whole = c.out.clone()
        for again in range(4):
            c.out.fill_(1.0)
            c.call(splits)
            torch.cuda.synchronize()
            assert torch.equal(whole.view(torch.int16), c.out.view(torch.int16)), splits
    order = [4, 2, 0, 3, 1]
    d = Case(torch, [1000, 37, 640, 0, 999], 2, 6, 128, seed=6)
    d.tables_dev, d.lens_dev = d.tables_dev[order].contiguous(), d.lens_dev[order].contiguous()
    d.q = d.q[order].contiguous()
    d.call(1)
    torch.cuda.synchronize()
    assert torch.equal(d.out.view(torch.int16), whole[order].view(torch.int16))


@pytest.mark.parametrize("batch", [63, 64, 65, 256, 257, 700])
def test_many_mixed_sequences_find_their_pieces(torch_cuda, batch):
    say(f"decode mxfp4 {batch} mixed sequences")
    rng = np.random.default_rng(batch)
    lens = np.where(rng.random(batch) < 0.1, rng.integers(0, 2000, batch), rng.integers(0, 40, batch))
    lens[batch // 2] = 2500
    c = Case(torch_cuda, lens.tolist(), 1, 2, 64, seed=batch)
    want = None
    for splits in (0, 2, 9):
        c.out.fill_(5.0)
        c.call(splits)
        want = c.check(want=want)


@pytest.mark.parametrize("splits", [1, 8])
def test_bad_lengths_and_ids_give_nan_to_their_sequence(torch_cuda, splits):
    torch = torch_cuda
    say(f"decode mxfp4 bad sequences splits={splits}")
    lens = [300, 300, 300, 300, 300, 40, 300]
    c = Case(torch, lens, 2, 3, 128, seed=8)
    c.tables[1, 7] = c.blocks          # one past the pools
    c.tables[2, 18] = -1               # its last block
    c.tables[3, 0] = 2 ** 31 - 1
    bad_lens = list(lens)
    bad_lens[4] = c.max_blocks * T + 1
    bad_lens[5] = -3
    c.upload()
    c.lens_dev.copy_(torch.tensor(bad_lens, dtype=torch.int32))
    c.call(splits)
    c.check(skip=(1, 2, 3, 4, 5))
    assert torch.isnan(c.out[[1, 2, 3, 4, 5]].float()).all()


def test_nan_reaches_the_heads_that_read_it(torch_cuda):
    torch = torch_cuda
    say("decode mxfp4 NaN groups and queries")
    heads, group, dim = 2, 3, 128
    c = Case(torch, [200, 200, 200, 200], heads, group, dim, seed=9)
    slot = lambda b, t: int(c.tables[b, t // T]) * T + t % T  # noqa: E731
    views = c.views()
    views[2][M.scale_at([slot(0, 30)], heads, dim)[0, 1, 2]] = 255   # K of KV head 1: every output of its query heads
    views[3][M.scale_at([slot(1, 77)], heads, dim)[0, 0, 3]] = 255   # V of KV head 0: dims 96..127
    c.upload()
    c.q[2, 4, 17] = float("nan")
    c.call(4)
    torch.cuda.synchronize()
    nan = torch.isnan(c.out.float()).cpu().numpy()
    want = np.zeros(nan.shape, bool)
    want[0, group:] = True
    want[1, :group, 96:] = True
    want[2, 4] = True
    np.testing.assert_array_equal(nan, want)


def test_infinite_queries_do_not_give_numbers(torch_cuda):
    """Softmax over scores of which one is +infinity, or all are -infinity, is NaN."""
    torch = torch_cuda
    say("decode mxfp4 infinite queries")
    c = Case(torch, [100], 1, 2, 64, seed=10)
    c.codes[:] = np.where(c.codes & 7, c.codes, c.codes | 1)   # no zero codes,
    c.codes[:] = np.where(c.codes & 0x70, c.codes, c.codes | 0x10)
    c.codes &= 0x77                                              # none negative
    c.upload()
    c.q[0, 0] = 0
    c.q[0, 0, 5] = float("inf")
    c.q[0, 1] = 0
    c.q[0, 1, 5] = float("-inf")
    c.call(1)
    torch.cuda.synchronize()
    assert torch.isnan(c.out.float()).all()


def test_pool_offsets_beyond_32_bits(torch_cuda):
    torch = torch_cuda
    heads, group, dim = 8, 2, 128
    half = M.half_bytes(heads, dim)
    blocks = (5 << 30) // half
    say("decode mxfp4 pools of 5 GiB")
    rng = np.random.default_rng(11)
    c = Case(torch, [500], heads, group, dim, seed=11)
    far = (blocks - 1 - rng.permutation(4000)[:c.max_blocks]).astype(np.int64)
    pools = [torch.zeros(blocks * per, dtype=torch.uint8, device="cuda") for per in (half, half, half // 16, half // 16)]
    for pool, view, per in zip(pools, c.views(), (half, half, half // 16, half // 16)):
        src = torch.from_numpy(view[: c.blocks * per].reshape(c.blocks, per)[c.tables[0]].copy()).cuda()
        pool.view(blocks, per)[torch.from_numpy(far).cuda()] = src
    tables = torch.from_numpy(far.astype(np.int32)).cuda()
    ws = c.workspace(8)
    P.paged_decode_mxfp4(pools[0].data_ptr(), pools[1].data_ptr(), pools[0].numel(), pools[2].data_ptr(), pools[3].data_ptr(), pools[2].numel(),
                         heads, dim, c.q.data_ptr(), c.out.data_ptr(), 1, heads * group, tables.data_ptr(), c.lens_dev.data_ptr(), c.max_blocks,
                         8, ws.data_ptr(), ws.numel(), stream=stream_ptr(torch))
    c.check()


@pytest.mark.parametrize("spare", [0, 17])
def test_longest_sequence_ends_inside_its_last_block(torch_cuda, spare):
    """2^31 - 1 - spare tokens: one block again and again, then another that is
    cut. The block's scores are 0; the last one's 64 above, so that all the others
    together weigh below 2^31 e^-64 < 2^-61; the token past the end's, 96. With equal
    scores the output is the mean of the last block's values that count: off by
    half a step of BF16 and, of 16 terms at most 6, by less than 2^-18."""
    torch = torch_cuda
    say("decode mxfp4 of 2^31 - 1 - %d tokens" % spare)
    rng = np.random.default_rng(3)
    n, dim = 2 ** 31 - 1 - spare, 64
    blocks, end = -(-n // T), (n - 1) % T + 1
    assert end < T
    k, v = np.zeros((2 * T, dim)), np.zeros((2 * T, dim))
    k[T:T + end], k[T + end:] = 8.0, 12.0
    v[T:] = rng.choice([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], (T, dim)) * rng.choice([-1.0, 1.0], (T, dim))
    v[T:, ::32] = 4.0
    rows = [torch.tensor(x, dtype=torch.bfloat16, device="cuda") for x in (k, v)]
    half = M.half_bytes(1, dim)
    pools = [torch.zeros(2 * size, dtype=torch.uint8, device="cuda") for size in (half, half, half // 16, half // 16)]
    slots = torch.arange(2 * T, dtype=torch.int32, device="cuda")
    P.scatter_kv_mxfp4(rows[0].data_ptr(), rows[1].data_ptr(), P.PBE_IN_BF16, 2 * T, slots.data_ptr(), 1, dim,
                       *(x for pool in pools for x in (pool.data_ptr(), pool.numel())), stream=stream_ptr(torch))
    tables = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    tables[-1] = 1
    q, out = torch.ones(1, 1, dim, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, dim, dtype=torch.bfloat16, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    ws = torch.full((P.decode_mxfp4_workspace_bytes(1, 1, dim, 1024),), 0xff, dtype=torch.uint8, device="cuda")
    P.paged_decode_mxfp4(pools[0].data_ptr(), pools[1].data_ptr(), pools[0].numel(), pools[2].data_ptr(), pools[3].data_ptr(), pools[2].numel(),
                         1, dim, q.data_ptr(), out.data_ptr(), 1, 1, tables.data_ptr(), lens.data_ptr(), blocks, 0, ws.data_ptr(), ws.numel(),
                         stream=stream_ptr(torch))
    torch.cuda.synchronize()
    want = v[T:T + end].mean(0)
    off = np.abs(out.double().cpu().numpy()[0, 0] - want)
    assert (off <= 2.0 ** -8 * np.abs(want) + 2.0 ** -18).all(), off.max()


def test_decode_replays_from_a_graph_as_lengths_grow(torch_cuda):
    torch = torch_cuda
    say("decode mxfp4 in a graph")
    c = Case(torch, [900, 500, 64, 1], 2, 6, 128, seed=12)
    ws = c.workspace(8)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            c.call(8, workspace=ws, stream=side.cuda_stream)
    full = list(c.lens)
    for rep in range(4):
        c.lens = [max(1, n - 13 * (3 - rep)) for n in full]
        c.lens_dev.copy_(torch.tensor(c.lens, dtype=torch.int32))
        ws.fill_(0xff)
        c.out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        c.check()
    c.out.fill_(5.0)
    c.call(8, workspace=ws)  # the same workspace, called
    c.check()


def test_two_calls_at_once_on_their_own_streams(torch_cuda):
    torch = torch_cuda
    say("decode mxfp4 on two streams")
    cases = [Case(torch, [2000, 31, 700], 2, 6, 128, seed=13), Case(torch, [1500, 1500], 4, 2, 64, seed=14)]
    streams = [torch.cuda.Stream() for _ in cases]
    spaces = [c.workspace(16) for c in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s, ws in zip(cases, streams, spaces):
            c.call(16, workspace=ws, stream=s.cuda_stream)
    for c in cases:
        c.check()


def test_workspace_rules(torch_cuda):
    torch = torch_cuda
    say("decode mxfp4 workspace")
    c = Case(torch, [900, 40], 2, 6, 128, seed=15)
    tight = torch.empty(P.decode_mxfp4_workspace_bytes(2, 12, 128, 3), dtype=torch.uint8, device="cuda")
    want = None
    for splits in (0, 3):
        c.out.fill_(5.0)
        c.call(splits, workspace=tight)
        want = c.check(want=want)
    with pytest.raises(P.PbeError) as e:
        c.call(4, workspace=tight)
    assert e.value.code == P.PBE_ERR_INVALID

    class Nothing:
        data_ptr, numel = staticmethod(lambda: 0), staticmethod(lambda: 0)
    for splits in (0, 1):  # no workspace: one piece
        c.out.fill_(5.0)
        c.call(splits, workspace=Nothing)
        c.check(want=want)
    host = np.zeros(1 << 20, np.uint8)

    class Pageable:
        data_ptr, numel = staticmethod(lambda: (host.ctypes.data + 15) // 16 * 16), staticmethod(lambda: 1 << 19)
    with pytest.raises(P.PbeError) as e:
        c.call(4, workspace=Pageable)
    assert e.value.code == P.PBE_ERR_INVALID
    pinned = torch.empty(P.decode_mxfp4_workspace_bytes(2, 12, 128, 4), dtype=torch.uint8).pin_memory()
    with pytest.raises(P.PbeError) as e:  # its tickets are device atomics
        c.call(4, workspace=pinned)
    assert e.value.code == P.PBE_ERR_INVALID


def test_two_graphs_share_a_workspace(torch_cuda):
    """Replayed one after the other, with other work in the workspace between."""
    torch = torch_cuda
    say("decode mxfp4 two graphs, one workspace")
    cases = [Case(torch, [700, 90, 1500], 2, 6, 128, seed=16), Case(torch, [64, 900], 4, 12, 64, seed=17)]
    ws = torch.full((max(c.workspace(12).numel() for c in cases),), 0x55, dtype=torch.uint8, device="cuda")
    graphs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.stream(side):
            with torch.cuda.graph(graphs[-1], stream=side):
                c.call(12, workspace=ws, stream=side.cuda_stream)
    want = [None, None]
    for rep in range(4):
        if rep == 2:
            ws.random_(0, 256)
        for i in (0, 1, 1, 0):
            cases[i].out.fill_(5.0)
            torch.cuda.synchronize()
            graphs[i].replay()
            want[i] = cases[i].check(want=want[i])
        cases[0].call(5, workspace=ws)
        cases[0].check(want=want[0])
