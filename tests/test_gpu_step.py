"""pbe_build_step_tables against the oracle: every array whole, canaries behind
each, for requests that are ordinary, empty, long, and wrong in each way."""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import step as S
from tests.conftest import say
from tests.gpu_util import stream_ptr

pytestmark = pytest.mark.gpu

CANARY = -77


class Step:
    def __init__(self, torch, pages, starts, cached, new, block_size, max_blocks, max_tokens):
        self.torch, self.case = torch, (pages, starts, cached, new, block_size, max_blocks, max_tokens)
        dev = lambda a: None if a is None else torch.tensor(np.asarray(a, np.int32), device="cuda")  # noqa: E731
        self.pages, self.starts, self.cached, self.new = dev(pages), dev(starts), dev(cached), dev(new)
        batch = len(cached)
        self.sizes = [batch * max_blocks, batch, batch + 1, max_tokens, max_tokens]
        self.out = [torch.full((n + 3,), CANARY, dtype=torch.int32, device="cuda") for n in self.sizes]

    def call(self, stream):
        t, lens, first, slots, pos = (o.data_ptr() for o in self.out)
        _, _, cached, _, block_size, max_blocks, max_tokens = self.case
        P.build_step_tables(self.pages.data_ptr() if len(self.pages) else 0, len(self.pages), self.starts.data_ptr(), self.cached.data_ptr(),
                            self.new.data_ptr() if self.new is not None else 0, len(cached), block_size, t, max_blocks, lens, first, slots, pos,
                            max_tokens, stream=stream)

    def check(self, note=""):
        self.torch.cuda.synchronize()
        want = S.tables(*self.case)
        for name, o, n, w in zip(("tables", "seq_lens", "token_starts", "slots", "positions"), self.out, self.sizes, want):
            got = o.cpu().numpy()
            np.testing.assert_array_equal(got[:n], w.ravel(), err_msg=f"{name} {note}")
            assert (got[n:] == CANARY).all(), (name, note)


def requests(rng, batch, most, chunk, block_size, spare=2):
    """Page lists, starts, cached and new lengths of ordinary requests."""
    cached = rng.integers(0, most, batch)
    new = np.where(rng.random(batch) < 0.3, rng.integers(0, chunk + 1, batch), 1)
    counts = -(-(cached + new) // block_size) + rng.integers(0, spare + 1, batch)
    starts = np.concatenate([[0], np.cumsum(counts)])
    pages = rng.permutation(int(starts[-1]) + 50)[: int(starts[-1])] * 6
    return pages, starts, cached, new


@pytest.mark.parametrize("batch,most,chunk,block_size,padded", [
    (1, 1, 1, 16, 0), (1, 5000, 1, 16, 3), (7, 100, 33, 16, 0), (64, 700, 40, 16, 100), (63, 90, 5, 1, 1), (65, 300, 200, 7, 0),
    (1023, 40, 3, 16, 5), (1024, 40, 3, 16, 0), (1025, 40, 3, 16, 70), (5000, 60, 4, 32, 0), (3, 9000, 6001, 16, 11), (200, 33, 0, 64, 1)])
def test_step_tables_match_the_oracle(torch_cuda, batch, most, chunk, block_size, padded):
    torch = torch_cuda
    say(f"step tables batch={batch} most={most} chunk={chunk} block={block_size} padded={padded}")
    rng = np.random.default_rng(batch + most)
    pages, starts, cached, new = requests(rng, batch, most, chunk, block_size)
    max_blocks = max(1, int(np.diff(starts).max()) - 1)
    s = Step(torch, pages, starts, cached, new, block_size, max_blocks, max(1, int(new.sum()) + padded))
    s.call(stream_ptr(torch))
    s.check()


def test_decode_step_without_new_lengths(torch_cuda):
    """new_lens NULL is one token each: the tables a host manager builds for its requests."""
    torch = torch_cuda
    say("step tables, one token each")
    cached = np.array([0, 15, 16, 17, 4095, 1])
    counts = cached // 16 + 1
    starts = np.concatenate([[0], np.cumsum(counts)])
    pages = np.random.default_rng(1).permutation(int(starts[-1])) * 56
    s = Step(torch, pages, starts, cached, None, 16, int(counts.max()), 6)
    s.call(stream_ptr(torch))
    s.check()
    slots = s.out[3].cpu().numpy()[:6]
    assert slots.tolist() == [int(pages[starts[b + 1] - 1]) * 16 + int(cached[b]) % 16 for b in range(6)]


def test_wrong_requests_do_not_touch_the_others(torch_cuda):
    torch = torch_cuda
    say("step tables, wrong requests among right ones")
    big = S.INT32_MAX
    pages = [4, 5, 6, 7, -3, 9, 200000000, 11, 12, 13]
    #          ok  neg  neg  sum        needs   empty  neg   slot   zero
    #              cach new  too big    pages   list   page  big    length
    starts = [0, 2, 3, 4, 4, 4, 4, 6, 7, 7]
    cached = [20, -1, 5, big, 1, 0, 3, 2, 0]
    new = [5, 2, -4, 5, 1, 0, 30, 9, 0]
    s = Step(torch, pages, starts, cached, new, 16, 3, 60)
    s.call(stream_ptr(torch))
    s.check()
    lens = s.out[1].cpu().numpy()
    assert lens[:9].tolist() == [25, -1, -1, -1, -1, 0, -1, 11, 0]  # 3 + 30 tokens need three pages
    # lists out of order or beyond page_ids
    for bad in ([0, 2, 1, 4, 4, 4, 4, 6, 7, 7], [0, 2, 3, 4, 4, 4, 4, 6, 7, 11], [-1, 2, 3, 4, 4, 4, 4, 6, 7, 7]):
        s = Step(torch, pages, bad, cached, new, 16, 3, 60)
        s.call(stream_ptr(torch))
        s.check(str(bad))
    # rows past max_tokens: the request that crosses, and all behind it that add any
    s = Step(torch, pages, starts, [0] * 9, [5, 6, 3, 0, 0, 0, 4, 1, 0], 16, 3, 12)
    s.call(stream_ptr(torch))
    s.check("past max_tokens")
    # more tokens than 32 bits count
    s = Step(torch, pages, [0] * 10, [0] * 9, [big] * 9, 16, 3, 12)
    s.call(stream_ptr(torch))
    s.check("saturated starts")
    # no pages at all
    s = Step(torch, [], [0] * 10, [0] * 9, [0] * 9, 16, 3, 12)
    s.call(stream_ptr(torch))
    s.check("no pages")


def test_sums_beyond_32_bits_keep_earlier_requests(torch_cuda):
    """2,000 requests of 2^31 - 1 tokens behind ordinary ones."""
    torch = torch_cuda
    say("step tables, sums beyond 32 bits")
    n = 2100
    new = np.concatenate([np.ones(100), np.full(n - 100, S.INT32_MAX)]).astype(np.int64)
    starts = np.minimum(np.arange(n + 1), 100)
    s = Step(torch, np.arange(100), starts, np.zeros(n), new, 16, 2, 300)
    s.call(stream_ptr(torch))
    s.check()


def test_step_tables_replay_from_a_graph_with_new_lengths(torch_cuda):
    """A captured step follows lengths that change in place between replays."""
    torch = torch_cuda
    say("step tables in a graph")
    rng = np.random.default_rng(4)
    pages, starts, cached, new = requests(rng, 40, 300, 20, 16)
    s = Step(torch, pages, starts, cached * 0, new, 16, int(np.diff(starts).max()), int(new.sum()) + 40)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            s.call(side.cuda_stream)
    for rep in range(4):
        c = np.maximum(cached - 10 * rep, 0)
        n = np.where(rng.random(40) < 0.5, new, 0)
        s.cached.copy_(torch.tensor(c, dtype=torch.int32))
        s.new.copy_(torch.tensor(n, dtype=torch.int32))
        for o in s.out:
            o.fill_(CANARY)
        torch.cuda.synchronize()
        s.case = (pages, starts, c, n, *s.case[4:])
        graph.replay()
        s.check(f"replay {rep}")
