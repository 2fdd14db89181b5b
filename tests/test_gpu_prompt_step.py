"""The prompt reader and the page movers as a worker runs them, with the step tables,
the page writer, the decode reader and the handoff beside them: a prompt in chunks,
requests that fork into drafts, drafts checked, the losers' pages given up, the pages
compacted and handed over."""
import numpy as np
import pytest

import pbe_handoff as P
from tests.conftest import say
from tests.gpu_util import stream_ptr
from tests.test_gpu_mxfp4_step import B, Worker
from tests.test_gpu_prompt import within

pytestmark = pytest.mark.gpu


class Prompts(Worker):
    """A worker over MXFP4 pages of a page-major arena of `layers` layers."""

    def planes(self):
        a, s = self.codes, self.scales
        page = 2 * self.layers * self.half
        return P.page_planes([(P.view_of(a.data_ptr(), a.numel()), page), (P.view_of(s.data_ptr(), s.numel()), page // 16)])

    def attend(self, q, out, tables, lens, starts, rows, stream):
        k, kb, v, vb, ks, ksb, vs, vsb = self.pools()
        batch, q_heads = len(lens), self.heads * self.group
        if getattr(self, "ws", None) is None:
            self.ws = self.torch.full((1 << 26,), 0xff, dtype=self.torch.uint8, device="cuda")
        P.paged_prompt_attention(k, v, vb, ks, vs, vsb, P.PBE_KV_MXFP4, self.heads, self.dim, q.data_ptr(), out.data_ptr(), rows, starts.data_ptr(),
                                 batch, q_heads, tables.data_ptr(), lens.data_ptr(), tables.numel() // batch, self.ws.data_ptr(), self.ws.numel(),
                                 stream=stream)

    def held(self, tables, b, n):
        """K and V of a sequence's n tokens, in 64 bits."""
        torch = self.torch
        t = torch.arange(n, device="cuda")
        slots = (tables.view(len(tables), -1)[b][t // B] * B + t % B).to(torch.int32)
        back = torch.zeros((2, n, self.heads, self.dim), dtype=torch.bfloat16, device="cuda")
        P.gather_kv_mxfp4(*self.pools(), slots.data_ptr(), n, self.heads, self.dim, back[0].data_ptr(), back[1].data_ptr(), stream=stream_ptr(torch))
        torch.cuda.synchronize()
        return back.double().cpu().numpy()

    def check(self, q, out, tables, lens, news):
        at = 0
        for b, (n, m) in enumerate(zip(lens, news)):
            k, v = self.held(tables, b, n)
            within(out[at:at + m].double().cpu().numpy(), q[at:at + m].double().cpu().numpy(), k, v)
            at += m


@pytest.mark.parametrize("heads,group,dim", [(2, 6, 128), (2, 7, 64)])
def test_chunks_forks_drafts_compaction_and_handoff(torch_cuda, heads, group, dim):
    torch = torch_cuda
    say(f"prompt chunks, forks, drafts, compaction, handoff H={heads}x{group} D={dim}")
    stream = stream_ptr(torch)
    lens = [150, 33, 16]
    w = Prompts(torch, lens, heads, group, dim, seed=dim)
    # the prompts, in chunks of at most 64 tokens
    cached = [0, 0, 0]
    while cached != lens:
        news = [min(64, n - c) for n, c in zip(lens, cached)]
        n = sum(news) + 5
        slots, positions = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        w.build(w.dev(cached), w.dev(news), slots, positions, stream)
        q = torch.full((n, heads * group, dim), 3.0, dtype=torch.bfloat16, device="cuda")
        w.write(w.rows(n), slots, positions, q, stream)
        out = torch.full_like(q, 9.0)
        w.attend(q, out, w.tables, w.seq_lens, w.token_starts, n, stream)
        cached = [c + x for c, x in zip(cached, news)]
        torch.cuda.synchronize()
        w.check(q, out, w.tables.view(3, -1), cached, news)
        assert (out[sum(news):] == 9.0).all()
    # two drafts of three tokens each from the first two, the third goes on by itself
    parents, news, stride = [1, 0, 0, 2, 1], [3, 3, 3, 3, 3], 2 * w.layers
    i32 = lambda *shape: torch.full(shape, 77, dtype=torch.int32, device="cuda")  # noqa: E731

    def fork(tables, lens, parents, news):
        rows, width = len(parents), tables.shape[1]
        t, n, counts = i32(rows, width), i32(rows), i32(2)
        ws = torch.full((P.fork_pages_workspace_bytes(w.n_pages, len(lens), rows),), 0xff, dtype=torch.uint8, device="cuda")
        p, x = w.dev(parents), w.dev(news)
        P.fork_pages(w.planes(), w.n_pages, stride, B, tables.data_ptr(), lens.data_ptr(), len(lens), p.data_ptr(), x.data_ptr(), rows, width, 0,
                     t.data_ptr(), n.data_ptr(), counts.data_ptr(), ws.data_ptr(), ws.numel(), stream=stream)
        torch.cuda.synchronize()
        return t, n, counts

    before = {b: w.held(w.tables.view(3, -1), b, n) for b, n in enumerate(lens)}
    tables, kept, counts = fork(w.tables.view(3, -1), w.seq_lens, parents, news)
    assert counts[0] <= counts[1] and kept.tolist() == [33, 150, 150, 16, 33]
    for b, p in enumerate(parents):
        np.testing.assert_array_equal(w.held(tables, b, lens[p]), before[p])
    positions = (kept[:, None] + torch.arange(3, device="cuda")).to(torch.int32)
    slots = (torch.gather(tables, 1, (positions // B).long()) * B + positions % B).to(torch.int32)
    assert len(set(slots.flatten().tolist())) == 15            # children write to pages of their own
    q = torch.zeros((15, heads * group, dim), dtype=torch.bfloat16, device="cuda")
    w.write(w.rows(15), slots.flatten(), positions.flatten(), q, stream)
    out, full = torch.full_like(q, 9.0), kept + 3
    w.attend(q, out, tables, full, torch.arange(0, 16, 3, dtype=torch.int32, device="cuda"), 15, stream)
    torch.cuda.synchronize()
    w.check(q, out, tables, full.tolist(), [3] * 5)
    # of each pair one is kept, with two, three and one of its drafted tokens
    accepted = torch.tensor([35, 153, 152, 17, 36], dtype=torch.int32, device="cuda")
    tables, kept, _ = fork(tables, accepted, [2, 3, 4], [0, 0, 0])
    assert kept.tolist() == [152, 17, 36]
    one = torch.zeros((3, heads * group, dim), dtype=torch.bfloat16, device="cuda")
    queries = q[:3].contiguous()
    w.tables, w.seq_lens = tables, kept
    w.max_blocks = tables.shape[1]
    w.read(queries, one, stream)
    # a decode row is a prompt row of one token
    same = torch.zeros_like(one)
    w.attend(queries, same, tables, kept, torch.arange(4, dtype=torch.int32, device="cuda"), 3, stream)
    torch.cuda.synchronize()
    w.check(queries, one, tables, kept.tolist(), [1] * 3)
    w.check(queries, same, tables, kept.tolist(), [1] * 3)
    # the pages to the front, one stretch; the same outputs
    moved, counts = i32(*tables.shape), i32(2)
    ws = torch.full((P.compact_pages_workspace_bytes(w.n_pages),), 0xff, dtype=torch.uint8, device="cuda")
    P.compact_pages(w.planes(), w.n_pages, stride, tables.data_ptr(), 3, tables.shape[1], 0, moved.data_ptr(), 0, counts.data_ptr(), ws.data_ptr(),
                    ws.numel(), stream=stream)
    again = torch.zeros_like(one)
    w.tables = moved
    w.read(queries, again, stream)
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), one.view(torch.int16))
    total = int(counts[0])
    assert sorted((moved[moved >= 0] // stride).tolist()) == list(range(total)) and total == 10 + 2 + 3
    # and handed over to the pages behind, as one run a plane
    src, dst = (np.arange(a, a + total, dtype=np.int32) * stride for a in (0, total))
    for buf, d in ((w.codes, dim // 2), (w.scales, dim // 32)):
        kv, view = P.shape(w.layers, heads, d), P.view_of(buf.data_ptr(), buf.numel())
        runs = P.build_runs(src, dst, kv, 1)
        assert len(runs) == 1
        with P.RunList.bf16(view, view, runs, kv, elem_bytes=1) as run:
            run.copy(stream)
            torch.cuda.synchronize()
    w.tables = torch.where(moved >= 0, moved + total * stride, moved)
    again.zero_()
    w.read(queries, again, stream)
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), one.view(torch.int16))


def test_a_captured_step_forks_and_checks_drafts(torch_cuda):
    """Fork, page writes and attention of two drafted tokens a request in one graph,
    replayed while the parents change, against another worker's calls."""
    torch = torch_cuda
    say("forks and drafts in a graph")
    lens, heads, group, dim, rows = [40, 31, 16, 200], 2, 6, 128, 4
    pair = [Prompts(torch, lens, heads, group, dim, seed=7) for _ in range(2)]
    stream = stream_ptr(torch)
    for w in pair:
        w.prefill(stream)
        w.now, w.lens_now = w.tables.view(rows, -1).clone(), w.seq_lens.clone()
        w.next, w.next_lens, w.counts = torch.zeros_like(w.now), torch.zeros_like(w.lens_now), w.dev([0, 0])
        w.parents, w.news, w.every = w.dev(range(rows)), w.dev([2] * rows), w.dev(range(0, 2 * rows + 1, 2))
        w.fork_ws = torch.full((P.fork_pages_workspace_bytes(w.n_pages, rows, rows),), 0xff, dtype=torch.uint8, device="cuda")
        w.qkv = w.rows(2 * rows)
        w.q = torch.zeros((2 * rows, heads * group, dim), dtype=torch.bfloat16, device="cuda")
        w.out = torch.zeros_like(w.q)
        w.ws = torch.full((1 << 26,), 0xff, dtype=torch.uint8, device="cuda")
        w.step = torch.arange(2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()

    def step(w, s):
        P.fork_pages(w.planes(), w.n_pages, 2 * w.layers, B, w.now.data_ptr(), w.lens_now.data_ptr(), rows, w.parents.data_ptr(), w.news.data_ptr(), rows,
                     w.now.shape[1], 0, w.next.data_ptr(), w.next_lens.data_ptr(), w.counts.data_ptr(), w.fork_ws.data_ptr(), w.fork_ws.numel(), stream=s)
        positions = w.next_lens[:, None] + w.step
        slots = torch.gather(w.next, 1, (positions // B).long()) * B + positions % B
        w.write(w.qkv, slots.flatten(), positions.flatten(), w.q, s)
        w.now.copy_(w.next)
        w.lens_now.copy_(w.next_lens + 2)
        w.attend(w.q, w.out, w.now, w.lens_now, w.every, 2 * rows, s)
        w.used = slots, positions  # alive until replays end

    a, b = pair
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(a, side.cuda_stream)
    kept = a.used
    rng = np.random.default_rng(1)
    for rep in range(12):   # past pages' ends
        x, parents = a.rows(2 * rows), rng.integers(0, rows, rows) if rep % 3 else np.arange(rows)
        for w in pair:
            w.qkv.copy_(x)
            w.parents.copy_(w.dev(parents))
            w.out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        step(b, stream)
        torch.cuda.synchronize()
        assert int(a.counts[0]) <= int(a.counts[1])
        for x, y in ((a.now, b.now), (a.lens_now, b.lens_now), (a.out.view(torch.int16), b.out.view(torch.int16)), (a.codes, b.codes), (a.scales, b.scales)):
            assert torch.equal(x, y), rep
        if rep % 4 == 3:
            a.check(a.q, a.out, a.now, a.lens_now.tolist(), [2] * rows)
    del kept
