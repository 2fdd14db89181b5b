"""The operators of a 4-bit decode worker together, as a worker runs them: a
prefill chunk's tables, rows and pages, the pages handed over, and decode steps
whose tables, rows, pages and attention run from one captured graph."""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import mxfp4 as M
from oracle import step as S
from tests.conftest import say
from tests.gpu_util import stream_ptr

pytestmark = pytest.mark.gpu

B = 16


class Worker:
    """Requests with their pages in a page-major arena of one of `layers` layers."""

    def __init__(self, torch, lens, heads, group, dim, layers=2, layer=1, room=64, seed=0):
        rng = np.random.default_rng(seed)
        self.torch, self.lens, self.heads, self.group, self.dim, self.layers = torch, list(lens), heads, group, dim, layers
        counts = [-(-(n + room) // B) for n in lens]
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.n_pages = 2 * int(self.starts[-1]) + 5
        self.perm = rng.permutation(self.n_pages)
        self.pages = (self.perm[: self.starts[-1]] * 2 * layers).astype(np.int32)
        self.max_blocks, self.batch, self.layer = max(counts), len(lens), layer
        self.half = M.half_bytes(heads, dim)
        self.codes = torch.zeros(self.n_pages * 2 * layers * self.half, dtype=torch.uint8, device="cuda")
        self.scales = torch.zeros(self.codes.numel() // 16, dtype=torch.uint8, device="cuda")
        self.dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")
        angle = np.arange(4096)[:, None] * 1e4 ** (-np.arange(0, dim, 2) / dim)
        self.table = torch.tensor(np.concatenate([np.cos(angle), np.sin(angle)], 1), dtype=torch.float32, device="cuda")
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.w = (1 + 0.2 * torch.randn((2, dim), generator=g, device="cuda")).to(torch.bfloat16)
        self.gen = g
        self.d_pages, self.d_starts = self.dev(self.pages), self.dev(self.starts)
        empty = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.tables, self.seq_lens, self.token_starts = empty(self.batch * self.max_blocks), empty(self.batch), empty(self.batch + 1)
        self.workspace = torch.full((P.decode_mxfp4_workspace_bytes(self.batch, heads * group, dim, 8),), 0xff, dtype=torch.uint8, device="cuda")

    def pools(self):
        a, s = self.codes, self.scales
        k, v = 2 * self.layer * self.half, (2 * self.layer + 1) * self.half
        return (a.data_ptr() + k, a.numel() - k, a.data_ptr() + v, a.numel() - v, s.data_ptr() + k // 16, s.numel() - k // 16,
                s.data_ptr() + v // 16, s.numel() - v // 16)

    def rows(self, n):
        q_heads = self.heads * self.group
        return (self.torch.randn((n, (q_heads + 2 * self.heads) * self.dim), generator=self.gen, device="cuda") * 1.3).to(self.torch.bfloat16)

    def build(self, cached, new, slots, positions, stream):
        P.build_step_tables(self.d_pages.data_ptr(), len(self.pages), self.d_starts.data_ptr(), cached.data_ptr(),
                            new.data_ptr() if new is not None else 0, self.batch, B, self.tables.data_ptr(), self.max_blocks,
                            self.seq_lens.data_ptr(), self.token_starts.data_ptr(), slots.data_ptr(), positions.data_ptr(), len(slots), stream=stream)

    def write(self, qkv, slots, positions, q_out, stream, kind=P.PBE_KV_MXFP4, pools=None):
        q_heads, dim = self.heads * self.group, self.dim
        at, width = qkv.data_ptr(), qkv.shape[1]
        P.qk_norm_rope_scatter(at, width, at + 2 * q_heads * dim, width, at + 2 * (q_heads + self.heads) * dim, width, P.PBE_IN_BF16, len(slots),
                               q_heads, self.heads, dim, self.w[0].data_ptr(), self.w[1].data_ptr(), 1e-6, positions.data_ptr(),
                               self.table.data_ptr(), 4096, dim, P.PBE_ROPE_HALVES, slots.data_ptr(), B, kind, q_out.data_ptr(),
                               *(pools or self.pools()), stream=stream)

    def read(self, q, out, stream):
        k, kb, v, vb, ks, ksb, vs, vsb = self.pools()
        P.paged_decode_mxfp4(k, v, vb, ks, vs, vsb, self.heads, self.dim, q.data_ptr(), out.data_ptr(), self.batch, self.heads * self.group,
                             self.tables.data_ptr(), self.seq_lens.data_ptr(), self.max_blocks, 8, self.workspace.data_ptr(),
                             self.workspace.numel(), stream=stream)

    def host_pools(self):
        a, s = self.codes.cpu().numpy(), self.scales.cpu().numpy()
        k, v = 2 * self.layer * self.half, (2 * self.layer + 1) * self.half
        return a[k:], a[v:], s[k // 16:], s[v // 16:]

    def prefill(self, stream, padded=7):
        torch, n = self.torch, sum(self.lens) + padded
        slots, positions = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        self.build(self.dev([0] * self.batch), self.dev(self.lens), slots, positions, stream)
        qkv, q_out = self.rows(n), torch.full((n, self.heads * self.group, self.dim), 3.0, dtype=torch.bfloat16, device="cuda")
        self.write(qkv, slots, positions, q_out, stream)
        return qkv, slots, positions, q_out

    def check_attention(self, q, out, lens):
        o, spread, size, reach = M.decode(q.double().cpu().numpy(), self.host_pools(), self.tables.cpu().numpy().reshape(self.batch, -1), lens,
                                          self.heads)
        n = np.array(lens)[:, None, None]
        e = (2 * (self.dim + 16) * 2.0 ** -24 * reach + 2.0 ** -20)[..., None]   # the reader's bound, as its own tests derive it
        bound = 2.0 ** -8 * np.abs(o) + (2.0 ** -8 / (1 - 2.0 ** -8) + e) * spread + (n / 32 + 64) * 2.0 ** -23 * size + 2.0 ** -110
        assert (np.abs(out.double().cpu().numpy() - o) <= bound).all()


@pytest.mark.parametrize("heads,group,dim", [(2, 6, 128), (2, 7, 64), (4, 7, 128)])
def test_prefill_pages_handed_over_and_decoded(torch_cuda, heads, group, dim):
    torch = torch_cuda
    say(f"mxfp4 prefill, handoff, decode H={heads}x{group} D={dim}")
    lens = [130, 1, 16, 300, 47]
    w = Worker(torch, lens, heads, group, dim, seed=dim + heads)
    stream = stream_ptr(torch)
    qkv, slots, positions, q_out = w.prefill(stream)
    torch.cuda.synchronize()
    want = S.tables(w.pages, w.starts, [0] * 5, lens, B, w.max_blocks, len(slots))
    for got, x in zip((w.tables, w.seq_lens, w.token_starts, slots, positions), want):
        np.testing.assert_array_equal(got.cpu().numpy(), x.ravel())
    n = sum(lens)
    assert (q_out[n:] == 3.0).all()                        # padding rows
    # what the pages hold is what the MXFP4 writer makes of the BF16 rows
    bf16 = torch.zeros((2, len(w.pages) * B, heads, dim), dtype=torch.bfloat16, device="cuda")
    local = torch.full((len(slots),), -1, dtype=torch.int32, device="cuda")
    local[:n] = torch.arange(n, dtype=torch.int32, device="cuda")
    size = bf16[0].numel() * 2
    w.write(qkv, local, positions, torch.empty_like(q_out), stream, kind=P.PBE_KV_BF16,
            pools=(bf16[0].data_ptr(), size, bf16[1].data_ptr(), size))
    back = torch.zeros((2, n, heads, dim), dtype=torch.bfloat16, device="cuda")
    P.gather_kv_mxfp4(*w.pools(), slots.data_ptr(), n, heads, dim, back[0].data_ptr(), back[1].data_ptr(), stream=stream)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(back.double().cpu().numpy(), M.values(*M.quantise(bf16[:, :n].double().cpu().numpy())))
    # each request's last query over its pages, before and after the handoff
    q = q_out[torch.tensor(np.cumsum(lens) - 1, device="cuda")].contiguous()
    out = torch.zeros_like(q)
    w.read(q, out, stream)
    torch.cuda.synchronize()
    w.check_attention(q, out, lens)
    dst = (w.perm[w.starts[-1]: 2 * w.starts[-1]] * 2 * w.layers).astype(np.int32)
    for buf, d in ((w.codes, dim // 2), (w.scales, dim // 32)):
        kv, view = P.shape(w.layers, heads, d), P.view_of(buf.data_ptr(), buf.numel())
        with P.RunList.bf16(view, view, P.build_runs(w.pages, dst, kv, 1), kv, elem_bytes=1) as run:
            run.copy(stream)
            torch.cuda.synchronize()
    w.d_pages = w.dev(dst)
    spare = torch.zeros(5, dtype=torch.int32, device="cuda")
    w.build(w.dev(lens), w.dev([0] * 5), spare, spare.clone(), stream)
    again = torch.zeros_like(q)
    w.read(q, again, stream)
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


def test_decode_steps_replay_from_one_graph(torch_cuda):
    """Tables, rows, pages and attention of a step in one graph; a host that adds
    one to the cached lengths between replays decodes on and on. Another worker
    runs the same steps call by call."""
    torch = torch_cuda
    say("mxfp4 decode steps in a graph")
    lens, heads, group, dim, slots_n = [33, 15, 16, 200], 2, 6, 128, 6   # captured for six rows, two of them padding
    pair = [Worker(torch, lens, heads, group, dim, seed=21) for _ in range(2)]
    stream = stream_ptr(torch)
    for w in pair:
        w.prefill(stream)
        w.cached = w.dev(lens)
        w.slots, w.positions = (torch.zeros(slots_n, dtype=torch.int32, device="cuda") for _ in range(2))
        w.qkv = w.rows(slots_n)
        w.q = torch.full((slots_n, heads * group, dim), 3.0, dtype=torch.bfloat16, device="cuda")
        w.out = torch.zeros((len(lens), heads * group, dim), dtype=torch.bfloat16, device="cuda")
    a, b = pair
    torch.cuda.synchronize()
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)

    def step(w, s):
        w.build(w.cached, None, w.slots, w.positions, s)
        w.write(w.qkv, w.slots, w.positions, w.q, s)
        w.read(w.q, w.out, s)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(a, side.cuda_stream)
    for rep in range(20):   # past a page's end for every request
        x = a.rows(slots_n)
        for w in pair:
            w.qkv.copy_(x)
            w.out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        step(b, stream)
        torch.cuda.synchronize()
        assert (a.q[4:] == 3.0).all()
        for name in ("tables", "seq_lens", "token_starts", "slots", "positions", "codes", "scales"):
            assert torch.equal(getattr(a, name), getattr(b, name)), (rep, name)
        assert torch.equal(a.out.view(torch.int16), b.out.view(torch.int16)), rep
        if rep % 7 == 0:
            a.check_attention(a.q[:4], a.out, [n + rep + 1 for n in lens])
        for w in pair:
            w.cached.add_(1)
