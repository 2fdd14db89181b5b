"""pbe_qk_norm_rope_scatter: queries and BF16 pages against the 64-bit oracle,
FP8 and MXFP4 pages bit for bit against the page writers on the same BF16 rows,
and everything that a call must leave alone.

Bound of a BF16 result z = a c - b s: half a step of the final rounding, 2^-8
|z|, and the FP32 error before it. That is at most 2^-18 (|a c| + |b s|): the
mean square of D <= 128 numbers sums 8 in a lane and 4 steps of lanes, 13
roundings of 2^-24, halved by the root; the root's own 2^-22, two products and
the weight's 3 x 2^-24, the rotation's 3 x 2^-24: below 20 x 2^-24 < 2^-19, and
twice that covers the second-order terms and the rounding of a value moved by it.
"""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import oracle as O
from oracle import mxfp4 as M
from oracle import step as S
from tests.conftest import say
from tests.gpu_util import stream_ptr

pytestmark = pytest.mark.gpu

B, CANARY = 16, 0x41


class Rope:
    def __init__(self, torch, n, heads, group, dim, rotary, f32=False, pairs=False, norm=(True, True), packed=True, blocks=None, seed=0, eps=1e-6):
        rng = np.random.default_rng(seed)
        self.torch, self.n, self.heads, self.group, self.dim = torch, n, heads, group, dim
        self.rotary, self.f32, self.pairs, self.eps, self.max_position = rotary, f32, pairs, eps, 5000
        self.blocks = blocks or -(-n // B) + 4
        q_heads = heads * group
        x = rng.standard_normal((n, q_heads + 2 * heads, dim)) * np.exp(rng.standard_normal((1, q_heads + 2 * heads, 1)))
        if n > 4:
            x[1, :, :] = 0.0
            x[2] *= 1e15
            x[3] *= 1e-12
        dtype = torch.float32 if f32 else torch.bfloat16
        x = torch.tensor(x, dtype=torch.float32).to(dtype)
        self.x = x.double().numpy()
        if packed:
            buf = x.reshape(n, -1).cuda()
            self.bufs = [buf]
            width, e = buf.shape[1], buf.element_size()
            self.rows = [(buf.data_ptr() + at * dim * e, width) for at in (0, q_heads, q_heads + heads)]
        else:  # rows of their own, with gaps
            self.bufs, self.rows = [], []
            for part, gap in ((x[:, :q_heads], 8), (x[:, q_heads:q_heads + heads], 0), (x[:, q_heads + heads:], 24)):
                buf = torch.full((n, part.shape[1] * dim + gap), 9.0, dtype=dtype)
                buf[:, :part.shape[1] * dim] = part.reshape(n, -1)
                self.bufs.append(buf.cuda())
                self.rows.append((self.bufs[-1].data_ptr(), buf.shape[1]))
        w = torch.tensor(1 + 0.3 * rng.standard_normal((2, dim)), dtype=torch.float32).to(dtype)
        self.w = [w[i].double().numpy() if norm[i] else None for i in range(2)]
        self.w_dev = [w[i].contiguous().cuda() if norm[i] else None for i in range(2)]
        angle = np.arange(self.max_position)[:, None] * 1e4 ** (-np.arange(0, rotary, 2) / max(rotary, 1))
        self.table = np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)
        self.table_dev = torch.from_numpy(self.table).cuda() if rotary else None
        self.positions = rng.integers(0, self.max_position, n).astype(np.int32)
        self.slots = rng.permutation(self.blocks * B)[:n].astype(np.int32)
        if n > 12:
            self.positions[7] = -1                    # padding
            self.positions[8] = self.max_position     # beyond the table
            self.positions[9] = 2 ** 31 - 1
            self.slots[10], self.slots[11], self.slots[12] = -1, self.blocks * B, 2 ** 31 - 1
        self.q_out = torch.full((n, q_heads, dim), 3.0, dtype=torch.bfloat16, device="cuda")

    def pools(self, kind):
        per = self.heads * self.dim * (B * 2 if kind == P.PBE_KV_BF16 else B if kind == P.PBE_KV_FP8_E4M3 else B // 2)
        sc = 0 if kind == P.PBE_KV_BF16 else self.heads * B * 4 if kind == P.PBE_KV_FP8_E4M3 else per // 16
        new = lambda size: self.torch.full((self.blocks * size + 64,), CANARY, dtype=self.torch.uint8, device="cuda")  # noqa: E731
        bufs = [new(per), new(per), new(sc), new(sc)]
        sizes = [self.blocks * per] * 2 + [self.blocks * sc] * 2
        return bufs, [v for b, size in zip(bufs, sizes) for v in (b.data_ptr() if size else 0, size)]

    def call(self, kind, args, stream):
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        self.pos_dev, self.slots_dev = self.torch.from_numpy(self.positions).cuda(), self.torch.from_numpy(self.slots).cuda()
        (q, qs), (k, ks), (v, vs) = self.rows
        P.qk_norm_rope_scatter(q, qs, k, ks, v, vs, P.PBE_IN_F32 if self.f32 else P.PBE_IN_BF16, self.n, self.heads * self.group, self.heads,
                               self.dim, ptr(self.w_dev[0]), ptr(self.w_dev[1]), self.eps, self.pos_dev.data_ptr(), ptr(self.table_dev),
                               self.max_position if self.rotary else 0, self.rotary, P.PBE_ROPE_PAIRS if self.pairs else P.PBE_ROPE_HALVES,
                               self.slots_dev.data_ptr(), B, kind, self.q_out.data_ptr(), *args, stream=stream)

    def written(self, t):
        in_table = self.rotary == 0 or self.positions[t] < self.max_position
        return self.positions[t] >= 0 and in_table and 0 <= self.slots[t] < self.blocks * B

    def check_bf16(self, bufs):
        torch, n, heads, dim = self.torch, self.n, self.heads, self.dim
        torch.cuda.synchronize()
        q_heads = heads * self.group
        q_got = self.q_out.double().cpu().numpy()
        size = self.blocks * B * heads * dim * 2
        pools = [b.cpu().numpy() for b in bufs[:2]]
        assert all((p[size:] == CANARY).all() for p in pools)
        got = [torch.from_numpy(p[:size].copy()).view(torch.bfloat16).double().numpy().reshape(-1, heads, dim) for p in pools]
        canary = torch.full((2,), CANARY, dtype=torch.uint8).view(torch.bfloat16).double().item()
        untouched = np.ones(len(got[0]), bool)
        for t in range(n):
            in_table = self.rotary == 0 or self.positions[t] < self.max_position
            line = self.table[self.positions[t]] if self.rotary and 0 <= self.positions[t] < self.max_position else np.zeros(self.rotary)
            parts = [(self.x[t, :q_heads], self.w[0]), (self.x[t, q_heads:q_heads + heads], self.w[1])]
            (q, q_size), (k, k_size) = (S.norm_rope(x, w, self.eps, line, self.rotary, self.pairs) for x, w in parts)
            if self.positions[t] < 0:
                assert (q_got[t] == 3.0).all(), t
            elif not in_table:
                assert np.isnan(q_got[t]).all(), t
            else:
                assert (np.abs(q_got[t] - q) <= 2.0 ** -8 * np.abs(q) + 2.0 ** -18 * q_size).all(), t
            if self.written(t):
                untouched[self.slots[t]] = False
                assert (np.abs(got[0][self.slots[t]] - k) <= 2.0 ** -8 * np.abs(k) + 2.0 ** -18 * k_size).all(), t
                v = torch.tensor(self.x[t, q_heads + heads:]).to(torch.float32).to(torch.bfloat16).double().numpy()
                np.testing.assert_array_equal(got[1][self.slots[t]], v)
        for g in got:
            assert (g[untouched] == canary).all()


@pytest.mark.parametrize("n", [1, 5, 61])
@pytest.mark.parametrize("heads,group,dim,rotary,pairs", [
    (2, 7, 64, 64, False), (2, 6, 128, 128, False), (4, 7, 128, 128, True), (2, 1, 64, 32, True), (1, 8, 128, 96, False), (3, 2, 64, 48, False),
    (1, 3, 64, 16, True), (2, 2, 128, 16, False), (1, 1, 128, 0, False), (1, 16, 128, 112, True)])
@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
def test_queries_and_bf16_pages_match_the_oracle(torch_cuda, n, heads, group, dim, rotary, pairs, f32):
    say(f"qk_norm_rope n={n} H={heads}x{group} D={dim} rot={rotary} pairs={pairs} f32={f32}")
    r = Rope(torch_cuda, n, heads, group, dim, rotary, f32, pairs, packed=n != 5, seed=n + rotary)
    bufs, args = r.pools(P.PBE_KV_BF16)
    r.call(P.PBE_KV_BF16, args, stream_ptr(torch_cuda))
    r.check_bf16(bufs)


@pytest.mark.parametrize("norm", [(False, False), (True, False), (False, True)])
def test_norms_are_optional_for_queries_and_keys(torch_cuda, norm):
    say(f"qk_norm_rope norm={norm}")
    r = Rope(torch_cuda, 20, 2, 3, 128, 128, norm=norm, seed=8)
    bufs, args = r.pools(P.PBE_KV_BF16)
    r.call(P.PBE_KV_BF16, args, stream_ptr(torch_cuda))
    r.check_bf16(bufs)


@pytest.mark.parametrize("n,heads,group,dim,rotary", [
    (700, 4, 7, 128, 128), (2100, 2, 3, 64, 64),          # a head at a time
    (1000, 4, 7, 128, 128), (3700, 2, 7, 64, 64), (1100, 3, 9, 128, 96),   # two
    (2800, 4, 7, 128, 128), (2001, 5, 7, 128, 64), (11000, 2, 7, 64, 64)])  # four
def test_long_prompts_take_runs_of_heads(torch_cuda, n, heads, group, dim, rotary):
    say(f"qk_norm_rope n={n} H={heads}x{group} D={dim}")
    r = Rope(torch_cuda, n, heads, group, dim, rotary, pairs=rotary == 64 and dim == 128, seed=n)
    bufs, args = r.pools(P.PBE_KV_BF16)
    r.call(P.PBE_KV_BF16, args, stream_ptr(torch_cuda))
    r.check_bf16(bufs)


@pytest.mark.parametrize("kind", [P.PBE_KV_FP8_E4M3, P.PBE_KV_MXFP4], ids=["fp8", "mxfp4"])
@pytest.mark.parametrize("n,heads,group,dim,f32", [(1, 2, 6, 128, False), (90, 2, 7, 64, False), (77, 4, 7, 128, True), (1600, 3, 5, 128, False),
                                                   (3000, 4, 7, 64, True), (3000, 4, 7, 128, False)])
def test_quantised_pages_are_those_of_the_page_writers(torch_cuda, kind, n, heads, group, dim, f32):
    """The BF16 rows of one call, written by the page writer of the other type."""
    torch = torch_cuda
    say(f"qk_norm_rope pages kind={kind} n={n} H={heads}x{group} D={dim} f32={f32}")
    r = Rope(torch, n, heads, group, dim, dim, f32, seed=n + heads)
    plain, plain_args = r.pools(P.PBE_KV_BF16)
    got, got_args = r.pools(kind)
    want, want_args = r.pools(kind)
    stream = stream_ptr(torch)
    r.call(P.PBE_KV_BF16, plain_args, stream)
    r.call(kind, got_args, stream)
    ok = np.array([r.written(t) for t in range(n)])
    slots = np.where(ok, r.slots, -1).astype(np.int32)
    d_slots = torch.from_numpy(slots).cuda()
    at = torch.from_numpy(np.where(ok, r.slots, 0).astype(np.int64)).cuda()
    size = r.blocks * B * heads * dim * 2
    rows = [b[:size].view(torch.bfloat16).view(-1, heads * dim)[at].contiguous() for b in plain[:2]]
    if kind == P.PBE_KV_MXFP4:
        P.scatter_kv_mxfp4(rows[0].data_ptr(), rows[1].data_ptr(), P.PBE_IN_BF16, n, d_slots.data_ptr(), heads, dim, *want_args, stream=stream)
    else:
        P.scatter_kv(rows[0].data_ptr(), rows[1].data_ptr(), P.PBE_IN_BF16, n, d_slots.data_ptr(), B, heads, dim, kind, *want_args, stream=stream)
    torch.cuda.synchronize()
    for i, (g, w) in enumerate(zip(got, want)):
        assert torch.equal(g, w), i


def test_no_positions_without_a_rotation(torch_cuda):
    torch = torch_cuda
    say("qk_norm_rope without positions")
    r = Rope(torch, 6, 2, 2, 64, 0, seed=2)
    bufs, args = r.pools(P.PBE_KV_BF16)
    (q, qs), (k, ks), (v, vs) = r.rows
    r.slots_dev = torch.from_numpy(r.slots).cuda()
    P.qk_norm_rope_scatter(q, qs, k, ks, v, vs, P.PBE_IN_BF16, 6, 4, 2, 64, r.w_dev[0].data_ptr(), r.w_dev[1].data_ptr(), r.eps, 0, 0, 0, 0,
                           P.PBE_ROPE_HALVES, r.slots_dev.data_ptr(), B, P.PBE_KV_BF16, r.q_out.data_ptr(), *args, stream=stream_ptr(torch))
    r.check_bf16(bufs)


def test_smallest_eps_under_squares_that_vanish(torch_cuda):
    """Squares below FP32's smallest number leave eps alone under the root: 1e-50
    against 2^-126 is far below the bound's 2^-18."""
    torch = torch_cuda
    say("qk_norm_rope with eps 2^-126")
    r = Rope(torch, 6, 2, 2, 128, 128, seed=9, eps=2.0 ** -126)
    r.bufs[0][3] *= 1e-13
    r.x = r.bufs[0].double().cpu().numpy().reshape(r.x.shape)
    bufs, args = r.pools(P.PBE_KV_BF16)
    r.call(P.PBE_KV_BF16, args, stream_ptr(torch))
    r.check_bf16(bufs)


def test_not_a_number_stays_in_its_head(torch_cuda):
    torch = torch_cuda
    say("qk_norm_rope with NaN and infinity")
    r = Rope(torch, 20, 2, 2, 64, 64, seed=5)
    buf = r.bufs[0].view(20, 8, 64)
    buf[13, 1, 3] = float("nan")
    buf[14, 4, 60] = float("inf")
    bufs, args = r.pools(P.PBE_KV_BF16)
    r.call(P.PBE_KV_BF16, args, stream_ptr(torch))
    torch.cuda.synchronize()
    q = r.q_out.float()
    assert torch.isnan(q[13, 1]).all() and torch.isfinite(q[13, [0, 2, 3]]).all() and torch.isfinite(q[14]).all()
    size = r.blocks * B * 2 * 64 * 2
    keys = bufs[0][:size].view(torch.bfloat16).view(-1, 2, 64)[int(r.slots[14])].float()
    assert torch.isnan(keys[0, [28, 60]]).all() and torch.isfinite(keys[1]).all()  # inf * 0 at its dims


def test_rope_writer_replays_from_a_graph(torch_cuda):
    torch = torch_cuda
    say("qk_norm_rope in a graph")
    r = Rope(torch, 33, 2, 6, 128, 128, seed=6)
    bufs, args = r.pools(P.PBE_KV_BF16)
    r.call(P.PBE_KV_BF16, args, stream_ptr(torch))  # makes its positions and slots on the device
    pos, slots = r.pos_dev, r.slots_dev
    (q, qs), (k, ks), (v, vs) = r.rows
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            P.qk_norm_rope_scatter(q, qs, k, ks, v, vs, P.PBE_IN_BF16, r.n, 12, 2, 128, r.w_dev[0].data_ptr(), r.w_dev[1].data_ptr(), r.eps,
                                   pos.data_ptr(), r.table_dev.data_ptr(), r.max_position, 128, P.PBE_ROPE_HALVES, slots.data_ptr(), B,
                                   P.PBE_KV_BF16, r.q_out.data_ptr(), *args, stream=side.cuda_stream)
    for rep in range(4):
        x = torch.randn(r.bufs[0].shape).to(torch.bfloat16)
        r.bufs[0].copy_(x)
        r.x = x.double().numpy().reshape(r.x.shape)
        r.positions = np.random.default_rng(rep).integers(0, 5000, r.n).astype(np.int32)
        pos.copy_(torch.from_numpy(r.positions))
        r.q_out.fill_(3.0)
        for b in bufs:
            b.fill_(CANARY)
        torch.cuda.synchronize()
        graph.replay()
        r.check_bf16(bufs)
