"""The MXFP4 page writer and the gather (pbe_scatter_kv_mxfp4,
pbe_gather_kv_mxfp4) against the oracle, bit for bit: whole pools and scale
pools, bytes that nothing writes being canaries, and whole rows read back."""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import mxfp4 as M
from oracle import oracle as O
from tests.conftest import say
from tests.gpu_util import first_diff, stream_ptr

pytestmark = pytest.mark.gpu

T = 16


def bf16_f64(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rows(rng, n, heads, dim, f32, special=True):
    """Rows [2][n][heads][dim] in the input's type and as doubles."""
    x = rng.standard_normal((2, n, heads, dim)).astype(np.float32) * 1.5
    if special and n > 8:
        x[0, 1] = 0.0
        x[1, 2, :, 32:64] = 0.0                            # one all-zero group
        x[0, 3, 0, 5] = np.nan
        x[1, 4, 0, dim - 1] = -np.inf
        x[0, 5] = 1e-38 * rng.standard_normal((heads, dim))  # scales at their smallest
        x[1, 5] = 1e-40                                    # subnormal
        x[1, 6] *= 2e38 / np.abs(x[1, 6]).max()
        x[0, 7] = np.resize([0.25, -0.75, 1.25, 1.75, -2.5, 3.5, 5.0, 7.5], (heads, dim)) * 2.0 ** -9  # ties
        x[1, 8] = -0.0
    if f32:
        return x, x.astype(np.float64)
    bits = O.bf16_from_f32(x.reshape(2, -1)).reshape(x.shape)
    return bits, bf16_f64(bits)


class Pools:
    """Layer `layer` of a page-major arena and its scale arena, filled with canaries."""

    def __init__(self, torch, heads, dim, pages, layers=1, layer=0, seed=0):
        rng = np.random.default_rng(seed)
        self.torch, self.heads, self.dim = torch, heads, dim
        self.half = M.half_bytes(heads, dim)
        self.stride = 2 * layers if layers > 1 else 1
        planes = 2 * layers * pages
        self.host = [rng.integers(0, 256, planes * self.half).astype(np.uint8),
                     rng.integers(100, 140, planes * self.half // 16).astype(np.uint8)]
        self.dev = [torch.from_numpy(h.copy()).cuda() for h in self.host]
        # local pools: K in the first half of the buffer; an arena: planes side by side
        self.k_at = 2 * layer if layers > 1 else 0
        self.v_at = self.k_at + 1 if layers > 1 else pages
        self.blocks = planes - self.k_at - 1 if layers > 1 else pages
        self.per = [self.half, self.half // 16]

    def host_views(self, host=None):
        """K, V, K scales and V scales from their first block on."""
        a, s = host or self.host
        return (a[self.k_at * self.per[0]:], a[self.v_at * self.per[0]:], s[self.k_at * self.per[1]:], s[self.v_at * self.per[1]:])

    def args(self):
        a, s = self.dev
        out = []
        for buf, per in ((a, self.per[0]), (s, self.per[1])):
            for at in (self.k_at, self.v_at):
                out += [buf.data_ptr() + at * per, self.blocks * per]
        return out

    def snapshot(self):
        self.torch.cuda.synchronize()
        return [d.cpu().numpy() for d in self.dev]


def put(views, slots, x, heads, dim, got_views):
    """Oracle's pools after the write. The codes of a group with an infinity or a
    NaN are whatever was stored there: its scale says NaN."""
    live = np.flatnonzero(slots >= 0)
    for i, is_value in enumerate((False, True)):
        codes, sc = M.quantise(x[i][live])
        M.put(views[i], views[2 + i], slots[live], codes, sc, is_value)
        nan = np.repeat(sc == 255, 32, -1)
        at = M.code_at(slots[live], heads, dim, is_value)[nan]
        views[i][at] = got_views[i][at]


def to_dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.uint8)).cuda()


@pytest.mark.parametrize("n", [1, 15, 16, 33, 301])
@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,dim", [(2, 64), (2, 128), (4, 128), (1, 64), (3, 128), (5, 64)])
def test_written_pages_match_the_oracle(torch_cuda, heads, dim, f32, n):
    torch = torch_cuda
    say(f"scatter_kv_mxfp4 H={heads} D={dim} f32={f32} n={n}")
    rng = np.random.default_rng(heads * 1000 + dim + n)
    pools = Pools(torch, heads, dim, pages=n // T + 6, layers=3, layer=1, seed=n)
    ids = rng.permutation(n // T + 6)[: n // T + 2] * 6
    slots = np.concatenate([i * T + np.arange(T) for i in ids])[3: 3 + n].astype(np.int32)  # starts inside a page
    if n > 16:
        slots = slots[rng.permutation(n)]
        slots[9], slots[10], slots[11] = -1, -2 ** 31, pools.blocks * T  # padding; a block beyond the pools
        slots[12] = 2 ** 31 - 1
    raw, x = rows(rng, n, heads, dim, f32)
    dk, dv, ds = to_dev(torch, raw[0]), to_dev(torch, raw[1]), torch.from_numpy(slots).cuda()
    P.scatter_kv_mxfp4(dk.data_ptr(), dv.data_ptr(), P.PBE_IN_F32 if f32 else P.PBE_IN_BF16, n, ds.data_ptr(), heads, dim,
                       *pools.args(), stream=stream_ptr(torch))
    got = pools.snapshot()
    want = [h.copy() for h in pools.host]
    inside = np.where(slots.astype(np.int64) // T < pools.blocks, slots, -1)
    put(pools.host_views(want), inside, x, heads, dim, pools.host_views(got))
    for g, w, what in zip(got, want, ("codes", "scales")):
        assert np.array_equal(g, w), (what, first_diff(g, w))


@pytest.mark.parametrize("n", [1, 16, 37, 300])
@pytest.mark.parametrize("heads,dim", [(2, 64), (2, 128), (4, 128), (1, 128), (3, 64)])
def test_gathered_rows_match_the_oracle(torch_cuda, heads, dim, n):
    torch = torch_cuda
    say(f"gather_kv_mxfp4 H={heads} D={dim} n={n}")
    rng = np.random.default_rng(heads * 100 + dim + n)
    pools = Pools(torch, heads, dim, pages=9, seed=n)
    views = pools.host_views()
    # every scale byte among them, 255 (NaN) and 0 (2^-127) too
    for i in (2, 3):
        at = rng.choice(9 * pools.per[1], 256, replace=False)
        views[i][at] = np.arange(256)
    pools.dev = [torch.from_numpy(h.copy()).cuda() for h in pools.host]
    slots = rng.integers(0, 9 * T, n).astype(np.int32)  # a slot may come twice
    if n > 16:
        slots[4], slots[5], slots[6], slots[7] = -1, -2 ** 31, 9 * T, 2 ** 31 - 1
    out = torch.full((2, n + 1, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ds = torch.from_numpy(slots).cuda()
    P.gather_kv_mxfp4(*pools.args(), ds.data_ptr(), n, heads, dim, out[0].data_ptr(), out[1].data_ptr(), stream=stream_ptr(torch))
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    want = np.full(got.shape, 7.0)
    beyond = slots.astype(np.int64) >= 9 * T
    ok = (slots >= 0) & ~beyond
    for i in range(2):
        want[i, :n][ok] = M.get(views[i], views[2 + i], slots[ok], heads, dim, bool(i))
        want[i, :n][beyond] = np.nan
    # codes of 4 and 6 under scales 253 and 254, which the writer never stores,
    # are 2^128 and more: beyond BF16 (its largest is below 2^128), so infinite
    want = np.where(np.abs(want) >= 2.0 ** 128, np.copysign(np.inf, want), want)
    np.testing.assert_array_equal(got, want)


def test_pools_written_read_back_and_handed_over(torch_cuda):
    """Rows written in one part of an arena, its pages handed over as one-byte
    elements, and the rows read from where they went."""
    torch = torch_cuda
    heads, dim, layers, layer, pages, n = 2, 128, 2, 1, 24, 100
    say("mxfp4 pages through the handoff")
    rng = np.random.default_rng(7)
    pools = Pools(torch, heads, dim, pages, layers=layers, layer=layer)
    order = rng.permutation(pages)
    src, dst = order[:7] * 2 * layers, order[7:14] * 2 * layers
    slots = [np.concatenate([i * T + np.arange(T) for i in ids])[:n].astype(np.int32) for ids in (src, dst)]
    raw, x = rows(rng, n, heads, dim, False, special=False)
    dk, dv = to_dev(torch, raw[0]), to_dev(torch, raw[1])
    d_slots = [torch.from_numpy(s).cuda() for s in slots]
    stream = stream_ptr(torch)
    P.scatter_kv_mxfp4(dk.data_ptr(), dv.data_ptr(), P.PBE_IN_BF16, n, d_slots[0].data_ptr(), heads, dim, *pools.args(), stream=stream)
    for buf, d in zip(pools.dev, (dim // 2, dim // 32)):
        kv = P.shape(layers, heads, d)
        view = P.view_of(buf.data_ptr(), buf.numel())
        with P.RunList.bf16(view, view, P.build_runs(src, dst, kv, 1), kv, elem_bytes=1) as run:
            run.copy(stream)
            torch.cuda.synchronize()
    out = torch.empty((2, n, heads, dim), dtype=torch.bfloat16, device="cuda")
    P.gather_kv_mxfp4(*pools.args(), d_slots[1].data_ptr(), n, heads, dim, out[0].data_ptr(), out[1].data_ptr(), stream=stream)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out.double().cpu().numpy(), M.values(*M.quantise(x)))


def test_writer_and_gather_replay_from_a_graph(torch_cuda):
    torch = torch_cuda
    heads, dim, n = 4, 128, 77
    say("mxfp4 writer and gather in a graph")
    rng = np.random.default_rng(9)
    pools = Pools(torch, heads, dim, pages=8)
    slots = rng.permutation(8 * T)[:n].astype(np.int32)
    ds = torch.from_numpy(slots).cuda()
    x = torch.zeros((2, n, heads, dim), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(x)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            P.scatter_kv_mxfp4(x[0].data_ptr(), x[1].data_ptr(), P.PBE_IN_BF16, n, ds.data_ptr(), heads, dim, *pools.args(),
                               stream=side.cuda_stream)
            P.gather_kv_mxfp4(*pools.args(), ds.data_ptr(), n, heads, dim, out[0].data_ptr(), out[1].data_ptr(), stream=side.cuda_stream)
    for rep in range(4):
        raw, want = rows(rng, n, heads, dim, False, special=False)
        x.copy_(torch.from_numpy(raw.view(np.int16)).cuda().view(torch.bfloat16))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(out.double().cpu().numpy(), M.values(*M.quantise(want)), err_msg=str(rep))


def test_pool_offsets_beyond_32_bits(torch_cuda):
    """Blocks past 4 GiB of codes: the first and the last of a large pool."""
    torch = torch_cuda
    heads, dim, n = 8, 128, 20
    half = M.half_bytes(heads, dim)
    blocks = (5 << 30) // half
    say("mxfp4 pools of 5 GiB")
    pools = [torch.zeros(blocks * per, dtype=torch.uint8, device="cuda") for per in (half, half, half // 16, half // 16)]
    args = [v for p in pools for v in (p.data_ptr(), p.numel())]
    slots = np.array([0, 5, (blocks - 1) * T + 15] + [blocks * T // 2 + i for i in range(n - 3)], np.int32)
    rng = np.random.default_rng(3)
    raw, x = rows(rng, n, heads, dim, False, special=False)
    dk, dv, ds = to_dev(torch, raw[0]), to_dev(torch, raw[1]), torch.from_numpy(slots).cuda()
    P.scatter_kv_mxfp4(dk.data_ptr(), dv.data_ptr(), P.PBE_IN_BF16, n, ds.data_ptr(), heads, dim, *args, stream=stream_ptr(torch))
    out = torch.empty((2, n, heads, dim), dtype=torch.bfloat16, device="cuda")
    P.gather_kv_mxfp4(*args, ds.data_ptr(), n, heads, dim, out[0].data_ptr(), out[1].data_ptr(), stream=stream_ptr(torch))
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out.double().cpu().numpy(), M.values(*M.quantise(x)))
    last = pools[0][(blocks - 1) * half:].cpu().numpy()
    want, sc = np.zeros(half, np.uint8), np.zeros(half // 16, np.uint8)
    M.put(want, sc, [15], *M.quantise(x[0][2:3]), False)
    assert np.array_equal(last, want), first_diff(last, want)


def test_misuse_is_refused_before_any_write(torch_cuda):
    torch = torch_cuda
    heads, dim = 2, 64
    pools = Pools(torch, heads, dim, pages=4)
    x = torch.zeros((4, heads * dim), dtype=torch.bfloat16, device="cuda")
    s = torch.zeros(4, dtype=torch.int32, device="cuda")
    say("mxfp4 misuse")
    host = np.zeros(1 << 16, np.uint8)
    a = pools.args()
    for i, (to, code) in enumerate([(a[:1] + [a[1] + (1 << 32)] + a[2:], P.PBE_ERR_INVALID),  # larger than its allocation
                                    ([a[0] + 2] + a[1:], P.PBE_ERR_INVALID), ([host.ctypes.data] + a[1:], P.PBE_ERR_INVALID)]):
        with pytest.raises(P.PbeError) as e:
            P.scatter_kv_mxfp4(x.data_ptr(), x.data_ptr(), P.PBE_IN_BF16, 4, s.data_ptr(), heads, dim, *to, stream=stream_ptr(torch))
        assert e.value.code == code, i
        with pytest.raises(P.PbeError) as e:
            P.gather_kv_mxfp4(*to, s.data_ptr(), 4, heads, dim, x.data_ptr(), x.data_ptr(), stream=stream_ptr(torch))
        assert e.value.code == code, i
    got = pools.snapshot()
    assert all(np.array_equal(g, h) for g, h in zip(got, pools.host))
