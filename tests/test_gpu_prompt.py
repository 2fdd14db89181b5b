"""pbe_prompt_attention and pbe_paged_prompt_attention against attention in 64 bits.

Bound of an output o = sum w v (w the softmax weights). Each weight goes into its
product rounded to BF16, off by at most 2^-8 of itself. Over rows, BF16 and MXFP4
pages the sum that divides is that of the rounded weights, so the mean moves by at
most 2^-8 / (1 - 2^-8) sum w |v - o|; over FP8 pages the weight is rounded with its
value's scale and the sum is of those before, so it moves by 2^-8 sum w |v|. An FP32
error e of a weight moves the mean by at most e sum w |v - o|, both in it and in the
sum: e is the score's error, (dim + 16) roundings of 2^-24 of sum |q k| / sqrt(dim)
(the FP8 scale's among them) and as much again for the maximum's, and 2^-20 for the
exponential, its argument's two roundings and the factors with which pieces are
joined. Sums of w v take a rounding per product of 16 keys, per change of the
maximum and per piece, below n / 16 + 600 of them, of 2^-23 each, relative to sum w
|v|. The output is rounded to BF16, 2^-8 of itself; below FP32's smallest normal
number a weight or a product may become zero, which with weights of at most 2^8 and
their sum at least 1 moves the output by at most 2^-118 (2 n max |v| + n + 1).
"""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import mxfp4 as M
from oracle import prompt as O
from tests.conftest import say
from tests.gpu_util import stream_ptr

pytestmark = pytest.mark.gpu

T = 16
KINDS = {"bf16": P.PBE_KV_BF16, "fp8": P.PBE_KV_FP8_E4M3, "mxfp4": P.PBE_KV_MXFP4}


def within(got, q, k, v, fp8=False):
    o, spread, size, reach = O.attend(q, k, v)
    n, dim = len(k), q.shape[2]
    finite = np.abs(v[np.isfinite(v)])
    e = (2 * (dim + 16) * 2.0 ** -24 * reach + 2.0 ** -20)[..., None]
    weights = 2.0 ** -8 * size if fp8 else 2.0 ** -8 / (1 - 2.0 ** -8) * spread
    bound = 2.0 ** -8 * np.abs(o) + weights + e * (spread + size * fp8) + (n / 16 + 600) * 2.0 ** -23 * size
    bound += 2.0 ** -118 * (2 * n * (finite.max() if finite.size else 0) + n + 1)
    same = np.isnan(o) & np.isnan(got) | np.isinf(o) & (o == got)
    with np.errstate(invalid="ignore"):
        ok = same | (np.abs(got - o) <= bound)
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], o[~ok][:5], bound[~ok][:5])


class Rows:
    """Prompts of `news` tokens behind `cached` ones, in rows of their own or parts
    of packed ones, with `spare` rows behind the last."""

    def __init__(self, torch, news, cached, heads, group, dim, packed=False, seed=0, spare=3, size=2.0):
        self.torch, self.news, self.heads, self.group, self.dim = torch, list(news), heads, group, dim
        self.lens = [n + c for n, c in zip(news, cached)]
        rng = np.random.default_rng(seed)
        q_heads, starts = heads * group, lambda x: np.concatenate([[0], np.cumsum(x)]).astype(np.int32)  # noqa: E731
        self.qs, self.ks = starts(self.news), starts(self.lens)
        n_q, n_k = int(self.qs[-1]) + spare, int(self.ks[-1]) + spare
        rand = lambda n, h, s: torch.tensor(rng.standard_normal((n, h * dim)) * s, dtype=torch.float32).to(torch.bfloat16)  # noqa: E731
        self.packed = packed
        if packed:
            assert n_q == n_k
            whole = torch.cat([rand(n_q, q_heads, size), rand(n_q, heads, 1), rand(n_q, heads, 1)], 1)
            self.q, self.k, self.v = whole.cuda().split([q_heads * dim, heads * dim, heads * dim], 1)
        else:
            self.q, self.k, self.v = rand(n_q, q_heads, size).cuda(), rand(n_k, heads, 1).cuda(), rand(n_k, heads, 1).cuda()
        self.out = torch.full((n_q, q_heads, dim), 5.0, dtype=torch.bfloat16, device="cuda")

    def call(self, workspace=None, out=None, stream=None, starts=None):
        torch = self.torch
        self.d_qs, self.d_ks = (torch.from_numpy(x).cuda() for x in (starts or (self.qs, self.ks)))
        if workspace is None:
            n = P.prompt_workspace_bytes(len(self.q), len(self.news), self.heads * self.group, self.heads, self.dim)
            workspace = torch.full((max(16, n),), 0xff, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        P.prompt_attention(self.q.data_ptr(), self.q.stride(0), self.k.data_ptr(), self.k.stride(0), self.v.data_ptr(), self.v.stride(0), len(self.q),
                           len(self.k), self.d_qs.data_ptr(), 0 if self.packed else self.d_ks.data_ptr(), len(self.news), self.heads * self.group,
                           self.heads, self.dim, (self.out if out is None else out).data_ptr(), workspace.data_ptr() if workspace.numel() else 0,
                           workspace.numel(), stream=stream_ptr(torch) if stream is None else stream)
        torch.cuda.synchronize()

    def check(self, skip=()):
        got = self.out.double().cpu().numpy()
        q, k, v = (x.double().cpu().numpy().reshape(len(x), -1, self.dim) for x in (self.q, self.k, self.v))
        for b in range(len(self.news)):
            if b not in skip:
                a, z, ka, kz = self.qs[b], self.qs[b + 1], self.ks[b], self.ks[b + 1]
                within(got[a:z], q[a:z], k[ka:kz], v[ka:kz])
        assert (got[self.qs[-1]:] == 5.0).all()


NEWS = [0, 1, 2, 15, 16, 17, 33, 64, 65, 130]
CACHED = [5, 0, 40, 0, 63, 1, 64, 0, 200, 3]


@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (4, 7, 128), (1, 1, 64), (3, 16, 128), (8, 4, 64), (1, 9, 128), (5, 2, 128), (1, 40, 64)])
@pytest.mark.parametrize("workspace", ["full", "none"])
def test_rows_of_odd_lengths(torch_cuda, heads, group, dim, workspace):
    torch = torch_cuda
    say(f"prompt rows H={heads}x{group} D={dim} workspace={workspace}")
    c = Rows(torch, NEWS, CACHED, heads, group, dim, seed=heads * 31 + group)
    c.call(None if workspace == "full" else torch.empty(0, dtype=torch.uint8, device="cuda"))
    c.check()


@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (1, 3, 128)])
def test_packed_rows_without_key_starts(torch_cuda, heads, group, dim):
    say(f"prompt packed rows H={heads}x{group} D={dim}")
    c = Rows(torch_cuda, [41, 1, 200, 0, 64], [0] * 5, heads, group, dim, packed=True, seed=dim, spare=0)
    c.call()
    c.check()


@pytest.mark.parametrize("new,cached", [(1, 0), (1, 4000), (4, 1500), (70, 1030), (300, 900), (513, 0)])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_sequence_is_read_in_pieces(torch_cuda, new, cached, dim):
    say(f"prompt rows {new} after {cached} D={dim}")
    c = Rows(torch_cuda, [new], [cached], 2, 3, dim, seed=new + dim)
    assert P.prompt_workspace_bytes(len(c.q), 1, 6, 2, dim) > 0
    c.call()
    c.check()


class Pages:
    """A step's new tokens over shuffled pages. Behind the sequences' last tokens, and
    in the pages that none has, lie NaN; behind a table's last block, ids that no
    pool has."""

    def __init__(self, torch, reqs, heads, group, dim, kind, seed=0, spare=3, width=2, padded=3):
        rng = np.random.default_rng(seed)
        self.torch, self.reqs, self.heads, self.group, self.dim, self.kind = torch, list(reqs), heads, group, dim, kind
        lens, news = [list(x) for x in zip(*reqs)]
        counts = [-(-n // T) for n in lens]
        self.blocks = sum(counts) + spare
        self.max_blocks = max(counts + [1]) + width
        perm = rng.permutation(self.blocks)
        self.tables = np.where(rng.random((len(reqs), self.max_blocks)) < 0.5, -5, 2 ** 31 - 1).astype(np.int32)
        self.slots, at = [], 0
        for b, (n, k) in enumerate(zip(lens, counts)):
            self.tables[b, :k] = perm[at:at + k]
            at += k
            t = np.arange(n)
            self.slots.append(self.tables[b, t // T].astype(np.int64) * T + t % T)
        live = np.zeros(self.blocks * T, bool)
        live[np.concatenate(self.slots)] = True
        self.pools, self.host = [], []
        for _ in range(2):
            x = rng.standard_normal((self.blocks * T, heads, dim)).astype(np.float32)
            if kind == "bf16":
                t = torch.from_numpy(x).to(torch.bfloat16)
                self.host.append(t.double().numpy())
                t[torch.from_numpy(~live)] = float("nan")
                self.pools.append([t.cuda(), None])
            elif kind == "fp8":
                scale = (np.abs(x).max(-1) / 448 * np.exp2(rng.integers(-3, 3, x.shape[:2]))).astype(np.float32)
                t = torch.from_numpy(np.clip(x / scale[..., None], -448, 448)).to(torch.float8_e4m3fn)
                self.host.append(t.double().numpy() * scale.astype(np.float64)[..., None])
                codes = t.view(torch.uint8)
                codes[torch.from_numpy(~live)] = 0x7f
                scale[~live] = np.inf
                self.pools.append([codes.cuda(), torch.from_numpy(scale).cuda()])
            else:
                codes, scales = M.quantise(x)
                self.host.append(M.values(codes, scales))
                scales[~live] = 255
                pool, sc = np.zeros(self.blocks * M.half_bytes(heads, dim), np.uint8), np.zeros(self.blocks * M.half_bytes(heads, dim) // 16, np.uint8)
                M.put(pool, sc, np.arange(self.blocks * T), codes, scales, len(self.pools) == 1)
                self.pools.append([torch.from_numpy(pool).cuda(), torch.from_numpy(sc).cuda()])
        self.starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        n = int(self.starts[-1]) + padded
        q = torch.tensor(rng.standard_normal((n, heads * group, dim)) * 2, dtype=torch.float32).to(torch.bfloat16)
        self.q, self.q_host = q.cuda(), q.double().numpy()
        self.lens = np.array(lens, np.int32)
        self.out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device="cuda")
        self.dev = [torch.from_numpy(x).cuda() for x in (self.starts, self.tables, self.lens)]

    def call(self, workspace=None, stream=None, out=None, q=None):
        torch = self.torch
        if workspace is None:
            n = P.prompt_workspace_bytes(len(self.q), len(self.reqs), self.heads * self.group, self.heads, self.dim)
            workspace = torch.full((max(16, n),), 0xff, dtype=torch.uint8, device="cuda")
        (k, ks), (v, vs) = self.pools
        starts, tables, lens = self.dev
        P.paged_prompt_attention(k.data_ptr(), v.data_ptr(), k.numel() * k.element_size(), ks.data_ptr() if ks is not None else 0,
                                 vs.data_ptr() if vs is not None else 0, ks.numel() * ks.element_size() if ks is not None else 0, KINDS[self.kind],
                                 self.heads, self.dim, (self.q if q is None else q).data_ptr(), (self.out if out is None else out).data_ptr(), len(self.q),
                                 starts.data_ptr(), len(self.reqs), self.heads * self.group, tables.data_ptr(), lens.data_ptr(), self.max_blocks,
                                 workspace.data_ptr() if workspace.numel() else 0, workspace.numel(), stream=stream_ptr(torch) if stream is None else stream)
        return workspace

    def check(self, skip=(), out=None):
        self.torch.cuda.synchronize()
        got = (self.out if out is None else out).double().cpu().numpy()
        for b in range(len(self.reqs)):
            if b not in skip:
                a, z, s = self.starts[b], self.starts[b + 1], self.slots[b]
                within(got[a:z], self.q_host[a:z], self.host[0][s], self.host[1][s], self.kind == "fp8")
        assert (got[self.starts[-1]:] == 5.0).all()
        return got


REQS = [(0, 0), (1, 1), (16, 16), (17, 1), (40, 40), (63, 2), (64, 64), (65, 3), (129, 1), (300, 130), (1, 0), (1040, 17)]


@pytest.mark.parametrize("heads,group,dim", [(2, 7, 64), (2, 6, 128), (4, 7, 128), (1, 1, 64), (3, 16, 128), (8, 4, 64), (1, 9, 128), (5, 2, 128)])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "mxfp4"])
def test_pages_of_odd_lengths(torch_cuda, kind, heads, group, dim):
    say(f"prompt pages {kind} H={heads}x{group} D={dim}")
    c = Pages(torch_cuda, REQS, heads, group, dim, kind, seed=heads * 31 + group)
    c.call()
    c.check()


@pytest.mark.parametrize("new,length", [(1, 4000), (5, 1500), (100, 1100), (300, 1200)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "mxfp4"])
def test_pages_of_one_sequence_in_pieces(torch_cuda, kind, dim, new, length):
    torch = torch_cuda
    say(f"prompt pages {kind} {new} of {length} D={dim}")
    c = Pages(torch, [(length, new)], 2, 3, dim, kind, seed=new + dim)
    whole = P.prompt_workspace_bytes(len(c.q), 1, 6, 2, dim)
    assert whole > 0
    for n in (whole, whole // 2 // 16 * 16, 0):
        c.out.fill_(5.0)
        c.call(torch.full((n,), 0xff, dtype=torch.uint8, device="cuda"))
        c.check()


def test_many_sequences(torch_cuda):
    torch = torch_cuda
    say("prompt: 150 sequences")
    rng = np.random.default_rng(5)
    news, cached = [int(x) for x in rng.integers(0, 12, 150)], [int(x) for x in rng.integers(0, 90, 150)]
    news[70], cached[70] = 90, 700
    c = Rows(torch, news, cached, 2, 3, 64, seed=8)
    for n in (None, torch.empty(0, dtype=torch.uint8, device="cuda")):
        c.out.fill_(5.0)
        c.call(n)
        c.check()
    p = Pages(torch, [(a + b, a) for a, b in zip(news, cached)], 1, 2, 128, "mxfp4", seed=8)
    p.call()
    p.check()


@pytest.mark.parametrize("kind", ["rows", "bf16", "fp8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("news,lens,group", [([1, 40, 3], [1, 40, 700], 3), ([300], [520], 7), ([70, 1], [600, 65], 1)])
def test_infinities_and_nans_reach_only_the_rows_that_see_them(torch_cuda, kind, dim, news, lens, group):
    """Keys and values of infinity and NaN, one a place of its own, on both sides of
    tiles' ends."""
    torch = torch_cuda
    say(f"prompt {kind} D={dim}: infinities and NaN, {news} of {lens}")
    heads = 2
    if kind == "rows":
        c = Rows(torch, news, [a - b for a, b in zip(lens, news)], heads, group, dim, seed=dim)
        at, k, v = c.ks, c.k.view(-1, heads, dim), c.v.view(-1, heads, dim)
    else:
        c = Pages(torch, list(zip(lens, news)), heads, group, dim, kind, seed=dim)
        k, v = (x[0].view(-1, heads, dim) for x in c.pools)
    inf, nan = float("inf"), float("nan")
    for b, n in enumerate(lens):
        for j, (what, value) in enumerate([("v", inf), ("v", -inf), ("v", nan), ("k", -inf), ("k", nan), ("v", inf), ("v", -inf)]):
            # places a row or two from the end, the last two on one dim; keys of one head
            t = n - 1 - (3 * j + 1) % max(1, min(n, 60))
            if t < 0 or (n == 1 and j):
                continue
            if kind == "fp8" and value != nan:
                continue                            # E4M3 has no infinities
            slot = int(at[b]) + t if kind == "rows" else int(c.slots[b][t])
            d, h = (5 if j >= 5 else (11 * j) % dim), (1 if what == "v" else 0)
            store = 0x7f if kind == "fp8" else value
            (v if what == "v" else k)[slot, h, d] = store
            if kind != "rows":
                c.host[1 if what == "v" else 0][slot, h, d] = value
    c.call()
    c.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1.0, 64.0, 2.0 ** 40, 2.0 ** 100])
def test_equal_scores_of_any_size_weigh_alike(torch_cuda, dim, size):
    """Keys that are all the same: whatever the scores, outputs are means, off by
    their own rounding and that of sums of n / 16 + 600 products."""
    torch = torch_cuda
    say(f"prompt: equal scores of size {size}")
    c = Rows(torch, [5, 300], [700, 0], 1, 2, dim, seed=dim, size=size)
    c.k[:] = c.k[:1].clone()
    c.call()
    v = c.v.double().cpu().numpy()
    got = c.out.double().cpu().numpy()
    for b in range(2):
        n, m = c.news[b], c.lens[b]
        for i in range(n):
            seen = v[c.ks[b]:c.ks[b] + m - n + i + 1]
            bound = 2.0 ** -8 * np.abs(seen.mean(0)) + (m / 16 + 600) * 2.0 ** -23 * np.abs(seen).mean(0)
            assert (np.abs(got[c.qs[b] + i] - seen.mean(0)) <= bound).all()


def test_constant_values_come_back_as_they_are(torch_cuda):
    say("prompt: constant values")
    for kind in ("bf16", "mxfp4"):
        c = Pages(torch_cuda, [(900, 200), (33, 33)], 2, 4, 128, kind, seed=3)
        pool = c.pools[1]
        if kind == "bf16":
            pool[0].fill_(1.5)
        else:
            pool[0].fill_(0x33)      # codes of 1.5
            pool[1].fill_(127)
        c.call()
        c.torch.cuda.synchronize()
        assert (c.out[: c.starts[-1]] == 1.5).all()


def test_rows_and_sequences_that_make_no_sense(torch_cuda):
    torch = torch_cuda
    say("prompt: bad starts, lengths and ids")
    # starts: rows before 0, behind the last, in the wrong order; keys beyond theirs
    c = Rows(torch, [20, 30, 10, 25], [0, 40, 5, 6], 2, 2, 64, seed=1)
    n_q, n_k = len(c.q), len(c.k)
    for qs, ks, nan, good in (([-4, 20, 50, 60, 85], c.ks, (0, 20), (1, 2, 3)), ([0, 20, 50, 60, n_q + 1], c.ks, (60, n_q), (0, 1, 2)),
                              (c.qs, [0, 20, 90, 105, n_k + 1], (60, 85), (0, 1, 2)), (c.qs, [0, 20, 90, 80, 111], (50, 60), (0, 1))):
        c.out.fill_(5.0)
        c.call(starts=(np.array(qs, np.int32), np.array(ks, np.int32)))
        got = c.out.double().cpu().numpy()
        assert np.isnan(got[nan[0]:nan[1]]).all()
        q, k, v = (x.double().cpu().numpy().reshape(len(x), -1, 64) for x in (c.q, c.k, c.v))
        for b in good:
            within(got[qs[b]:qs[b + 1]], q[qs[b]:qs[b + 1]], k[ks[b]:ks[b + 1]], v[ks[b]:ks[b + 1]])
    c.out.fill_(5.0)
    c.call(starts=(np.array([0, 20, 10, 60, 85], np.int32), c.ks))   # the second ends before it begins: it has no rows
    assert not (c.out[60:85] == 5.0).any() and (c.out[85:] == 5.0).all()
    # a length of more queries than keys: the first see nothing
    c = Rows(torch, [20], [0], 1, 3, 64, seed=2, spare=0)
    c.lens, c.ks = [8], np.array([0, 8], np.int32)
    c.call()
    got = c.out.double().cpu().numpy()
    assert (got[:12] == 0).all()
    q, k, v = (x.double().cpu().numpy().reshape(20, -1, 64) for x in (c.q, c.k, c.v))
    within(got[12:], q[12:], k[:8], v[:8])
    for kind in ("bf16", "fp8", "mxfp4"):
        reqs = [(100, 40), (50, 50), (70, 3), (1500, 20), (33, 2)]
        p = Pages(torch, reqs, 2, 3, 128, kind, seed=5)
        lens, tables = p.lens.copy(), p.tables.copy()
        lens[0], lens[4] = -1, (p.max_blocks + 1) * T
        tables[1, 2], tables[3, 70] = p.blocks, -1      # keys 32..47 and 1120..1135
        p.dev[1:] = [torch.from_numpy(tables).cuda(), torch.from_numpy(lens).cuda()]
        p.call()
        got = p.check(skip=(0, 1, 3, 4))
        s = p.starts
        assert np.isnan(got[s[0]:s[1]]).all() and np.isnan(got[s[4]:s[5]]).all() and np.isnan(got[s[3]:s[4]]).all()
        assert np.isnan(got[s[1] + 32:s[2]]).all()
        slots = p.slots[1]
        within(got[s[1]:s[1] + 32], p.q_host[s[1]:s[1] + 32], p.host[0][slots[:32]], p.host[1][slots[:32]], kind == "fp8")


@pytest.mark.parametrize("kind", ["bf16", "fp8", "mxfp4"])
def test_captured_calls_follow_what_changes_between_replays(torch_cuda, kind):
    """Two graphs that share a workspace, replayed in turn on a stream of their own
    while lengths and queries change, against eager calls."""
    torch = torch_cuda
    say(f"prompt {kind}: captured")
    cases = [Pages(torch, [(1500, 30), (200, 64), (17, 1)], 2, 3, 128, kind, seed=s) for s in (1, 2)]
    need = max(P.prompt_workspace_bytes(len(c.q), 3, 6, 2, 128) for c in cases)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    side, graphs = torch.cuda.Stream(), []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                c.call(ws, stream=side.cuda_stream)
        graphs.append(g)
    for rep in range(4):
        for c, g in zip(cases, graphs):
            lens = torch.tensor([1500 - 64 * rep, 200 - rep, 17], dtype=torch.int32, device="cuda")
            c.dev[2].copy_(lens)
            c.q.copy_(c.q.roll(1, 0))
            want = torch.full_like(c.out, 5.0)
            c.call(out=want)
            c.out.fill_(5.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                g.replay()
            torch.cuda.synchronize()
            assert torch.equal(c.out.view(torch.int16), want.view(torch.int16)), rep


def test_calls_beside_each_other_and_in_place(torch_cuda):
    torch = torch_cuda
    say("prompt: two streams, outputs over queries")
    cases = [Pages(torch, [(2500, 200), (300, 7)], 2, 6, 128, k, seed=i) for i, k in enumerate(("bf16", "fp8", "mxfp4", "bf16"))]
    for c in cases:
        c.call()
    torch.cuda.synchronize()
    want = [c.out.clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    kept = []
    for c in cases:
        c.out.fill_(5.0)
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                kept.append(c.call(stream=s.cuda_stream))
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.out.view(torch.int16), w.view(torch.int16))
        n = int(c.starts[-1])
        q = c.q.clone()
        c.call(out=q, q=q)
        torch.cuda.synchronize()
        assert torch.equal(q[:n].view(torch.int16), w[:n].view(torch.int16)) and torch.equal(q[n:], c.q[n:])
    r = Rows(torch, [300, 20], [50, 900], 2, 3, 64, seed=4)
    r.call()
    w = r.out.clone()
    q = r.q
    r.call(out=q.view(len(q), 6, 64))
    assert torch.equal(q.view(len(q), 6, 64)[:320].view(torch.int16), w[:320].view(torch.int16))


def test_pages_beyond_four_gigabytes(torch_cuda):
    torch = torch_cuda
    say("prompt: pools of 5 GiB")
    heads, dim, group = 2, 128, 3
    half = T * heads * dim * 2
    blocks = 5 * 2 ** 30 // half
    c = Pages(torch, [(150, 40), (70, 2)], heads, group, dim, "bf16", seed=6, spare=0)
    big = [torch.zeros((blocks * T, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    far = blocks - c.blocks
    for x, (small, _) in zip(big, c.pools):
        x[far * T:] = small
    tables = c.tables.copy()
    for b, (n, _) in enumerate(c.reqs):
        tables[b, : -(-n // T)] += far
    c.dev[1] = torch.from_numpy(tables).cuda()
    c.pools = [[x, None] for x in big]
    c.blocks = blocks
    c.call()
    c.check()


def test_long_sequences_and_each_tile_size(torch_cuda):
    """Rows per sequence of 32, 64, 128, 256 and more, a query head or two each, over a
    few thousand keys; the last rows against the oracle."""
    torch = torch_cuda
    for kind, dim in (("bf16", 128), ("fp8", 128), ("fp8", 64), ("mxfp4", 64), ("mxfp4", 128), ("bf16", 64)):
        for new in (20, 33, 100, 200, 700):
            say(f"prompt pages {kind} D={dim}: {new} rows over 3000 keys")
            c = Pages(torch, [(3001, new), (2999, new)], 1, 1, dim, kind, seed=new)
            c.call()
            c.check()


def test_no_keys_at_all_give_zeros(torch_cuda):
    torch = torch_cuda
    say("prompt: no keys")
    q = torch.randn((70, 128), device="cuda").to(torch.bfloat16)
    out = torch.full((70, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([0, 1, 65], dtype=torch.int32, device="cuda")
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    P.prompt_attention(q.data_ptr(), 128, 0, 64, 0, 64, 70, 0, starts.data_ptr(), none.data_ptr(), 2, 2, 1, 64, out.data_ptr(), 0, 0,
                       stream=stream_ptr(torch))
    torch.cuda.synchronize()
    assert (out[:65] == 0).all() and (out[65:] == 5.0).all()


def test_values_up_to_the_sums_range(torch_cuda):
    """Values of 2^100 and queries whose scores climb from key to key, so that the
    maximum moves all the time."""
    torch = torch_cuda
    say("prompt: large values, climbing scores")
    for kind in ("bf16", "fp8"):
        c = Pages(torch, [(700, 90), (64, 64)], 1, 2, 64, kind, seed=12)
        slots = np.concatenate(c.slots)
        climb = np.concatenate([np.arange(n) / 64.0 for n, _ in c.reqs])
        c.q.fill_(1.0)
        c.q_host[:] = 1.0
        at = torch.from_numpy(slots).cuda()
        if kind == "bf16":
            k = torch.from_numpy(climb).to(torch.bfloat16)
            c.pools[0][0][at] = k.cuda()[:, None, None]
            c.host[0][slots] = k.double().numpy()[:, None, None]
            big = (c.pools[1][0][at].float() * 2.0 ** 100).to(torch.bfloat16)
            c.pools[1][0][at] = big
            c.host[1][slots] = big.double().cpu().numpy()
        else:
            scale = torch.from_numpy(climb).float()
            c.pools[0][0][at] = 0x38                                   # 1.0
            c.pools[0][1].view(-1, 1)[at] = scale.cuda()[:, None]
            c.host[0][slots] = scale.double().numpy()[:, None, None]
            c.pools[1][1].view(-1, 1)[at] *= 2.0 ** 100
            c.host[1][slots] *= 2.0 ** 100
        c.call()
        c.check()
