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
