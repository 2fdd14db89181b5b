"""Calls of pbe_prompt_attention and pbe_paged_prompt_attention at the ends of what
they take, over values for which every output is known, or within the bound of
test_gpu_prompt.py."""
import numpy as np
import pytest

import pbe_handoff as P
from oracle import prompt as O
from tests.conftest import say
from tests.gpu_util import stream_ptr
from tests.test_gpu_prompt import Pages, Rows, within

pytestmark = pytest.mark.gpu

T = 16


def test_whole_tiles_of_very_long_sequences(torch_cuda):
    """Sequences of 2^24 tokens and more, in tables that name one block again and again,
    without a workspace. All keys are zeros and all values 1.5. Sums of 1 and of 1.5 are
    exact but for the last tile's (below 2^25, so off by at most 1 of 2^24, far below half
    a BF16 step), so the outputs are 1.5."""
    torch = torch_cuda
    say("prompt: 2 of 24 sequences, of 16,777,287 and 16,777,344 tokens, 256 heads")
    news, lens, heads, dim = [0] * 10 + [1] + [0] * 5 + [5] + [0] * 7, [0] * 24, 256, 64
    lens[10], lens[16] = 16777287, 16777344
    blocks = -(-max(lens) // T)
    k, v = (torch.full((T, dim), x, dtype=torch.bfloat16, device="cuda") for x in (0.0, 1.5))
    q = torch.randn((8, heads, dim), device="cuda").to(torch.bfloat16)
    out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device="cuda")
    tables, d_lens = torch.zeros((24, blocks), dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    P.paged_prompt_attention(k.data_ptr(), v.data_ptr(), T * dim * 2, 0, 0, 0, P.PBE_KV_BF16, 1, dim, q.data_ptr(), out.data_ptr(), 8,
                             starts.data_ptr(), 24, heads, tables.data_ptr(), d_lens.data_ptr(), blocks, 0, 0, stream=stream_ptr(torch))
    torch.cuda.synchronize()
    assert (out[:6] == 1.5).all() and (out[6:] == 5.0).all()


@pytest.mark.parametrize("workspace", ["full", "none"])
@pytest.mark.parametrize("times", [4, 32, 40])
@pytest.mark.parametrize("kind", ["rows", "mxfp4"])
def test_rows_claimed_many_times_and_rows_behind_them(torch_cuda, kind, times, workspace):
    """Starts that go back: `times` sequences claim the first 900 rows, each with the same
    keys, and one behind them all the last 100, so every row has one result. Over pages
    all values are 1.5."""
    torch = torch_cuda
    say(f"prompt {kind}: rows claimed {times} times, workspace={workspace}")
    n, dim, batch = 1000, 64, 2 * times
    starts = [0, 900] * times + [n]
    d_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(times)
    rand = lambda s: torch.tensor(rng.standard_normal((n, dim)) * s, dtype=torch.float32).to(torch.bfloat16).cuda()  # noqa: E731
    q, k, v = rand(2), rand(1), rand(1)
    out = torch.full((n + 2, 1, dim), 5.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((P.prompt_workspace_bytes(n, batch, 1, 1, dim) if workspace == "full" else 0,), 0xff, dtype=torch.uint8, device="cuda")
    at = (ws.data_ptr() if ws.numel() else 0, ws.numel())
    if kind == "rows":
        P.prompt_attention(q.data_ptr(), dim, k.data_ptr(), dim, v.data_ptr(), dim, n, n, d_starts.data_ptr(), 0, batch, 1, 1, dim, out.data_ptr(),
                           *at, stream=stream_ptr(torch))
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        q, k, v = (x.double().cpu().numpy()[:, None] for x in (q, k, v))
        for a, z in ((0, 900), (900, n)):
            within(got[a:z], q[a:z], k[a:z], v[a:z])
    else:
        half = T * dim // 2
        pools = [torch.randint(0, 256, (half,), dtype=torch.uint8, device="cuda"), torch.full((half,), 0x33, dtype=torch.uint8, device="cuda")]
        scales = [torch.full((half // 16,), 127, dtype=torch.uint8, device="cuda") for _ in range(2)]
        lens = torch.tensor([1000 if z > a else 7 for a, z in zip(starts, starts[1:])], dtype=torch.int32, device="cuda")
        tables = torch.zeros((batch, 63), dtype=torch.int32, device="cuda")
        P.paged_prompt_attention(pools[0].data_ptr(), pools[1].data_ptr(), half, scales[0].data_ptr(), scales[1].data_ptr(), half // 16, P.PBE_KV_MXFP4, 1,
                                 dim, q.data_ptr(), out.data_ptr(), n, d_starts.data_ptr(), batch, 1, tables.data_ptr(), lens.data_ptr(), 63, *at,
                                 stream=stream_ptr(torch))
        torch.cuda.synchronize()
        assert (out[:n] == 1.5).all()
    assert (out[n:] == 5.0).all()


def none(torch):
    return torch.empty(0, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("heads,group", [(2, 7), (4, 6), (8, 1), (2, 8), (3, 5)])
@pytest.mark.parametrize("lens", [(500, 530), (1, 90), (0, 1500)])
@pytest.mark.parametrize("batch", [64, 70])
def test_drafted_tokens_of_many_requests_over_fp8_pages(torch_cuda, batch, lens, heads, group):
    """Heads of 128 dims, 4 * batch * heads above any GPU's compute units and at most 32
    rows a sequence: tiles of 32 rows, whole and in parts."""
    torch = torch_cuda
    say(f"prompt pages fp8 D=128 H={heads}x{group}: {batch} x 4 tokens, {lens[0]} to {lens[1]} keys")
    rng = np.random.default_rng(batch + heads + lens[1])
    reqs = [(int(rng.integers(lens[0], lens[1] + 1)), min(4, int(rng.integers(1, 9)))) for _ in range(batch)]
    reqs = [(max(n, 4 - i % 3), m) for i, (n, m) in enumerate(reqs)]
    c = Pages(torch, reqs, heads, group, 128, "fp8", seed=batch)
    assert len(c.q) * group <= 32 * batch and 4 * batch * heads >= 2 * torch.cuda.get_device_properties(0).multi_processor_count
    for ws in (None, none(torch)):
        c.out.fill_(5.0)
        c.call(ws)
        c.check()


def near(got, q, k, v, fp8):
    """within(), for keys and values that hold infinities and NaN: how far a score may be
    off goes by its finite products (a key with others has a weight of zero or takes its
    rows to NaN), and what has a NaN or an infinity to show, shows it. Returns how many."""
    finite_k, finite_v = (np.where(np.isfinite(x), x, 0.0) for x in (k, v))
    with np.errstate(invalid="ignore"):
        o, spread, size, _ = O.attend(q, k, v)
        _, _, _, reach = O.attend(q, finite_k, finite_v)
        shown = ~np.isfinite(o)
        assert ((np.isnan(o) & np.isnan(got)) | (np.isinf(o) & (o == got)))[shown].all()
        n, dim = len(k), q.shape[2]
        e = (2 * (dim + 16) * 2.0 ** -24 * reach + 2.0 ** -20)[..., None]
        bound = 2.0 ** -8 * np.abs(o) + (2.0 ** -8 * size if fp8 else 2.0 ** -8 / (1 - 2.0 ** -8) * spread) + e * (spread + size * fp8)
        bound += (n / 16 + 600) * 2.0 ** -23 * size + 2.0 ** -118 * (2 * n * np.abs(finite_v).max() + n + 1)
        assert np.isfinite(bound[~shown]).all() and (np.abs(got - o) <= bound)[~shown].all()
    return int(shown.sum())


def without(got, q, k, v, token, score):
    """Rows of one KV head (fp8) to whose scores with `token`, infinities of the sign of
    score [new][group], a key's scale led: +infinity takes them to NaN, -infinity as if
    the key were not there (if there are others)."""
    n, new = len(k), len(q)
    sees = np.arange(new)[:, None] + n - new >= np.full(score.shape, token)
    assert np.isnan(got[sees & (score > 0)]).all()
    for i, h in np.argwhere(~(sees & (score > 0))):
        keep = np.arange(n - new + i + 1)
        keep = keep[keep != token] if sees[i, h] else keep
        if len(keep):
            within(got[i, h][None, None], q[i, h][None, None], k[keep], v[keep], True)
    return int(sees.sum())


class Special:
    """Three sequences of two heads, of which the second is given numbers that are none,
    a token at a time; the first head and the other sequences must not notice."""

    REQS, GROUP = [(1200, 70), (65, 65), (130, 3)], 3

    def __init__(self, torch, kind, dim, workspace):
        self.torch, self.kind, self.dim = torch, kind, dim
        lens, news = zip(*self.REQS)
        if kind == "rows":
            c = Rows(torch, news, [n - m for n, m in self.REQS], 2, self.GROUP, dim, seed=dim)
            self.starts, self.pools = c.qs, [x.view(-1, 2, dim) for x in (c.k, c.v)]
            self.slots = [np.arange(c.ks[b], c.ks[b + 1]) for b in range(3)]
            self.host = [x.double().cpu().numpy() for x in self.pools]
            self.q = c.q.double().cpu().numpy().reshape(len(c.q), -1, dim)
        else:
            c = Pages(torch, self.REQS, 2, self.GROUP, dim, kind, seed=dim)
            self.starts, self.slots, self.host, self.q = c.starts, c.slots, c.host, c.q_host
            self.pools = [x[0].view(-1, 2, dim) if kind != "mxfp4" else None for x in c.pools]
        self.case, self.workspace = c, workspace
        self.want = self.run().copy()

    def run(self):
        self.case.out.fill_(5.0)
        self.case.call(self.workspace)
        self.torch.cuda.synchronize()
        return self.case.out.double().cpu().numpy()

    def scale(self, which, slot):
        """The scale of a token of the second head: FP32, or bytes of the groups."""
        x = self.case.pools[which][1]
        return x.view(-1, 2)[slot, 1:] if self.kind == "fp8" else x.view(self.case.blocks, 2, self.dim // 32, T)[slot // T, 1, :, slot % T]

    def check(self, b, look):
        got, a, z = self.run(), self.starts[b], self.starts[b + 1]
        others = np.ones(got.shape[:2], bool)
        others[a:z, self.GROUP:] = False
        assert (got[others] == self.want[others]).all()
        return look(got[a:z, self.GROUP:], self.q[a:z, self.GROUP:], *(x[self.slots[b]][:, 1:] for x in self.host))

    def tokens(self):
        """Tokens on both sides of tiles' ends, cached ones and new ones."""
        for b, (n, new) in enumerate(self.REQS):
            for t in sorted({0, 1, 63, 64, 65, 127, n // 2, n - new - 1, n - new, n - new + 1, n - new // 2, n - 2, n - 1}):
                if 0 <= t < n:
                    yield b, t, int(self.slots[b][t])


@pytest.mark.parametrize("workspace", ["full", "none"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind,what", [(k, w) for k in ("rows", "bf16") for w in ("key -inf", "key nan", "value inf", "value -inf", "value nan")] +
                         [(k, w) for k in ("fp8", "mxfp4") for w in ("key nan", "value nan")])
def test_one_special_number_at_a_time(torch_cuda, kind, what, dim, workspace):
    """BF16 numbers as they are; E4M3's NaN; MXFP4 scales of NaN (groups of 32 dims)."""
    torch = torch_cuda
    say(f"prompt {kind} D={dim}: {what}, workspace={workspace}")
    s = Special(torch, kind, dim, none(torch) if workspace == "none" else None)
    which, value, seen = int(what.startswith("value")), float(what.split()[1]), 0
    for b, t, slot in s.tokens():
        d = (7 * t + 5) % dim
        row, dims = s.host[which][slot, 1].copy(), slice(d // 32 * 32, d // 32 * 32 + 32) if kind == "mxfp4" else slice(d, d + 1)
        place = s.scale(which, slot)[d // 32:][:1] if kind == "mxfp4" else s.pools[which][slot, 1, d:d + 1]
        kept = place.clone()
        place.fill_(255 if kind == "mxfp4" else 0xff if kind == "fp8" else value)
        s.host[which][slot, 1, dims] = value
        seen += s.check(b, lambda *x: near(*x, kind == "fp8"))
        place.copy_(kept)
        s.host[which][slot, 1] = row
    assert seen > 0 and (s.run() == s.want).all()


@pytest.mark.parametrize("workspace", ["full", "none"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", [0, 1])
def test_fp8_scales_that_are_no_numbers(torch_cuda, which, value, dim, workspace):
    """A key's or value's FP32 scale of infinity or NaN: of a key, weights of zero or NaN
    by the sign of its score; of a value, infinities, and NaN where its code is 0."""
    torch = torch_cuda
    say(f"prompt fp8 D={dim}: {'value' if which else 'key'} scale {value}, workspace={workspace}")
    s, seen = Special(torch, "fp8", dim, none(torch) if workspace == "none" else None), 0
    for b, t, slot in s.tokens():
        row, place = s.host[which][slot, 1].copy(), s.scale(which, slot)
        kept, codes = place.clone(), s.pools[which].view(torch.float8_e4m3fn)[slot, 1].double().cpu().numpy()
        place.fill_(value)
        if which == 0 and np.isinf(value):
            a, z = s.starts[b], s.starts[b + 1]
            seen += s.check(b, lambda *x: without(*x, t, s.q[a:z, s.GROUP:] @ codes))
        else:
            with np.errstate(invalid="ignore"):
                s.host[which][slot, 1] = codes * value
            seen += s.check(b, lambda *x: near(*x, True))
        place.copy_(kept)
        s.host[which][slot, 1] = row
    assert seen > 0 and (s.run() == s.want).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("apart", [2 ** 28 - 16, 2 ** 28, 2 ** 28 + 16])
def test_rows_that_lie_far_apart(torch_cuda, apart, dim):
    """Rows of keys and values 256 MiB apart and a little less and more, K and V in one
    buffer of 35 GB: places in a tile pass 32 bits."""
    torch = torch_cuda
    say(f"prompt: rows {apart} bytes apart, D={dim}")
    heads, group, new, n = 1, 3, 40, 130
    c = Rows(torch, [new], [n - new], heads, group, dim, seed=dim, spare=0)
    buffer = torch.empty(apart * (n - 1) // 2 + 4096, dtype=torch.bfloat16, device="cuda")
    far = [buffer[at:].as_strided((n, heads * dim), (apart // 2, 1)) for at in (0, 1024)]
    far[0].copy_(c.k)
    far[1].copy_(c.v)
    kept = c.k, c.v
    for k, v in (far, (far[0], kept[1]), (kept[0], far[1])):
        c.k, c.v = k, v
        for ws in (None, none(torch)):
            c.out.fill_(5.0)
            c.call(ws)
            c.check()
