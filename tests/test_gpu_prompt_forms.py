"""Calls of pbe_prompt_attention and pbe_paged_prompt_attention at the ends of what
they take, over values for which every output is known, or within the bound of
test_gpu_prompt.py."""
import numpy as np
import pytest

import pbe_handoff as P
from tests.conftest import say
from tests.gpu_util import stream_ptr
from tests.test_gpu_prompt import within

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
