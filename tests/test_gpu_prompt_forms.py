"""Calls of pbe_prompt_attention and pbe_paged_prompt_attention at the ends of what
they take, over values for which every output is known, or within the bound of
test_gpu_prompt.py."""
import numpy as np
import pytest

import pbe_handoff as P
from tests.conftest import say
from tests.gpu_util import stream_ptr

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
