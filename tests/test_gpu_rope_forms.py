"""Forms of pbe_qk_norm_rope_scatter that long prompts of FP32 rows, and of heads
of which a part turns in halves, take: runs of two and of four heads."""
import pytest

import pbe_handoff as P
from tests.conftest import say
from tests.gpu_util import stream_ptr
from tests.test_gpu_rope import Rope

pytestmark = pytest.mark.gpu

RUNS_OF_TWO = [(1000, 4, 7, 128), (3700, 2, 7, 64)]
RUNS_OF_FOUR = [(2800, 4, 7, 128), (2001, 5, 7, 128), (11000, 2, 7, 64)]


FORMS = [("whole", True), ("half", True), ("half", False), ("half in pairs", True), ("none", True)]


@pytest.mark.parametrize("turned,f32", FORMS, ids=[f"{t}-{'f32' if f else 'bf16'}" for t, f in FORMS])
@pytest.mark.parametrize("n,heads,group,dim", RUNS_OF_TWO + RUNS_OF_FOUR)
def test_long_prompts_of_either_type(torch_cuda, n, heads, group, dim, turned, f32):
    say(f"qk_norm_rope n={n} H={heads}x{group} D={dim} turned={turned} f32={f32}")
    rotary = {"whole": dim, "none": 0}.get(turned, dim // 2)
    r = Rope(torch_cuda, n, heads, group, dim, rotary, f32, pairs="pairs" in turned, seed=n + rotary)
    bufs, args = r.pools(P.PBE_KV_BF16)
    r.call(P.PBE_KV_BF16, args, stream_ptr(torch_cuda))
    r.check_bf16(bufs)
