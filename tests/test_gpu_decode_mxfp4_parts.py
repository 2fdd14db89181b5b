"""pbe_paged_decode_mxfp4 on batches of more workgroups than a launch takes (fewer
than 2^24 of 256 threads), which it reads in parts one after another."""
import pytest

import pbe_handoff as P
from tests.conftest import say
from tests.gpu_util import stream_ptr

pytestmark = pytest.mark.gpu

T = 16


def test_batches_beyond_one_launch(torch_cuda):
    """65,532 sequences of 256 KV heads: 65,528 whole ones fill a launch, and 65,526
    that may be cut, so that the last six are read by themselves, the long one of them
    in pieces. Whole sequences give the bits that they give in smaller batches; in
    pieces, a sum in another order moves an output by a step of BF16 at most, 2^-7 of
    it, and by 2^-15 of the values for the weights, and their 700 tokens' FP32
    roundings, on either side: below 2^-13 of the largest value."""
    torch = torch_cuda
    say("decode mxfp4 of 65,532 sequences x 256 heads")
    batch, heads, dim, blocks, longest = 65532, 256, 64, 50, 700
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    half = T * heads * dim // 2
    k, v = (torch.randint(0, 256, (blocks * half,), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.randint(122, 127, (blocks * half // 16,), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
    most = -(-longest // T)
    tables = torch.randint(0, blocks, (batch, most), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, 40, (batch,), generator=g, device="cuda", dtype=torch.int32)
    for b, n in ((0, longest), (7, 0), (65524, 500), (65525, 333), (65530, longest)):
        lens[b] = n
    q = torch.randn((batch, heads, dim), generator=g, device="cuda", dtype=torch.bfloat16)

    def call(first, n, splits, out, ws):
        P.paged_decode_mxfp4(k.data_ptr(), v.data_ptr(), k.numel(), ks.data_ptr(), vs.data_ptr(), ks.numel(), heads, dim, q[first].data_ptr(),
                             out[first].data_ptr(), n, heads, tables[first].data_ptr(), lens[first:].data_ptr(), most, splits,
                             ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0, stream=stream_ptr(torch))
        torch.cuda.synchronize()

    want, got = torch.empty_like(q), torch.full_like(q, 5.0)
    step = batch // 3
    for first in range(0, batch, step):
        call(first, step, 1, want, None)
    assert torch.isfinite(want[::97].float()).all() and (want[7] == 0).all()
    call(0, batch, 1, got, None)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    ws = torch.full((P.decode_mxfp4_workspace_bytes(batch, heads, dim, 2),), 0xff, dtype=torch.uint8, device="cuda")
    got.fill_(5.0)
    call(0, batch, 2, got, ws)
    for first in range(0, batch, step):
        a, b = got[first:first + step].float(), want[first:first + step].float()
        assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -13 * 6 * 2.0 ** (126 - 127)).all(), first
