"""What the operators of a 4-bit decode step refuse, checked on the host before
any HIP call, and the calls that have nothing to do. No GPU needed."""
import pytest

import pbe_handoff as P

FAKE = 1 << 40  # never dereferenced: every case fails (or returns) first
POOLS = dict(key_pool=FAKE, key_pool_bytes=1 << 20, value_pool=FAKE, value_pool_bytes=1 << 20, key_scales=FAKE,
             key_scale_bytes=1 << 16, value_scales=FAKE, value_scale_bytes=1 << 16)
INVALID, UNSUPPORTED = P.PBE_ERR_INVALID, P.PBE_ERR_UNSUPPORTED


def refused(call, args, change, code):
    with pytest.raises(P.PbeError) as e:
        call(**{**args, **change})
    assert e.value.code == code, change
    assert str(e.value)


ROWS = [(dict(n_tokens=-1), INVALID), (dict(kv_heads=0), INVALID), (dict(head_dim=0), INVALID), (dict(head_dim=96), UNSUPPORTED),
        (dict(head_dim=256), UNSUPPORTED), (dict(slots=0), INVALID), (dict(keys=0), INVALID), (dict(values=0), INVALID),
        (dict(keys=FAKE + 8), INVALID), (dict(values=FAKE + 2), INVALID), (dict(key_pool=0), INVALID), (dict(value_pool=0), INVALID),
        (dict(key_scales=0), INVALID), (dict(value_scales=0), INVALID), (dict(key_pool=FAKE + 2), INVALID),
        (dict(value_scales=FAKE + 1), INVALID), (dict(n_tokens=2 ** 31 - 1), INVALID), (dict(kv_heads=2 ** 31 - 1), INVALID),
        (dict(device=-1), INVALID)]


@pytest.mark.parametrize("change,code", ROWS + [(dict(in_dtype=7), INVALID)])
def test_mxfp4_writer_refuses(change, code):
    refused(P.scatter_kv_mxfp4, dict(POOLS, keys=FAKE, values=FAKE, in_dtype=P.PBE_IN_BF16, n_tokens=4, slots=FAKE, kv_heads=2, head_dim=64),
            change, code)


@pytest.mark.parametrize("change,code", ROWS)
def test_mxfp4_gather_refuses(change, code):
    refused(P.gather_kv_mxfp4, dict(POOLS, keys=FAKE, values=FAKE, n_tokens=4, slots=FAKE, kv_heads=2, head_dim=64), change, code)


def test_no_tokens_are_no_work():
    P.scatter_kv_mxfp4(**POOLS, keys=0, values=0, in_dtype=P.PBE_IN_F32, n_tokens=0, slots=0, kv_heads=2, head_dim=64)
    P.gather_kv_mxfp4(**POOLS, keys=0, values=0, n_tokens=0, slots=0, kv_heads=2, head_dim=64)
