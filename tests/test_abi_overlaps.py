"""Calls of a 4-bit decode step whose outputs lie over what they read, and slots
that are not aligned: refused on the host, before any HIP call. No GPU needed."""
import pytest

import pbe_handoff as P

KEY, VALUE, KEY_SCALES, VALUE_SCALES, ROWS_K, ROWS_V, SLOTS, OTHER = (1 << 40 | i << 24 for i in range(8))
POOLS = dict(key_pool=KEY, key_pool_bytes=1 << 20, value_pool=VALUE, value_pool_bytes=1 << 20, key_scales=KEY_SCALES,
             key_scale_bytes=1 << 16, value_scales=VALUE_SCALES, value_scale_bytes=1 << 16)
ROWS = dict(POOLS, keys=ROWS_K, values=ROWS_V, n_tokens=4, slots=SLOTS, kv_heads=2, head_dim=64)   # rows of 4 x 256 bytes
FULL, SCALES = 1 << 20, 1 << 16


def refused(call, args, change, says):
    with pytest.raises(P.PbeError, match=says) as e:
        call(**{**args, **change})
    assert e.value.code == P.PBE_ERR_INVALID


def passed(call, args, change):
    """Gets as far as the device, which has no such addresses (or is none)."""
    with pytest.raises(P.PbeError) as e:
        call(**{**args, **change})
    assert "must be memory of device" in str(e.value) or e.value.code == P.PBE_ERR_HIP


PAGES = [("key_pool", FULL), ("value_pool", FULL), ("key_scales", SCALES), ("value_scales", SCALES)]
AT = dict(key_pool=KEY, value_pool=VALUE, key_scales=KEY_SCALES, value_scales=VALUE_SCALES)
OVER = [(rows, AT[name] + off) for rows in ("keys", "values") for name, size in PAGES for off in (0, size - 16, -1008)]
BESIDE = [(rows, AT[name] + off) for rows in ("keys", "values") for name, size in PAGES for off in (size, -1024)]


@pytest.mark.parametrize("what,to", OVER)
def test_rows_over_pages(what, to):
    refused(P.scatter_kv_mxfp4, dict(ROWS, in_dtype=P.PBE_IN_BF16), {what: to}, "apart")
    refused(P.gather_kv_mxfp4, ROWS, {what: to}, "apart")


@pytest.mark.parametrize("what,to", BESIDE)
def test_rows_beside_pages(what, to):
    passed(P.scatter_kv_mxfp4, dict(ROWS, in_dtype=P.PBE_IN_BF16), {what: to})
    passed(P.gather_kv_mxfp4, ROWS, {what: to})


def test_slots_and_rows():
    writer = dict(ROWS, in_dtype=P.PBE_IN_BF16)
    for off in (1, 2, 3):
        refused(P.scatter_kv_mxfp4, writer, dict(slots=SLOTS + off), "aligned")
        refused(P.gather_kv_mxfp4, ROWS, dict(slots=SLOTS + off), "aligned")
    refused(P.scatter_kv_mxfp4, writer, dict(slots=KEY_SCALES + SCALES - 4), "apart")
    refused(P.gather_kv_mxfp4, ROWS, dict(slots=ROWS_V - 12), "apart")
    refused(P.gather_kv_mxfp4, ROWS, dict(values=ROWS_K), "apart")
    refused(P.gather_kv_mxfp4, ROWS, dict(values=ROWS_K + 1008), "apart")
    passed(P.gather_kv_mxfp4, ROWS, dict(values=ROWS_K + 1024, slots=ROWS_K - 16))
    passed(P.gather_kv_mxfp4, ROWS, dict(slots=KEY))                         # both are read
    passed(P.scatter_kv_mxfp4, writer, dict(values=ROWS_K, slots=ROWS_K))    # all are read
    # K's and V's planes of an arena's layer, which lie within each other's bytes
    passed(P.scatter_kv_mxfp4, writer, dict(value_pool=KEY + 1024, value_scales=KEY_SCALES + 64))


Q, K, V, W, COS, POS, Q_OUT = (OTHER + (i << 16) for i in range(7))
ROPE = dict(POOLS, q=Q, q_stride=128, k=K, k_stride=64, v=V, v_stride=64, in_dtype=P.PBE_IN_BF16, n_tokens=4, q_heads=2, kv_heads=1, head_dim=64,
            q_weight=W, k_weight=W + 128, eps=1e-6, positions=POS, cos_sin=COS, max_position=64, rotary_dim=64, rope_style=P.PBE_ROPE_HALVES,
            slots=SLOTS, block_size=16, kv_dtype=P.PBE_KV_MXFP4, q_out=Q_OUT)


@pytest.mark.parametrize("name,size", PAGES)
def test_rope_writers_pages_lie_apart(name, size):
    at = AT[name]
    for change in (dict(q_out=at), dict(q_out=at + size - 16), dict(q=at - 1008), dict(k=at), dict(v=at + 64), dict(q_weight=at),
                   dict(k_weight=at + 16), dict(cos_sin=at - 64 * 64 * 4 + 16), dict(positions=at + size - 4), dict(slots=at - 12)):
        refused(P.qk_norm_rope_scatter, ROPE, change, "apart")
    passed(P.qk_norm_rope_scatter, ROPE, dict(q_out=at + size))
    passed(P.qk_norm_rope_scatter, ROPE, dict(q_out=at - 1024))


def test_rope_writers_bf16_pages_have_no_scales():
    bf16 = dict(ROPE, kv_dtype=P.PBE_KV_BF16)
    passed(P.qk_norm_rope_scatter, bf16, dict(q_out=KEY_SCALES))
    refused(P.qk_norm_rope_scatter, bf16, dict(q_out=VALUE), "apart")


READ = dict(key_pool=KEY, value_pool=VALUE, pool_bytes=FULL, key_scales=KEY_SCALES, value_scales=VALUE_SCALES, scale_pool_bytes=SCALES, kv_heads=2,
            head_dim=128, queries=ROWS_K, outputs=ROWS_V, batch=2, q_heads=12, tables=SLOTS, seq_lens=SLOTS + 4096, max_blocks=4, splits=2,
            workspace=OTHER, workspace_bytes=1 << 20)
OUT, NEED = 2 * 12 * 128 * 2, 2 * 12 * 2 * (130 * 4 + 8)


def test_reader_writes_apart_from_what_it_reads():
    for what, size in (("outputs", OUT), ("workspace", NEED)):
        for at, end in ((KEY, FULL), (VALUE, FULL), (KEY_SCALES, SCALES), (VALUE_SCALES, SCALES), (SLOTS, 2 * 4 * 4)):
            refused(P.paged_decode_mxfp4, READ, {what: at}, "apart")
            refused(P.paged_decode_mxfp4, READ, {what: at - size + 16}, "apart")
            passed(P.paged_decode_mxfp4, READ, {what: at - size})
        refused(P.paged_decode_mxfp4, READ, {what: SLOTS + 4096}, "apart")
    refused(P.paged_decode_mxfp4, READ, dict(workspace=ROWS_K + OUT - 16), "apart")
    refused(P.paged_decode_mxfp4, READ, dict(workspace=ROWS_V - NEED + 16), "apart")
    refused(P.paged_decode_mxfp4, READ, dict(outputs=ROWS_K + 16), "apart")
    passed(P.paged_decode_mxfp4, READ, dict(outputs=ROWS_K))
    passed(P.paged_decode_mxfp4, READ, dict(outputs=ROWS_K + OUT))
    passed(P.paged_decode_mxfp4, READ, dict(splits=1, workspace=ROWS_V))   # one piece takes no workspace
