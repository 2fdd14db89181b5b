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


STEP = dict(page_ids=FAKE, n_page_ids=8, page_starts=FAKE + 0x1000, cached_lens=FAKE + 0x2000, new_lens=FAKE + 0x3000, batch=4, block_size=16,
            block_tables=FAKE + 0x4000, max_blocks=4, seq_lens=FAKE + 0x5000, token_starts=FAKE + 0x6000, slots=FAKE + 0x7000,
            positions=FAKE + 0x8000, max_tokens=9)


@pytest.mark.parametrize("change", [
    dict(batch=0), dict(batch=-1), dict(block_size=0), dict(max_blocks=0), dict(max_tokens=0), dict(n_page_ids=-1), dict(n_page_ids=1 << 31),
    dict(batch=1 << 20, max_blocks=1 << 11), dict(page_ids=0), dict(page_starts=0), dict(cached_lens=0), dict(block_tables=0), dict(seq_lens=0),
    dict(token_starts=0), dict(slots=0), dict(positions=0), dict(slots=FAKE + 0x7002), dict(device=-1),
    dict(seq_lens=FAKE + 0x2000), dict(positions=FAKE + 0x7000 + 4 * 8), dict(block_tables=FAKE + 4 * 7), dict(token_starts=FAKE + 0x3000 - 16)])
def test_step_tables_refuse(change):
    refused(P.build_step_tables, STEP, change, INVALID)


ROPE = dict(q=FAKE, q_stride=256, k=FAKE + 512, k_stride=256, v=FAKE + 768, v_stride=256, in_dtype=P.PBE_IN_BF16, n_tokens=4, q_heads=2, kv_heads=1,
            head_dim=64, q_weight=FAKE, k_weight=FAKE, eps=1e-6, positions=FAKE, cos_sin=FAKE, max_position=64, rotary_dim=64,
            rope_style=P.PBE_ROPE_HALVES, slots=FAKE, block_size=16, kv_dtype=P.PBE_KV_BF16, q_out=FAKE + (1 << 20), key_pool=FAKE,
            key_pool_bytes=1 << 20, value_pool=FAKE, value_pool_bytes=1 << 20)
SCALES = dict(key_scales=FAKE, key_scale_bytes=1 << 16, value_scales=FAKE, value_scale_bytes=1 << 16)


@pytest.mark.parametrize("change,code", [
    (dict(in_dtype=2), INVALID), (dict(kv_dtype=3), INVALID), (dict(rope_style=2), INVALID), (dict(n_tokens=-1), INVALID), (dict(q_heads=0), INVALID),
    (dict(kv_heads=0), INVALID), (dict(block_size=0), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED),
    (dict(kv_dtype=P.PBE_KV_MXFP4, block_size=32, **SCALES), UNSUPPORTED), (dict(rotary_dim=24), INVALID), (dict(rotary_dim=80), INVALID),
    (dict(rotary_dim=-16), INVALID), (dict(max_position=0), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(eps=float("inf")), INVALID), (dict(n_tokens=2 ** 31 - 1), INVALID), (dict(q_heads=2 ** 31 - 1), INVALID), (dict(q=0), INVALID),
    (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(slots=0), INVALID), (dict(q_out=0), INVALID), (dict(key_pool=0), INVALID),
    (dict(value_pool=0), INVALID), (dict(positions=0), INVALID), (dict(cos_sin=0), INVALID), (dict(kv_dtype=P.PBE_KV_FP8_E4M3), INVALID),
    (dict(kv_dtype=P.PBE_KV_MXFP4), INVALID), (dict(q_stride=120), INVALID), (dict(k_stride=8), INVALID), (dict(v_stride=65), INVALID),
    (dict(q_stride=-256), INVALID), (dict(q_stride=1 << 62), INVALID), (dict(q=FAKE + 8), INVALID), (dict(q_weight=FAKE + 4), INVALID),
    (dict(cos_sin=FAKE + 4), INVALID), (dict(q_out=FAKE + (1 << 20) + 8), INVALID), (dict(positions=FAKE + 2), INVALID),
    (dict(key_pool=FAKE + 8), INVALID), (dict(SCALES, kv_dtype=P.PBE_KV_FP8_E4M3, value_pool=FAKE + 4), INVALID),
    (dict(SCALES, kv_dtype=P.PBE_KV_MXFP4, key_pool=FAKE + 2), INVALID), (dict(q_out=FAKE + 1024), INVALID), (dict(device=-1), INVALID)])
def test_rope_writer_refuses(change, code):
    refused(P.qk_norm_rope_scatter, ROPE, change, code)


@pytest.mark.parametrize("change,says", [
    (dict(eps=0.0), "eps"), (dict(eps=2.0 ** -127), "eps"), (dict(eps=0.0, q_weight=0), "eps"),
    (dict(n_tokens=1, q_heads=2 ** 24, head_dim=128), "4 GiB"),
    (dict(n_tokens=1, q_heads=2 ** 23, head_dim=128, in_dtype=P.PBE_IN_F32), "4 GiB"),
    (dict(q_weight=FAKE + (1 << 20)), "apart"), (dict(k_weight=FAKE + (1 << 20) + 1008), "apart"), (dict(cos_sin=FAKE + (1 << 20) - 256), "apart"),
    (dict(positions=FAKE + (1 << 20) - 12), "apart"), (dict(slots=FAKE + (1 << 20) + 4), "apart")])
def test_rope_writer_names_what_it_refuses(change, says):
    with pytest.raises(P.PbeError, match=says) as e:
        P.qk_norm_rope_scatter(**{**ROPE, **change})
    assert e.value.code == INVALID


def test_rope_writer_without_tokens_is_no_work():
    P.qk_norm_rope_scatter(**{**ROPE, "n_tokens": 0, "q": 0, "k": 0, "v": 0, "slots": 0, "q_out": 0})


READ = dict(key_pool=FAKE, value_pool=FAKE, pool_bytes=1 << 20, key_scales=FAKE, value_scales=FAKE, scale_pool_bytes=1 << 16, kv_heads=2,
            head_dim=128, queries=FAKE, outputs=FAKE, batch=2, q_heads=12, tables=FAKE, seq_lens=FAKE, max_blocks=4, splits=2, workspace=FAKE,
            workspace_bytes=1 << 20)


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), INVALID), (dict(q_heads=0), INVALID), (dict(kv_heads=0), INVALID), (dict(max_blocks=0), INVALID), (dict(head_dim=96), UNSUPPORTED),
    (dict(q_heads=13), UNSUPPORTED), (dict(q_heads=34), UNSUPPORTED), (dict(key_pool=0), INVALID), (dict(value_pool=0), INVALID),
    (dict(key_scales=0), INVALID), (dict(value_scales=0), INVALID), (dict(queries=0), INVALID), (dict(outputs=0), INVALID), (dict(tables=0), INVALID),
    (dict(seq_lens=0), INVALID), (dict(queries=FAKE + 8), INVALID), (dict(outputs=FAKE + 2), INVALID), (dict(value_pool=FAKE + 8), INVALID),
    (dict(key_scales=FAKE + 2), INVALID), (dict(workspace=FAKE + 8), INVALID), (dict(splits=-1), INVALID), (dict(splits=1025), INVALID),
    (dict(workspace=0), INVALID), (dict(workspace_bytes=2 * 12 * 2 * (130 * 4 + 8) - 1), INVALID), (dict(pool_bytes=2047), INVALID),
    (dict(scale_pool_bytes=127), INVALID), (dict(kv_heads=2 ** 27, q_heads=2 ** 27), INVALID), (dict(batch=2 ** 30, q_heads=32), INVALID),
    (dict(batch=2 ** 20, max_blocks=2 ** 30), INVALID), (dict(device=-1), INVALID)])
def test_mxfp4_reader_refuses(change, code):
    refused(P.paged_decode_mxfp4, READ, change, code)


def test_mxfp4_splits_and_workspace():
    assert P.decode_mxfp4_splits(0, 2, 10) == P.decode_mxfp4_splits(2, 0, 10) == P.decode_mxfp4_splits(2, 2, 0) == 1
    assert P.decode_mxfp4_splits(100000, 8, 4096) == P.decode_mxfp4_splits(512, 8, 4096) == 1
    for batch, heads, blocks in ((1, 2, 315), (64, 4, 2048), (7, 1, 1), (1, 1, 1 << 27)):
        assert 1 <= P.decode_mxfp4_splits(batch, heads, blocks) <= min(1024, blocks)
    assert P.decode_mxfp4_workspace_bytes(3, 12, 128, 1) == 0
    assert P.decode_mxfp4_workspace_bytes(3, 12, 128, 7) == 3 * 12 * 7 * (130 * 4 + 8)
    assert P.decode_mxfp4_workspace_bytes(0, 12, 128, 7) == 0
