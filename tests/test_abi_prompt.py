"""What the prompt readers and page movers refuse, checked on the host before any HIP
call, and the calls that have nothing to do. No GPU needed."""
import pytest

import pbe_handoff as P

FAKE = 1 << 40  # never dereferenced: every case fails (or returns) first
INVALID, UNSUPPORTED = P.PBE_ERR_INVALID, P.PBE_ERR_UNSUPPORTED


def refused(call, args, change, code):
    with pytest.raises(P.PbeError) as e:
        call(**{**args, **change})
    assert e.value.code == code, change
    assert str(e.value)


MB = 1 << 20
ROWS = dict(q=FAKE, q_stride=768, k=FAKE + MB, k_stride=256, v=FAKE + 2 * MB, v_stride=256, n_queries=10, n_keys=12, q_starts=FAKE + 3 * MB,
            k_starts=FAKE + 3 * MB + 64, batch=2, q_heads=6, kv_heads=2, head_dim=128, outputs=FAKE + 4 * MB, workspace=FAKE + 64 * MB,
            workspace_bytes=1 << 30)


@pytest.mark.parametrize("change,code", [
    (dict(n_queries=-1), INVALID), (dict(n_keys=-1), INVALID), (dict(n_keys=2 ** 31 - 1), INVALID), (dict(batch=0), INVALID), (dict(q_heads=0), INVALID),
    (dict(kv_heads=0), INVALID), (dict(device=-1), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED),
    (dict(q_heads=7), UNSUPPORTED), (dict(n_queries=2 ** 30), INVALID), (dict(q=0), INVALID), (dict(k=0), INVALID), (dict(v=0), INVALID),
    (dict(outputs=0), INVALID), (dict(q_starts=0), INVALID), (dict(k_starts=0), INVALID), (dict(q=FAKE + 8), INVALID), (dict(k=FAKE + MB + 2), INVALID),
    (dict(outputs=FAKE + 4 * MB + 8), INVALID), (dict(workspace=FAKE + 64 * MB + 4), INVALID), (dict(q_starts=FAKE + 3 * MB + 2), INVALID),
    (dict(k_starts=FAKE + 3 * MB + 65), INVALID), (dict(q_stride=760), INVALID), (dict(k_stride=128), INVALID), (dict(v_stride=260), INVALID),
    (dict(q_stride=-768), INVALID), (dict(k_stride=1 << 60), INVALID), (dict(outputs=FAKE + MB), INVALID), (dict(outputs=FAKE + 16), INVALID),
    (dict(outputs=FAKE + 3 * MB - 16), INVALID), (dict(outputs=FAKE, q_stride=776), INVALID), (dict(workspace=FAKE + 2 * MB, n_keys=4000), INVALID),
    (dict(workspace=FAKE + 4 * MB, n_keys=4000), INVALID), (dict(q_heads=2 ** 25, kv_heads=2 ** 24, n_queries=1), INVALID)])
def test_row_reader_refuses(change, code):
    refused(P.prompt_attention, ROWS, change, code)


PAGES = dict(key_pool=FAKE, value_pool=FAKE + MB, pool_bytes=MB, key_scales=FAKE + 2 * MB, value_scales=FAKE + 3 * MB, scale_pool_bytes=MB,
             kv_dtype=P.PBE_KV_FP8_E4M3, kv_heads=2, head_dim=128, queries=FAKE + 4 * MB, outputs=FAKE + 5 * MB, n_rows=10,
             token_starts=FAKE + 6 * MB, batch=2, q_heads=6, tables=FAKE + 7 * MB, seq_lens=FAKE + 8 * MB, max_blocks=50,
             workspace=FAKE + 64 * MB, workspace_bytes=1 << 30)


@pytest.mark.parametrize("change,code", [
    (dict(n_rows=-1), INVALID), (dict(batch=0), INVALID), (dict(q_heads=0), INVALID), (dict(kv_heads=0), INVALID), (dict(max_blocks=0), INVALID),
    (dict(device=-1), INVALID), (dict(kv_dtype=3), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(q_heads=7), UNSUPPORTED),
    (dict(key_pool=0), INVALID), (dict(value_pool=0), INVALID), (dict(key_scales=0), INVALID), (dict(value_scales=0), INVALID), (dict(queries=0), INVALID),
    (dict(outputs=0), INVALID), (dict(token_starts=0), INVALID), (dict(tables=0), INVALID), (dict(seq_lens=0), INVALID), (dict(key_pool=FAKE + 8), INVALID),
    (dict(value_scales=FAKE + 3 * MB + 2), INVALID), (dict(queries=FAKE + 4 * MB + 8), INVALID), (dict(outputs=FAKE + 5 * MB + 2), INVALID),
    (dict(tables=FAKE + 7 * MB + 1), INVALID), (dict(pool_bytes=4095), INVALID), (dict(scale_pool_bytes=127), INVALID),
    (dict(kv_dtype=P.PBE_KV_MXFP4, pool_bytes=2047), INVALID), (dict(kv_dtype=P.PBE_KV_BF16, pool_bytes=8191), INVALID), (dict(outputs=FAKE + 16), INVALID),
    (dict(outputs=FAKE + 4 * MB + 16), INVALID), (dict(outputs=FAKE + 6 * MB - 16), INVALID), (dict(workspace=FAKE + 5 * MB), INVALID),
    (dict(batch=2 ** 20, max_blocks=2 ** 30), INVALID), (dict(n_rows=2 ** 30), INVALID)])
def test_page_reader_refuses(change, code):
    refused(P.paged_prompt_attention, PAGES, change, code)


def test_no_rows_are_no_work():
    P.prompt_attention(**{**ROWS, "n_queries": 0, "q": 0, "outputs": 0, "q_starts": 0, "workspace": 0, "workspace_bytes": 0})
    P.paged_prompt_attention(**{**PAGES, "n_rows": 0, "queries": 0, "outputs": 0, "token_starts": 0})


def test_workspace_sizes():
    assert P.prompt_workspace_bytes(0, 1, 12, 2, 128) == P.prompt_workspace_bytes(5, 1, 13, 2, 128) == P.prompt_workspace_bytes(5, 0, 12, 2, 128) == 0
    assert P.prompt_workspace_bytes(100000, 1, 28, 4, 128) == 0     # tiles enough to fill any GPU
    assert 0 < P.prompt_workspace_bytes(64, 1, 12, 2, 128) < 1 << 28
    assert P.fork_pages_workspace_bytes(100, 3, 5) == 4 * (16 + 100 + 3 + 20)
    assert P.compact_pages_workspace_bytes(100) == 4 * 316
    assert P.fork_pages_workspace_bytes(0, 3, 5) == P.compact_pages_workspace_bytes(0) == 0


def planes(n=1, page=4096, pages=64, at=FAKE, segment=0, apart=16 * MB):
    views = []
    for i in range(n):
        seg = segment or page * pages
        views.append((P.view_of([at + i * apart + s * seg for s in range(-(-page * pages // seg))], page * pages, seg), page))
    return P.page_planes(views)


FORK = dict(planes=planes(), n_pages=64, id_stride=2, block_size=16, tables_in=FAKE + 1024 * MB, lens_in=FAKE + 1025 * MB, rows_in=4,
            parents=FAKE + 1026 * MB, new_lens=FAKE + 1027 * MB, rows_out=6, max_blocks=8, reserved=FAKE + 1028 * MB, tables_out=FAKE + 1029 * MB,
            lens_out=FAKE + 1030 * MB, counts=FAKE + 1031 * MB, workspace=FAKE + 1032 * MB, workspace_bytes=MB)
COMPACT = dict(planes=planes(), n_pages=64, id_stride=2, tables_in=FAKE + 1024 * MB, rows=4, max_blocks=8, reserved=FAKE + 1025 * MB,
               tables_out=FAKE + 1026 * MB, moved_to=FAKE + 1027 * MB, counts=FAKE + 1028 * MB, workspace=FAKE + 1029 * MB, workspace_bytes=MB)
POOL = [(dict(n_pages=0), INVALID), (dict(id_stride=0), INVALID), (dict(n_pages=(1 << 20) + 1), UNSUPPORTED), (dict(id_stride=2 ** 26), INVALID),
        (dict(max_blocks=0), INVALID), (dict(max_blocks=2 ** 30), INVALID), (dict(device=-1), INVALID), (dict(tables_in=0), INVALID),
        (dict(tables_out=0), INVALID), (dict(counts=0), INVALID), (dict(workspace=0), INVALID), (dict(workspace_bytes=300), INVALID),
        (dict(planes=planes(113)), UNSUPPORTED), (dict(planes=planes(page=4104)), INVALID), (dict(planes=planes(pages=63)), INVALID),
        (dict(planes=planes(at=FAKE + 8)), INVALID), (dict(planes=planes(segment=4096 * 5 + 16)), INVALID), (dict(planes=planes(2, apart=4096)), INVALID),
        (dict(planes=planes(20, segment=4096 * 4)), UNSUPPORTED), (dict(tables_in=FAKE + 1024 * MB + 2), INVALID), (dict(tables_out=FAKE + 1024 * MB), INVALID),
        (dict(counts=FAKE + 4096), INVALID), (dict(tables_in=FAKE + 4096), INVALID), (dict(workspace=FAKE + 1024 * MB), INVALID)]


@pytest.mark.parametrize("change,code", POOL + [
    (dict(block_size=0), INVALID), (dict(rows_in=0), INVALID), (dict(rows_out=0), INVALID), (dict(lens_in=0), INVALID), (dict(parents=0), INVALID),
    (dict(lens_out=0), INVALID), (dict(lens_out=FAKE + 1025 * MB), INVALID), (dict(parents=FAKE + 1030 * MB + 4), INVALID)])
def test_fork_refuses(change, code):
    refused(P.fork_pages, FORK, change, code)


@pytest.mark.parametrize("change,code", POOL + [(dict(rows=0), INVALID), (dict(moved_to=FAKE + 1025 * MB), INVALID)])
def test_compact_refuses(change, code):
    refused(P.compact_pages, COMPACT, change, code)
