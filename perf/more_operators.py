"""A prefill worker's attention over prompts, and the page moves of requests that
share a cache, operator by operator, as measurable cases through the package's
public entry points.

Kinds of work (`case["kind"]`):
  rows     causal attention over whole prompts, packed one after another, with
           grouped query heads; keys and values as BF16 rows (prompt_attention)
  pages    the same for the new tokens of a step, whose keys and values lie in
           the pages of a cache together with those before them: BF16 pages, FP8
           E4M3 pages with a scale per token and head, or MXFP4 pages
           (paged_prompt_attention)
  fork     the next step's requests from the last one's: requests that go on,
           fork, end and grow, with the pages that forks write to copied
           (fork_pages)
  compact  the pages in use moved to the front of their pool (compact_pages)

A query i of a request's n new tokens, of `length` tokens in all, sees the tokens
up to position length - n + i. Pages hold 16 tokens; FP8 and BF16 pages are rows
[token][head][dim], MXFP4 pages per KV head
  K       [4 quarters of the dims][16 tokens][dim/8 bytes]
  V       [4 quads of tokens][16 columns of dim/16 dims][4 tokens][dim/32 bytes]
  scales  [dim/32 groups][16 tokens], one byte each, for K and V alike
with the even dim of a byte's two E2M1 codes in its low four bits; a scale byte e
stands for 2^(e - 127).

Head layouts and page sizes are those of this repository's workloads (2 KV heads x
64, 2 x 128 and 4 x 128 with 7, 6 and 7 query heads each; 24, 28 and 28 layers);
drawn cases take others too.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

B = 16    # tokens of a page
G = 32    # head dims that share an MXFP4 scale
# KV heads, head dim, query heads per KV head, layers
GEOMETRY = {"0.5b": (2, 64, 7, 24), "1.5b": (2, 128, 6, 28), "7b": (4, 128, 7, 28)}


def _layout(name):
    heads, dim, group, _ = GEOMETRY[name]
    return dict(heads=heads, dim=dim, group=group)


def _page(name):
    heads, dim, _, layers = GEOMETRY[name]
    return dict(page=2 * layers * B * heads * dim * 2, stride=2 * layers)


def listed():
    return [
        # One short question, one layer: launch-bound.
        dict(name="rows_0.5b_41", kind="rows", batch=1, new=41, cached=0, **_layout("0.5b"), mixed=False, packed=True),
        # Prompts of every length in one prefill batch, parts of packed QKV rows.
        dict(name="rows_1.5b_16_mixed", kind="rows", batch=16, new=2500, cached=0, **_layout("1.5b"), mixed=True, packed=True),
        # A chunk behind the 5040-token prefix, whose rows were read back from 4-bit pages.
        dict(name="rows_1.5b_2041_after_5040", kind="rows", batch=1, new=2041, cached=5040, **_layout("1.5b"), mixed=False, packed=False),
        # A whole long prompt: as much arithmetic as a layer's attention has.
        dict(name="rows_7b_8192", kind="rows", batch=1, new=8192, cached=0, **_layout("7b"), mixed=False, packed=False),
        # Four drafted tokens a request to be checked over long contexts.
        dict(name="pages_0.5b_64x4_fp8", kind="pages", batch=64, context=5040, new=4, **_layout("0.5b"), pages="fp8", mixed=False),
        # A chunk of a long prompt over BF16 pages.
        dict(name="pages_1.5b_2041_bf16", kind="pages", batch=1, context=7040, new=2041, **_layout("1.5b"), pages="bf16", mixed=False),
        # The last short chunk of a long prompt: few rows, many tokens to read.
        dict(name="pages_7b_128_fp8", kind="pages", batch=1, context=32768, new=128, **_layout("7b"), pages="fp8", mixed=False),
        # Chunked prefill beside decoding requests over a 4-bit cache.
        dict(name="pages_7b_24_mxfp4", kind="pages", batch=24, context=4096, new=512, **_layout("7b"), pages="mxfp4", mixed=True),
        # One prompt, four samples of it.
        dict(name="fork_1.5b_1to4", kind="fork", requests=1, beams=4, first=True, context=5051, pool=640, **_page("1.5b")),
        # A step of beam search: 64 requests of four beams each.
        dict(name="fork_0.5b_64x4", kind="fork", requests=64, beams=4, first=False, context=600, pool=3000, **_page("0.5b")),
        # A few pages of a small pool.
        dict(name="compact_0.5b_96", kind="compact", requests=4, context=200, pool=96, **_page("0.5b")),
        # A pool that requests have come to and left for long, before it is handed over.
        dict(name="compact_7b_1024", kind="compact", requests=24, context=700, pool=1024, **_page("7b")),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case: any kind, head layout, pages and option, sizes over their logarithm."""
    kind = rng.choice(["rows", "rows", "rows", "pages", "pages", "pages", "pages", "fork", "compact"])
    if kind in ("fork", "compact"):
        heads, dim, layers = rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.randint(1, 32)
        page = dict(page=2 * layers * B * heads * dim * 2, stride=2 * layers)
        pool = max(24, min(_log_int(rng, 24, 8192), 900000000 // page["page"]))
        if kind == "compact":
            requests = min(_log_int(rng, 1, 64), pool // 4)
            return dict(kind=kind, requests=requests, context=_log_int(rng, 8, max(16, pool // 2 // requests * B)), pool=pool, **page)
        beams = rng.randint(1, 6)
        requests = max(1, min(_log_int(rng, 1, 64), pool // (4 * beams)))
        room = max(1, pool // (requests * beams) - 3) * B
        return dict(kind=kind, requests=requests, beams=beams, first=rng.random() < 0.4, context=_log_int(rng, 8, max(16, room)), pool=pool, **page)
    layout = dict(heads=rng.choice([1, 2, 2, 3, 4, 4, 8]), dim=rng.choice([64, 128]), group=rng.randint(1, 8))
    batch = _log_int(rng, 1, 64)
    q_heads = layout["heads"] * layout["group"]
    most = 0.9e9 / (q_heads * batch)  # scores, as if all requests were the longest
    if kind == "rows":
        new = _log_int(rng, 1, min(8192, math.sqrt(most) * 0.8))
        cached = rng.choice([0, 0, _log_int(rng, 1, max(1, min(8192, most / new - new)))])
        return dict(kind=kind, batch=batch, new=new, cached=cached, **layout, mixed=batch > 1 and rng.random() < 0.7, packed=cached == 0 and rng.random() < 0.5)
    new = _log_int(rng, 1, min(4096, math.sqrt(most) * 0.7))
    context = _log_int(rng, max(new, 16), max(new, 16, min(32768, most / new, 1.5e8 / (batch * layout["heads"] * layout["dim"]))))
    return dict(kind=kind, batch=batch, context=context, new=new, **layout, pages=rng.choice(["bf16", "fp8", "mxfp4"]), mixed=batch > 1 and rng.random() < 0.6)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _requests(case, seed=0):
    """(tokens in all, new tokens of them) of each request, the same ones for
    every seed in an order of its own."""
    n, new = case["batch"], case["new"]
    r = random.Random(n * 100003 + new)
    if case["kind"] == "rows":
        cached = case["cached"]
        all_ = [(cached + new, new)] * n
        if case["mixed"]:
            news = [new] + [_log_int(r, min(16, new), new) for _ in range(n - 1)]
            all_ = [((r.randint(0, cached) if i else cached) + k, k) for i, k in enumerate(news)]
    else:
        most = case["context"]
        all_ = [(most, new)] * n
        if case["mixed"]:  # a quarter of them in prefill, the others decode
            news = [new] + [_log_int(r, 1, new) if i % 4 == 0 else 1 for i in range(1, n)]
            all_ = [(max(k, _log_int(r, min(16, most), most)) if i else most, k) for i, k in enumerate(news)]
    random.Random(seed).shuffle(all_)
    return all_


def _prepare_rows(case, seed):
    gen, reqs = _gen(seed), _requests(case, seed)
    heads, dim, group = case["heads"], case["dim"], case["group"]
    q_heads = heads * group
    lens, new = [list(x) for x in zip(*reqs)]
    n_q, n_k = sum(new), sum(lens)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    if case["packed"]:
        qkv = rand(n_q, (q_heads + 2 * heads) * dim)
        qkv[:, : q_heads * dim] *= 2
        qkv = qkv.to(torch.bfloat16)
        q, k, v = qkv.split([q_heads * dim, heads * dim, heads * dim], 1)
    else:
        q, k, v = ((rand(n, h * dim) * s).to(torch.bfloat16) for n, h, s in ((n_q, q_heads, 2), (n_k, heads, 1), (n_k, heads, 1)))
    s = dict(q=q, k=k, v=v, q_starts=_int(_starts(new)), k_starts=_int(_starts(lens)), out=torch.zeros((n_q, q_heads, dim), dtype=torch.bfloat16, device="cuda"),
             longest=max(lens), most_new=max(new))
    # partial results of rows whose keys are read in parts: at most 64 MB
    s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    return s


def _quantise(x):
    """E2M1 codes and E8M0 bytes of rows x[..., dim]: a group's power of two is
    that of its largest value less 2; values round to the nearest code."""
    x = x.unflatten(-1, (-1, G))
    scale = (torch.frexp(x.abs().amax(-1)).exponent - 3 + 127).clamp(0, 254)
    a = torch.ldexp(x.abs(), 127 - scale[..., None])
    code = sum((a > t).to(torch.uint8) for t in (0.25, 1.25, 2.5, 5.0)) + sum((a >= t).to(torch.uint8) for t in (0.75, 1.75, 3.5))
    code = (code | (x < 0).to(torch.uint8) << 3).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.to(torch.uint8)


def _fill_pages(case, blocks, gen):
    """Pools of one layer with N(0, 1) rows in every slot."""
    heads, dim, kind = case["heads"], case["dim"], case["pages"]
    s = {}
    for pool in ("k", "v"):
        rows = torch.randn((blocks, B, heads, dim), generator=gen, device="cuda")
        if kind == "bf16":
            s[pool] = rows.to(torch.bfloat16)
        elif kind == "fp8":
            scale = rows.abs().amax(-1) / 448
            s[pool], s[pool + "_scales"] = (rows / scale[..., None]).to(torch.float8_e4m3fn), scale
        else:
            codes, scale = _quantise(rows)
            codes = codes.transpose(1, 2)                                        # [block][head][token][dim/2]
            if pool == "k":
                codes = codes.unflatten(-1, (4, -1)).transpose(2, 3)             # [block][head][quarter][token][dim/8]
            else:
                codes = codes.unflatten(2, (4, 4)).unflatten(-1, (16, -1)).transpose(3, 4)  # [block][head][quad][column][token][dim/32]
            s[pool], s[pool + "_scales"] = codes.contiguous(), scale.permute(0, 2, 3, 1).contiguous()  # [block][head][group][token]
    return s


def _prepare_pages(case, seed):
    gen, reqs = _gen(seed), _requests(case, seed)
    q_heads, dim = case["heads"] * case["group"], case["dim"]
    lens, new = [list(x) for x in zip(*reqs)]
    counts = [-(-n // B) for n in lens]
    blocks, most = sum(counts) + 16, max(counts)
    s = _fill_pages(case, blocks, gen)
    ids = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    j = torch.arange(most, device="cuda")
    at = _int(_starts(counts)[:-1])[:, None] + j
    s["tables"] = torch.where(j < _int(counts)[:, None], ids[at.clamp(max=blocks - 1)], torch.full_like(at, -1, dtype=torch.int32)).contiguous()
    s["q"] = (torch.randn((sum(new), q_heads, dim), generator=gen, device="cuda") * 2).to(torch.bfloat16)
    s["out"] = torch.zeros_like(s["q"])
    s["q_starts"], s["lens"] = _int(_starts(new)), _int(lens)
    s["longest"], s["most_new"] = max(lens), max(new)
    s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    return s


def _rows_of(case):
    """Lengths of the requests' rows and, of a fork, each new row's parent."""
    r = random.Random(case["requests"] * 1009 + case["context"])
    lens = [case["context"]] + [r.randint(max(1, case["context"] // 3), case["context"]) for _ in range(case["requests"] - 1)]
    if case["kind"] == "compact":
        return lens, None
    beams = case["beams"]
    if case["first"]:
        return lens, [i // beams for i in range(len(lens) * beams)]
    # of a request's beams some go on more than once and others end; now and then a request ends
    parents = [-1 if r.random() < 0.02 and i else i * beams + r.randrange(beams) for i in range(len(lens)) for _ in range(beams)]
    return [n for n in lens for _ in range(beams)], parents


def _tables(case, seed):
    """Rows of page indexes, and the pages that others hold. Of a request's beams
    all share its pages but each one's last."""
    lens, parents = _rows_of(case)
    width = max(-(-(n + 1) // B) for n in lens)
    order = np.random.default_rng(seed).permutation(case["pool"])
    held, order = order[: case["pool"] // 50], list(order[case["pool"] // 50:])
    rows = np.full((len(lens), width), -1, np.int64)
    beams = 1 if case["kind"] == "compact" or case["first"] else case["beams"]
    for i, n in enumerate(lens):
        full = n // B
        if i % beams:
            rows[i, :full] = rows[i - 1, :full]
        else:
            rows[i, :full] = [order.pop() for _ in range(full)]
        if n % B:
            rows[i, full] = order.pop()
    return lens, parents, rows, held


def _prepare_pool(case, seed):
    lens, parents, rows, held = _tables(case, seed)
    gen = _gen(seed)
    pool = torch.randn((case["pool"], case["page"] // 2), generator=gen, device="cuda", dtype=torch.bfloat16).view(torch.int32)
    reserved = np.zeros(case["pool"], np.int32)
    reserved[held] = 1
    s = dict(pool=pool, tables=_int(np.where(rows >= 0, rows * case["stride"], -1)), lens=_int(lens), reserved=_int(reserved))
    n = len(parents) if parents else len(lens)
    if parents:
        s["parents"] = _int(parents)
        s["new_lens"] = _int([1] * n)
        s["lens_out"] = _int([0] * n)
    s["tables_out"] = torch.zeros((n, rows.shape[1]), dtype=torch.int32, device="cuda")
    s["counts"] = _int([0, 0])
    s["moved_to"] = _int([0] * case["pool"])
    s["workspace"] = torch.empty(8 * (case["pool"] + 4 * n) + 65536, dtype=torch.uint8, device="cuda")
    return s


def prepare(case, seed):
    s = {"rows": _prepare_rows, "pages": _prepare_pages, "fork": _prepare_pool, "compact": _prepare_pool}[case["kind"]](case, seed)
    s["case"] = case
    return s


# ------------------------------------------------------------------ plain forms
def _padded(starts, most, last):
    """Rows of all requests as if they were the longest, and which of them there are."""
    i = torch.arange(most, device="cuda")
    return (starts[:-1, None] + i).clamp(max=last), i < starts.diff()[:, None]


def _attend(s, k, v, lens):
    """Attention in FP32 of the packed queries over k, v [batch][heads][tokens][dim]."""
    case = s["case"]
    heads, dim, group = case["heads"], case["dim"], case["group"]
    n_q = len(s["out"])
    at, there = _padded(s["q_starts"], s["most_new"], n_q - 1)
    q = s["q"].reshape(n_q, heads, group, dim)[at].float().permute(0, 2, 3, 1, 4).reshape(len(at), heads, -1, dim)   # [batch][heads][group * new][dim]
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).view(len(at), heads, group, s["most_new"], -1)
    sees = lens - s["q_starts"].diff() + 1                      # of query 0
    j = torch.arange(k.shape[2], device="cuda")
    seen = j < (sees[:, None] + torch.arange(s["most_new"], device="cuda"))[:, :, None]
    scores = torch.where(seen[:, None, None], scores, -math.inf).mul_(1 / math.sqrt(dim))
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).view(len(at), heads, group, s["most_new"], dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(len(at), s["most_new"], heads * group, dim)
    s["out"][at[there]] = o[there].to(torch.bfloat16)


def _plain_rows(s):
    heads, dim = s["case"]["heads"], s["case"]["dim"]
    n_k = len(s["k"])
    at, there = _padded(s["k_starts"], s["longest"], n_k - 1)
    k, v = (s[x].reshape(n_k, heads, dim)[at].float().transpose(1, 2).contiguous() for x in ("k", "v"))
    _attend(s, k, v, s["k_starts"].diff())


def _values(codes, scale):
    """The FP32 values that E2M1 codes [..., n/2] and scales, one of each two codes, stand for."""
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    lut = torch.cat([lut, -lut])
    v = lut[torch.stack([codes & 15, codes >> 4], -1).int()]
    return torch.ldexp(v, scale.int()[..., None] - 127).flatten(-2)


def _plain_pages(s):
    case = s["case"]
    heads, dim, kind = case["heads"], case["dim"], case["pages"]
    ids = s["tables"].clamp(min=0)
    out = []
    for pool in ("k", "v"):
        pages = s[pool][ids] if kind != "fp8" else s[pool].view(torch.uint8)[ids].view(torch.float8_e4m3fn)
        if kind == "bf16":
            x = pages.float().permute(0, 3, 1, 2, 4)                                      # [batch][heads][block][token][dim]
        elif kind == "fp8":
            x = (pages.float() * s[pool + "_scales"][ids][..., None]).permute(0, 3, 1, 2, 4)
        else:
            scale = s[pool + "_scales"][ids].repeat_interleave(G // 2, 3).transpose(3, 4)  # [batch][block][heads][token][dim/2]
            if pool == "k":
                codes = pages.transpose(3, 4).flatten(-2)                                 # quarters side by side
            else:
                codes = pages.transpose(4, 5).flatten(-2).flatten(3, 4)                   # columns side by side, quads one after another
            x = _values(codes, scale).transpose(1, 2)
        out.append(x.flatten(2, 3).contiguous())
    _attend(s, out[0], out[1], s["lens"])


def _plain_fork(s):
    case = s["case"]
    stride, n_pages, width = case["stride"], case["pool"], s["tables"].shape[1]
    live, p = s["parents"] >= 0, s["parents"].clamp(min=0).long()
    n = len(p)
    lens = torch.where(live, s["lens"][p], 0)
    kept = (lens + B - 1).div(B, rounding_mode="floor")
    want = (lens + s["new_lens"] + B - 1).div(B, rounding_mode="floor")
    i = torch.arange(n, device="cuda")
    first = torch.full((len(s["lens"]),), n, device="cuda").scatter_reduce(0, p, torch.where(live, i, n), "amin")
    copied = live & (lens % B > 0) & (first[p] < i)
    rows = s["tables"][p]
    j = torch.arange(width, device="cuda")
    used = s["reserved"] > 0
    used[rows[live[:, None] & (j < kept[:, None])].long() // stride] = True
    free = torch.nonzero(~used)[:, 0]
    need = torch.where(live, want - kept + copied.int(), 0)
    ends = need.cumsum(0)
    ok = live & ((need == 0) | (ends <= len(free)))
    own_from = (kept - copied.int())[:, None]
    fresh = free[((ends - need)[:, None] + j - own_from).clamp(0, max(0, len(free) - 1))] * stride
    out = torch.where(j < own_from, rows, torch.where(j < want[:, None], fresh.int(), -1))
    s["tables_out"].copy_(torch.where(ok[:, None], out, -1))
    s["lens_out"].copy_(torch.where(ok, lens, torch.where(live, -1, 0)))
    s["counts"].copy_(torch.stack([need.sum(), torch.full_like(need.sum(), len(free))]))
    c = copied & ok
    src = rows.gather(1, (kept - 1).clamp(min=0)[:, None].long())[c, 0].long() // stride
    dst = s["tables_out"].gather(1, (kept - 1).clamp(min=0)[:, None].long())[c, 0].long() // stride
    s["pool"][dst] = s["pool"][src]


def _plain_compact(s):
    stride, n_pages = s["case"]["stride"], s["case"]["pool"]
    t = s["tables"]
    held = s["reserved"] > 0
    used = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
    used[t[t >= 0].long() // stride] = True
    moves = used & ~held
    place = (~held).cumsum(0)                                     # of the pages that may be taken, from 1
    front = ~held & (place <= moves.sum())
    src, dst = torch.nonzero(moves & ~front)[:, 0], torch.nonzero(front & ~moves)[:, 0]
    s["moved_to"].copy_(torch.where(used, torch.arange(n_pages, device="cuda"), -1))
    s["moved_to"][src] = dst.int()
    s["tables_out"].copy_(torch.where(t >= 0, s["moved_to"][(t.clamp(min=0) // stride).long()] * stride, -1))
    s["counts"].copy_(torch.stack([moves.sum(), torch.full_like(moves.sum(), len(src))]))
    s["pool"][dst] = s["pool"][src]


# ------------------------------------------------------------------ the calls
def _package():
    if "pbe_handoff" in sys.modules:  # imported once, not looked for in every pass
        return sys.modules["pbe_handoff"]
    path = str(Path(__file__).resolve().parent.parent / "paged-batch-engine_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pbe_handoff
    return pbe_handoff


def _own_rows(s):
    P, case = _package(), s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    P.prompt_attention(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), len(q), len(k), s["q_starts"].data_ptr(),
                       s["k_starts"].data_ptr(), case["batch"], case["heads"] * case["group"], case["heads"], case["dim"], s["out"].data_ptr(),
                       s["workspace"].data_ptr(), s["workspace"].numel(), stream=torch.cuda.current_stream().cuda_stream)


def _own_pages(s):
    P, case = _package(), s["case"]
    kind = {"bf16": P.PBE_KV_BF16, "fp8": P.PBE_KV_FP8_E4M3, "mxfp4": P.PBE_KV_MXFP4}[case["pages"]]
    k, v, scales = s["k"], s["v"], [0, 0, 0]
    if "k_scales" in s:
        scales = [s["k_scales"].data_ptr(), s["v_scales"].data_ptr(), s["k_scales"].numel() * s["k_scales"].element_size()]
    P.paged_prompt_attention(k.data_ptr(), v.data_ptr(), k.numel() * k.element_size(), *scales, kind, case["heads"], case["dim"], s["q"].data_ptr(),
                             s["out"].data_ptr(), len(s["q"]), s["q_starts"].data_ptr(), case["batch"], case["heads"] * case["group"],
                             s["tables"].data_ptr(), s["lens"].data_ptr(), s["tables"].shape[1], s["workspace"].data_ptr(), s["workspace"].numel(),
                             stream=torch.cuda.current_stream().cuda_stream)


def _planes(s):
    """What a program keeps of its arena: made once."""
    if "planes" not in s:
        P = _package()
        s["planes"] = P.page_planes([(P.view_of(s["pool"].data_ptr(), s["pool"].numel() * 4), s["case"]["page"])])
    return s["planes"]


def _own_fork(s):
    P, case = _package(), s["case"]
    P.fork_pages(_planes(s), case["pool"], case["stride"], B, s["tables"].data_ptr(), s["lens"].data_ptr(), len(s["lens"]), s["parents"].data_ptr(),
                 s["new_lens"].data_ptr(), len(s["parents"]), s["tables"].shape[1], s["reserved"].data_ptr(), s["tables_out"].data_ptr(),
                 s["lens_out"].data_ptr(), s["counts"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(),
                 stream=torch.cuda.current_stream().cuda_stream)


def _own_compact(s):
    P, case = _package(), s["case"]
    P.compact_pages(_planes(s), case["pool"], case["stride"], s["tables"].data_ptr(), len(s["tables"]), s["tables"].shape[1], s["reserved"].data_ptr(),
                    s["tables_out"].data_ptr(), s["moved_to"].data_ptr(), s["counts"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(),
                    stream=torch.cuda.current_stream().cuda_stream)


def run(state):
    s, kind = state, state["case"]["kind"]
    if kind == "rows":
        _own_rows(s) if own else _plain_rows(s)
    elif kind == "pages":
        _own_pages(s) if own else _plain_pages(s)
    elif kind == "fork":
        _own_fork(s) if own else _plain_fork(s)
        return {k: s[k] for k in ("pool", "tables_out", "lens_out", "counts")}
    else:
        _own_compact(s) if own else _plain_compact(s)
        return {k: s[k] for k in ("pool", "tables_out", "moved_to", "counts")}
    return {"out": s["out"]}


def work(case):
    if case["kind"] in ("fork", "compact"):
        lens, parents, rows, held = _tables(case, 0)
        if parents:
            moved = sum(p >= 0 and lens[p] % B > 0 and p in parents[:i] for i, p in enumerate(parents))
            ints = sum(-(-n // B) for n in lens) + rows.shape[1] * len(parents) + 4 * len(parents) + case["pool"]
        else:
            used = np.zeros(case["pool"], bool)
            used[rows[rows >= 0]] = True
            taken = np.ones(case["pool"], bool)
            taken[held] = False
            front = taken & (np.cumsum(taken) <= used.sum())
            moved = int((used & ~front).sum())
            ints = 2 * rows.size + 2 * case["pool"]
        return {"bytes": 2 * moved * case["page"] + 4 * ints, "flops": 0}
    heads, dim, q_heads = case["heads"], case["dim"], case["heads"] * case["group"]
    reqs = _requests(case)
    seen = sum(new * (n - new) + new * (new + 1) // 2 for n, new in reqs)
    row = {"bf16": 2 * dim, "fp8": dim + 4, "mxfp4": dim // 2 + dim // G}[case.get("pages", "bf16")]
    ints = 2 * len(reqs) + sum(-(-n // B) for n, _ in reqs) if case["kind"] == "pages" else 2 * len(reqs)
    return {"bytes": sum(n for n, _ in reqs) * 2 * heads * row + sum(new for _, new in reqs) * q_heads * dim * 4 + 4 * ints, "flops": 4 * seen * q_heads * dim}


# ------------------------------------------------------------------ in 64 bits
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _decoded(s, pool, block, at):
    """Rows [tokens][heads][dim] of the given blocks and tokens in 64 bits, byte
    by byte of the MXFP4 layout."""
    heads, dim = s["case"]["heads"], s["case"]["dim"]
    codes, scales = s[pool].reshape(-1), s[pool + "_scales"].reshape(-1)
    d, h = torch.arange(dim, device="cuda"), torch.arange(heads, device="cuda")[:, None]
    if pool == "v":
        byte = (at // 4)[:, None, None] * (2 * dim) + (d // (dim // 16)) * (dim // 8) + (at % 4)[:, None, None] * (dim // 32) + d % (dim // 16) // 2
    else:
        byte = (d // (dim // 4)) * (2 * dim) + at[:, None, None] * (dim // 8) + d % (dim // 4) // 2
    raw = codes[(block[:, None, None] * heads + h) * (8 * dim) + byte]
    code = torch.where(d % 2 == 1, raw >> 4, raw & 15).long()
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device="cuda")
    exponent = scales[(block[:, None, None] * heads + h) * (dim // 2) + (d // G) * B + at[:, None, None]]
    return table[code] * 2.0 ** (exponent.double() - 127)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "compact"):
        return None  # whole numbers
    s = (_prepare_rows if kind == "rows" else _prepare_pages)(case, seed)
    s["case"] = case
    heads, dim, group = case["heads"], case["dim"], case["group"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    begin, k_begin = 0, 0
    for b, (n, new) in enumerate(_requests(case, seed)):
        t = torch.arange(n, device="cuda")
        if kind == "rows":
            k, v = (s[x][k_begin:k_begin + n].double().reshape(n, heads, dim) for x in ("k", "v"))
        else:
            block, at = s["tables"][b].long()[t // B], t % B
            if case["pages"] == "mxfp4":
                k, v = (_decoded(s, x, block, at) for x in ("k", "v"))
            elif case["pages"] == "fp8":
                k, v = (s[x].view(torch.uint8)[block, at].view(torch.float8_e4m3fn).double() * s[x + "_scales"][block, at].double()[..., None] for x in ("k", "v"))
            else:
                k, v = (s[x][block, at].double() for x in ("k", "v"))
        k_begin += n
        q = s["q"][begin:begin + new].double().reshape(new, heads, group, dim)
        for h in range(heads):
            keys, values = k[:, h].t().contiguous(), v[:, h].contiguous()
            for g in range(group):
                score = torch.mm(q[:, h, g].contiguous(), keys) / math.sqrt(dim)
                score.masked_fill_(t[None] > (n - new + torch.arange(new, device="cuda"))[:, None], -math.inf)
                out[begin:begin + new, h * group + g] = torch.mm(torch.softmax(score, -1), values)
        begin += new
    return {"out": out}
