// C ABI: attention of prompts (many query tokens a sequence) over rows and over
// pages of keys and values.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "capi_internal.h"
#include "../kernels/prompt_kernels.h"

using namespace pbe_capi;

namespace {

constexpr uint64_t kTokens = 16;
constexpr int32_t kMostTokens = INT32_MAX - 255;  // so that a tile's end fits 31 bits, and 64 sequences behind the last

struct Call {
  const void* queries;
  void* outputs;
  int32_t n_rows;
  const int32_t* starts;
  int32_t batch, q_heads, kv_heads, head_dim;
  void* workspace;
  uint64_t workspace_bytes;
};

// What both forms check first: sizes, heads, alignment.
int check(const Call& c, int device) {
  if (c.n_rows < 0 || c.batch <= 0 || c.q_heads <= 0 || c.kv_heads <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "query rows >= 0, batch, q_heads, kv_heads > 0 and a device");
  if (c.batch > kMostTokens) return fail(PBE_ERR_INVALID, "batch must be at most %d", (int)kMostTokens);
  if (c.head_dim != 64 && c.head_dim != 128) return fail(PBE_ERR_UNSUPPORTED, "heads of 64 or 128 dims");
  if (c.q_heads % c.kv_heads) return fail(PBE_ERR_UNSUPPORTED, "q_heads must be a multiple of kv_heads");
  if ((int64_t)c.n_rows * c.q_heads > kMostTokens) return fail(PBE_ERR_INVALID, "rows * q_heads must be at most %d", (int)kMostTokens);
  if ((uint64_t)c.q_heads * c.head_dim * 2 > 0xffffffffull) return fail(PBE_ERR_INVALID, "a token's heads must be smaller than 4 GiB");
  if (c.n_rows == 0) return PBE_OK;
  if (!c.queries || !c.outputs || !c.starts) return fail(PBE_ERR_INVALID, "null prompt operand");
  auto at = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
  if ((at(c.queries) | at(c.outputs) | at(c.workspace)) % 16 || at(c.starts) % 4)
    return fail(PBE_ERR_INVALID, "queries, outputs and workspace must be 16-byte aligned, starts 4-byte aligned");
  return PBE_OK;
}

// Tiles, parts and workspace; *need: the bytes of it that the launch uses.
int plan(const Call& c, pbe::KeyKind kind, int64_t most_keys, int device, pbe::PromptParams* p, pbe::PromptPlan* plan, uint64_t* need) {
  p->group = c.q_heads / c.kv_heads;
  *plan = pbe::plan_prompt(c.n_rows, c.batch, p->group, c.kv_heads, kind, most_keys, compute_units(device), c.workspace ? c.workspace_bytes : 0, c.head_dim);
  // fewer than 2^32 threads in a launch: eight workgroups more than are needed, the join's of 1,024
  if ((std::max<int64_t>(plan->tiles, plan->parts) + 8) * c.kv_heads >= 0xffffffffll / (plan->parts ? 1024 : 2 * plan->rows))
    return fail(PBE_ERR_INVALID, "too many rows and heads for one launch");
  *need = (uint64_t)plan->parts * plan->each;
  p->part_acc = static_cast<float*>(c.workspace);
  p->part_ml = p->part_acc + 2ull * (uint64_t)plan->parts * (uint64_t)c.kv_heads * (uint64_t)plan->rows * (uint64_t)c.head_dim;
  p->q = static_cast<const uint8_t*>(c.queries);
  p->out = static_cast<uint8_t*>(c.outputs);
  p->q_starts = c.starts;
  p->n_q = c.n_rows;
  p->batch = c.batch;
  p->kv_heads = c.kv_heads;
  p->by_group = pbe::make_fast_div((uint32_t)p->group);
  p->scale = (1.f / std::sqrt((float)c.head_dim)) * 1.4426950408889634f;
  return PBE_OK;
}

}  // namespace

extern "C" {

uint64_t pbe_prompt_workspace_bytes(int32_t n_rows, int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (n_rows <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || q_heads % kv_heads) return 0;
  uint64_t most = 0;  // over the kinds of keys and values
  for (const pbe::KeyKind kind : {pbe::KeyKind::kRows, pbe::KeyKind::kBf16, pbe::KeyKind::kFp8, pbe::KeyKind::kMxfp4}) {
    for (const int64_t keys : {(int64_t)INT32_MAX, (int64_t)512 * batch - 1}) {  // over sequences, long and short
      const pbe::PromptPlan r = pbe::plan_prompt(n_rows, batch, q_heads / kv_heads, kv_heads, kind, keys, compute_units(), ~0ull, head_dim);
      most = std::max(most, (uint64_t)r.parts * r.each);
    }
  }
  return most;
}

int pbe_prompt_attention(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                         const void* v, int64_t v_stride, int32_t n_queries, int32_t n_keys,
                         const int32_t* q_starts, const int32_t* k_starts, int32_t batch,
                         int32_t q_heads, int32_t kv_heads, int32_t head_dim, void* outputs,
                         void* workspace, uint64_t workspace_bytes, int device, void* stream) {
  const Call c{q, outputs, n_queries, q_starts, batch, q_heads, kv_heads, head_dim, workspace, workspace_bytes};
  if (n_keys < 0 || n_keys > kMostTokens) return fail(PBE_ERR_INVALID, "n_keys must be 0..%d", (int)kMostTokens);
  int rc = check(c, device);
  if (rc != PBE_OK || n_queries == 0) return rc;
  if (!k_starts && n_keys != n_queries) return fail(PBE_ERR_INVALID, "without k_starts there are as many keys as queries");
  if (!k_starts) k_starts = q_starts;
  if (n_keys && (!k || !v)) return fail(PBE_ERR_INVALID, "null prompt operand");
  auto at = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
  if ((at(k) | at(v)) % 16 || at(k_starts) % 4) return fail(PBE_ERR_INVALID, "rows must be 16-byte aligned, starts 4-byte aligned");
  const int64_t dim = head_dim, widest = INT64_MAX / 8 / std::max(1, std::max(n_queries, n_keys));
  const struct {
    int64_t stride, row, count;
  } parts[] = {{q_stride, q_heads * dim, n_queries}, {k_stride, kv_heads * dim, n_keys}, {v_stride, kv_heads * dim, n_keys}};
  uint64_t spans[3];
  for (int i = 0; i < 3; ++i) {
    const auto& r = parts[i];
    if ((r.count > 1 && r.stride < r.row) || r.stride < 0 || r.stride > widest || r.stride % 8)
      return fail(PBE_ERR_INVALID, "row strides must hold a row and be whole multiples of 16 bytes");
    spans[i] = r.count ? (uint64_t)((r.count - 1) * r.stride + r.row) * 2 : 0;
  }
  pbe::PromptParams p{};
  pbe::PromptPlan laid;
  uint64_t need = 0;
  rc = plan(c, pbe::KeyKind::kRows, n_keys, device, &p, &laid, &need);
  if (rc != PBE_OK) return rc;
  const uint64_t out_bytes = (uint64_t)n_queries * (uint64_t)q_heads * (uint64_t)dim * 2, starts = ((uint64_t)batch + 1) * 4;
  const Span out{outputs, out_bytes}, partials{workspace, need}, queries{q, spans[0]};
  const bool in_place = q == outputs && (q_stride == q_heads * dim || n_queries == 1);
  if (any_meet({out, partials}, {{k, spans[1]}, {v, spans[2]}, {q_starts, starts}, {k_starts, starts}}) || meet(out, partials) ||
      meet(queries, partials) || (!in_place && meet(queries, out)))
    return fail(PBE_ERR_INVALID, "prompt outputs and workspace must lie apart from each other and from what is read");
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    auto ok = [&](const void* ptr, uint64_t bytes) { return bytes == 0 || accessible(ptr, bytes, device, &known); };
    if (!ok(q, spans[0]) || !ok(k, spans[1]) || !ok(v, spans[2]) || !ok(q_starts, starts) || !ok(k_starts, starts) || !ok(outputs, out_bytes) ||
        !ok(workspace, need))
      return fail(PBE_ERR_INVALID, "prompt operands must be memory of device %d", device);
  }
  p.k = static_cast<const uint8_t*>(k);
  p.v = static_cast<const uint8_t*>(v);
  p.q_stride = (uint64_t)q_stride * 2;
  p.k_stride = (uint64_t)k_stride * 2;
  p.v_stride = (uint64_t)v_stride * 2;
  p.lens = k_starts;
  p.n_k = n_keys;
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_prompt_attention(p, laid, head_dim, pbe::KeyKind::kRows, static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

int pbe_paged_prompt_attention(const void* key_pool, const void* value_pool, uint64_t pool_bytes,
                               const void* key_scales, const void* value_scales,
                               uint64_t scale_pool_bytes, int32_t kv_dtype, int32_t kv_heads,
                               int32_t head_dim, const void* queries, void* outputs,
                               int32_t n_rows, const int32_t* token_starts, int32_t batch,
                               int32_t q_heads, const int32_t* block_tables,
                               const int32_t* seq_lens, int32_t max_blocks_per_seq,
                               void* workspace, uint64_t workspace_bytes, int device,
                               void* stream) {
  const Call c{queries, outputs, n_rows, token_starts, batch, q_heads, kv_heads, head_dim, workspace, workspace_bytes};
  if (kv_dtype != PBE_KV_BF16 && kv_dtype != PBE_KV_FP8_E4M3 && kv_dtype != PBE_KV_MXFP4)
    return fail(PBE_ERR_INVALID, "unknown KV dtype %d", (int)kv_dtype);
  if (max_blocks_per_seq <= 0) return fail(PBE_ERR_INVALID, "max_blocks_per_seq > 0");
  int rc = check(c, device);
  if (rc != PBE_OK || n_rows == 0) return rc;
  const bool fp8 = kv_dtype == PBE_KV_FP8_E4M3, mx = kv_dtype == PBE_KV_MXFP4, scaled = fp8 || mx;
  if (!key_pool || !value_pool || !block_tables || !seq_lens || (scaled && (!key_scales || !value_scales)))
    return fail(PBE_ERR_INVALID, "null prompt operand");
  auto at = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
  if ((at(key_pool) | at(value_pool)) % 16 || (at(block_tables) | at(seq_lens)) % 4 || (scaled && (at(key_scales) | at(value_scales)) % 4))
    return fail(PBE_ERR_INVALID, "pools must be 16-byte aligned, scale pools, tables and lengths 4-byte aligned");
  if ((int64_t)batch * max_blocks_per_seq > (1ll << 40)) return fail(PBE_ERR_INVALID, "batch * max_blocks_per_seq must be at most 2^40");
  const uint64_t values = kTokens * (uint64_t)kv_heads * (uint64_t)head_dim;  // of a block, K or V
  const uint64_t half = mx ? values / 2 : fp8 ? values : 2 * values;
  const uint64_t block_scales = mx ? half / 16 : fp8 ? kTokens * (uint64_t)kv_heads * 4 : 0;
  if (half > 0xffffffffull) return fail(PBE_ERR_INVALID, "a block of one plane must be smaller than 4 GiB");
  if (pool_bytes < half || (scaled && scale_pool_bytes < block_scales))
    return fail(PBE_ERR_INVALID, "pools and scale pools must hold at least one block");
  pbe::PromptParams p{};
  pbe::PromptPlan laid;
  uint64_t need = 0;
  const pbe::KeyKind kind = mx ? pbe::KeyKind::kMxfp4 : fp8 ? pbe::KeyKind::kFp8 : pbe::KeyKind::kBf16;
  rc = plan(c, kind, (int64_t)max_blocks_per_seq * (int64_t)kTokens, device, &p, &laid, &need);
  if (rc != PBE_OK) return rc;
  const uint64_t row_bytes = (uint64_t)n_rows * (uint64_t)q_heads * (uint64_t)head_dim * 2;
  const uint64_t starts = ((uint64_t)batch + 1) * 4, lens = (uint64_t)batch * 4, tables = (uint64_t)batch * (uint64_t)max_blocks_per_seq * 4;
  const uint64_t scale_bytes = scaled ? scale_pool_bytes : 0;
  const Span q{queries, row_bytes}, out{outputs, row_bytes}, partials{workspace, need};
  if (any_meet({out, partials}, {{key_pool, pool_bytes}, {value_pool, pool_bytes}, {key_scales, scale_bytes}, {value_scales, scale_bytes},
                                 {token_starts, starts}, {seq_lens, lens}, {block_tables, tables}}) ||
      meet(out, partials) || meet(q, partials) || (queries != outputs && meet(q, out)))
    return fail(PBE_ERR_INVALID, "prompt outputs and workspace must lie apart from each other and from what is read");
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    auto ok = [&](const void* ptr, uint64_t bytes) { return bytes == 0 || accessible(ptr, bytes, device, &known); };
    if (!ok(key_pool, pool_bytes) || !ok(value_pool, pool_bytes) || !ok(key_scales, scale_bytes) || !ok(value_scales, scale_bytes) ||
        !ok(queries, row_bytes) || !ok(outputs, row_bytes) || !ok(token_starts, starts) || !ok(seq_lens, lens) || !ok(block_tables, tables) ||
        !ok(workspace, need))
      return fail(PBE_ERR_INVALID, "prompt operands must be memory of device %d", device);
  }
  p.k = static_cast<const uint8_t*>(key_pool);
  p.v = static_cast<const uint8_t*>(value_pool);
  p.k_scales = static_cast<const uint8_t*>(key_scales);
  p.v_scales = static_cast<const uint8_t*>(value_scales);
  p.q_stride = (uint64_t)q_heads * (uint64_t)head_dim * 2;
  p.k_stride = p.v_stride = half / kTokens;
  p.half = half;
  p.lens = seq_lens;
  p.tables = block_tables;
  p.max_blocks = max_blocks_per_seq;
  uint64_t blocks = pool_bytes / half;
  if (scaled) blocks = std::min(blocks, scale_pool_bytes / block_scales);
  p.blocks = (int32_t)std::min<uint64_t>(blocks, INT32_MAX);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_prompt_attention(p, laid, head_dim, kind, static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

}  // extern "C"
