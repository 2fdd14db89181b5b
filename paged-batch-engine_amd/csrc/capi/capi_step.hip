// C ABI: what a decode worker makes ready for a step (its tables) and for each
// layer's attention (normed and rotated heads, in the reader's form and in pages).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <utility>
#include <vector>

#include "capi_internal.h"
#include "../kernels/rope_kernels.h"
#include "../kernels/step_kernels.h"

using namespace pbe_capi;

extern "C" {

int pbe_build_step_tables(const int32_t* page_ids, int64_t n_page_ids, const int32_t* page_starts,
                          const int32_t* cached_lens, const int32_t* new_lens, int32_t batch,
                          int32_t block_size, int32_t* block_tables, int32_t max_blocks_per_seq,
                          int32_t* seq_lens, int32_t* token_starts, int32_t* slot_mapping,
                          int32_t* positions, int32_t max_tokens, int device, void* stream) {
  if (batch <= 0 || block_size <= 0 || max_blocks_per_seq <= 0 || max_tokens <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "batch, block_size, max_blocks_per_seq, max_tokens > 0 and a device");
  if (n_page_ids < 0 || n_page_ids > INT32_MAX) return fail(PBE_ERR_INVALID, "n_page_ids must be 0..INT32_MAX");
  if ((int64_t)batch * max_blocks_per_seq > INT32_MAX)
    return fail(PBE_ERR_INVALID, "batch * max_blocks_per_seq must be at most INT32_MAX");
  if ((n_page_ids && !page_ids) || !page_starts || !cached_lens || !block_tables || !seq_lens || !token_starts || !slot_mapping || !positions)
    return fail(PBE_ERR_INVALID, "null step table operand");
  const struct {
    const int32_t* at;
    uint64_t count;
    bool out;
  } arrays[] = {{page_ids, (uint64_t)n_page_ids, false},
                {page_starts, (uint64_t)batch + 1, false},
                {cached_lens, (uint64_t)batch, false},
                {new_lens, new_lens ? (uint64_t)batch : 0, false},
                {block_tables, (uint64_t)batch * (uint64_t)max_blocks_per_seq, true},
                {seq_lens, (uint64_t)batch, true},
                {token_starts, (uint64_t)batch + 1, true},
                {slot_mapping, (uint64_t)max_tokens, true},
                {positions, (uint64_t)max_tokens, true}};
  for (const auto& a : arrays) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(a.at);
    if (begin % 4) return fail(PBE_ERR_INVALID, "step table arrays must be 4-byte aligned");
    // Workgroups read lengths and lists while others write: an output in the
    // place of an input (seq_lens over cached_lens) would race with them.
    for (const auto& o : arrays) {
      const uintptr_t o_begin = reinterpret_cast<uintptr_t>(o.at);
      if (&a != &o && o.out && begin < o_begin + 4 * o.count && o_begin < begin + 4 * a.count)
        return fail(PBE_ERR_INVALID, "a step table output overlaps another array");
    }
  }
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    for (const auto& a : arrays)
      if (a.count && !accessible(a.at, 4 * a.count, device, &known))
        return fail(PBE_ERR_INVALID, "step table operands must be memory of device %d", device);
  }
  pbe::StepTablesParams p{};
  p.page_ids = page_ids;
  p.page_starts = page_starts;
  p.cached_lens = cached_lens;
  p.new_lens = new_lens;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.token_starts = token_starts;
  p.slots = slot_mapping;
  p.positions = positions;
  p.n_page_ids = (uint32_t)n_page_ids;
  p.batch = (uint32_t)batch;
  p.max_blocks = (uint32_t)max_blocks_per_seq;
  p.max_tokens = (uint32_t)max_tokens;
  p.block_size = (uint32_t)block_size;
  p.by_block_size = pbe::make_fast_div((uint32_t)block_size);
  p.by_max_blocks = pbe::make_fast_div((uint32_t)max_blocks_per_seq);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_step_tables(p, static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

int pbe_qk_norm_rope_scatter(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                             const void* v, int64_t v_stride, int32_t in_dtype, int32_t n_tokens,
                             int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                             const void* q_weight, const void* k_weight, float eps,
                             const int32_t* positions, const float* cos_sin, int32_t max_position,
                             int32_t rotary_dim, int32_t rope_style, const int32_t* slot_mapping,
                             int32_t block_size, int32_t kv_dtype, void* q_out, void* key_pool,
                             uint64_t key_pool_bytes, void* value_pool, uint64_t value_pool_bytes,
                             void* key_scales, uint64_t key_scale_bytes, void* value_scales,
                             uint64_t value_scale_bytes, int device, void* stream) {
  if (in_dtype != PBE_IN_BF16 && in_dtype != PBE_IN_F32) return fail(PBE_ERR_INVALID, "unknown input dtype %d", (int)in_dtype);
  if (kv_dtype != PBE_KV_BF16 && kv_dtype != PBE_KV_FP8_E4M3 && kv_dtype != PBE_KV_MXFP4)
    return fail(PBE_ERR_INVALID, "unknown KV dtype %d", (int)kv_dtype);
  if (rope_style != PBE_ROPE_HALVES && rope_style != PBE_ROPE_PAIRS) return fail(PBE_ERR_INVALID, "unknown rope style %d", (int)rope_style);
  if (n_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || block_size <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "n_tokens >= 0, q_heads, kv_heads, block_size > 0 and a device");
  if (head_dim != 64 && head_dim != 128) return fail(PBE_ERR_UNSUPPORTED, "heads of 64 or 128 dims");
  if (kv_dtype == PBE_KV_MXFP4 && block_size != 16) return fail(PBE_ERR_UNSUPPORTED, "MXFP4 pages hold 16 tokens");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16)
    return fail(PBE_ERR_INVALID, "rotary_dim must be a multiple of 16 up to head_dim");
  if (rotary_dim && max_position <= 0) return fail(PBE_ERR_INVALID, "a rotation needs max_position > 0");
  if (!(eps >= 0.f) || std::isinf(eps)) return fail(PBE_ERR_INVALID, "eps must be finite and not negative");
  // The root of a mean below FP32's normal numbers, which v_rsq_f32 takes for 0.
  if ((q_weight || k_weight) && eps < std::numeric_limits<float>::min()) return fail(PBE_ERR_INVALID, "a norm needs eps of at least 2^-126");
  if (n_tokens == 0) return PBE_OK;
  const bool f32 = in_dtype == PBE_IN_F32, fp8 = kv_dtype == PBE_KV_FP8_E4M3, mx = kv_dtype == PBE_KV_MXFP4;
  const int64_t elem = f32 ? 4 : 2, dim = head_dim;
  // A token's heads fit one launch's 2^31 lanes, so the products below fit 64 bits.
  if (((int64_t)q_heads + 2 * (int64_t)kv_heads) * (dim / 8) >= (1ll << 31) / n_tokens)
    return fail(PBE_ERR_INVALID, "too many tokens for one launch");
  if (std::max(q_heads, kv_heads) * dim * elem > 0xffffffffll) return fail(PBE_ERR_INVALID, "a token's heads must be smaller than 4 GiB");
  if (!q || !k || !v || !slot_mapping || !q_out || !key_pool || !value_pool || (rotary_dim && (!positions || !cos_sin)))
    return fail(PBE_ERR_INVALID, "null operand");
  if ((fp8 || mx) && (!key_scales || !value_scales)) return fail(PBE_ERR_INVALID, "FP8 and MXFP4 pools need K and V scale pools");
  const int64_t widest = INT64_MAX / 4 / elem / n_tokens;  // a stride whose rows 64 bits address
  for (const auto& row : {std::pair<int64_t, int64_t>(q_stride, q_heads * dim), {k_stride, kv_heads * dim}, {v_stride, kv_heads * dim}})
    if ((n_tokens > 1 && row.first < row.second) || row.first < 0 || row.first > widest || row.first * elem % 16)
      return fail(PBE_ERR_INVALID, "row strides must hold a row and be whole multiples of 16 bytes");
  auto at = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
  if ((at(q) | at(k) | at(v) | at(q_weight) | at(k_weight) | at(cos_sin) | at(q_out)) % 16 || (at(positions) | at(slot_mapping)) % 4)
    return fail(PBE_ERR_INVALID, "rows, weights, cos_sin and q_out must be 16-byte aligned");
  if ((at(key_pool) | at(value_pool)) % (mx ? 4 : fp8 ? 8 : 16) || ((fp8 || mx) && (at(key_scales) | at(value_scales)) % 4))
    return fail(PBE_ERR_INVALID, "pools must be aligned to their stores and scale pools to 4 bytes");
  auto span = [&](int64_t stride, int64_t heads) { return (uint64_t)(((int64_t)n_tokens - 1) * stride + heads * dim) * (uint64_t)elem; };
  const uint64_t q_span = span(q_stride, q_heads), k_span = span(k_stride, kv_heads), v_span = span(v_stride, kv_heads);
  const uint64_t out_bytes = (uint64_t)n_tokens * (uint64_t)q_heads * (uint64_t)dim * 2;
  const uint64_t weight = (uint64_t)(dim * elem), table = rotary_dim ? (uint64_t)max_position * (uint64_t)rotary_dim * 4 : 0;
  const uint64_t ints = (uint64_t)n_tokens * 4;
  const std::initializer_list<Span> inputs = {{q, q_span}, {k, k_span}, {v, v_span}, {q_weight, weight}, {k_weight, weight}, {cos_sin, table},
                                              {positions, ints}, {slot_mapping, ints}};
  const bool scaled = fp8 || mx;
  const std::initializer_list<Span> pools = {{key_pool, key_pool_bytes}, {value_pool, value_pool_bytes},
                                             {key_scales, scaled ? key_scale_bytes : 0}, {value_scales, scaled ? value_scale_bytes : 0}};
  if (any_meet({{q_out, out_bytes}}, inputs)) return fail(PBE_ERR_INVALID, "q_out must lie apart from the inputs");
  if (any_meet(pools, inputs) || any_meet(pools, {{q_out, out_bytes}}))
    return fail(PBE_ERR_INVALID, "pools and scale pools must lie apart from the inputs and q_out");
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    auto ok = [&](const void* ptr, uint64_t bytes) { return !ptr || bytes == 0 || accessible(ptr, bytes, device, &known); };
    if (!ok(q, q_span) || !ok(k, k_span) || !ok(v, v_span) || !ok(q_weight, weight) || !ok(k_weight, weight) ||
        !ok(positions, ints) || !ok(slot_mapping, ints) || (table && !ok(cos_sin, table)) || !ok(q_out, out_bytes) || !ok(key_pool, key_pool_bytes) ||
        !ok(value_pool, value_pool_bytes) ||
        ((fp8 || mx) && (!ok(key_scales, key_scale_bytes) || !ok(value_scales, value_scale_bytes))))
      return fail(PBE_ERR_INVALID, "operands must be memory of device %d", device);
  }
  // Slots that every pool and scale pool holds: by token, or (MXFP4) by block.
  const uint64_t row = (uint64_t)kv_heads * (uint64_t)dim;
  uint64_t slots = std::min(key_pool_bytes, value_pool_bytes);
  if (mx) slots = std::min(slots / (8 * row), std::min(key_scale_bytes, value_scale_bytes) / (row / 2)) * 16;
  else if (fp8) slots = std::min(slots / row, std::min(key_scale_bytes, value_scale_bytes) / ((uint64_t)kv_heads * 4));
  else slots /= 2 * row;
  pbe::RopeParams p{};
  p.q = static_cast<const uint8_t*>(q);
  p.k = static_cast<const uint8_t*>(k);
  p.v = static_cast<const uint8_t*>(v);
  p.q_stride = (uint64_t)(q_stride * elem);
  p.k_stride = (uint64_t)(k_stride * elem);
  p.v_stride = (uint64_t)(v_stride * elem);
  p.q_weight = static_cast<const uint8_t*>(q_weight);
  p.k_weight = static_cast<const uint8_t*>(k_weight);
  p.positions = positions;
  p.cos_sin = cos_sin;
  p.slots = slot_mapping;
  p.q_out = static_cast<uint8_t*>(q_out);
  p.key_pool = static_cast<uint8_t*>(key_pool);
  p.value_pool = static_cast<uint8_t*>(value_pool);
  p.key_scales = static_cast<uint8_t*>(key_scales);
  p.value_scales = static_cast<uint8_t*>(value_scales);
  p.slots_in_pools = (uint32_t)std::min<uint64_t>(slots, 0x80000000u);
  p.n_tokens = (uint32_t)n_tokens;
  p.q_heads = (uint32_t)q_heads;
  p.kv_heads = (uint32_t)kv_heads;
  p.max_position = rotary_dim ? (uint32_t)max_position : 0;
  p.rotary = (uint32_t)rotary_dim;
  p.eps = eps;
  const pbe::PageKind pages = mx ? pbe::PageKind::kMxfp4 : fp8 ? pbe::PageKind::kFp8 : pbe::PageKind::kBf16;
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_qk_norm_rope(p, head_dim, f32, rope_style == PBE_ROPE_PAIRS, pages, compute_units(device), static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

}  // extern "C"
