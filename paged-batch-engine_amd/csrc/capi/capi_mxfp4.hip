// C ABI: MXFP4 pages (their writer, the gather that reads rows back and the
// decode reader).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "capi_internal.h"
#include "../kernels/decode_mxfp4_kernels.h"
#include "../kernels/mxfp4_kernels.h"

using namespace pbe_capi;

namespace {

constexpr uint64_t kTokens = 16;

struct Pools {
  const void* key;
  uint64_t key_bytes;
  const void* value;
  uint64_t value_bytes;
  const uint8_t* key_scales;
  uint64_t key_scale_bytes;
  const uint8_t* value_scales;
  uint64_t value_scale_bytes;
};

// Checks what writer and gather share, and fills `p` but for the rows.
int rows_params(const Pools& pools, const int32_t* slots, int32_t n_tokens, int32_t kv_heads, int32_t head_dim, const void* keys,
                const void* values, uint64_t elem, bool rows_written, int device, pbe::Mxfp4RowsParams* p) {
  if (head_dim != 64 && head_dim != 128) return fail(PBE_ERR_UNSUPPORTED, "MXFP4 pages hold heads of 64 or 128 dims");
  if (!slots || !keys || !values || !pools.key || !pools.value || !pools.key_scales || !pools.value_scales)
    return fail(PBE_ERR_INVALID, "null MXFP4 operand");
  const uint64_t half = kTokens * (uint64_t)kv_heads * (uint64_t)head_dim / 2;
  if (half > 0xffffffffull) return fail(PBE_ERR_INVALID, "a block of one plane must be smaller than 4 GiB");
  const uint64_t units = ((uint64_t)n_tokens + kTokens - 1) / kTokens * kTokens * (uint64_t)kv_heads * (uint64_t)(head_dim / 8);
  if (units >= 0x80000000ull) return fail(PBE_ERR_INVALID, "too many tokens for one launch");
  if ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) % 16)
    return fail(PBE_ERR_INVALID, "K/V rows must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(pools.key) | reinterpret_cast<uintptr_t>(pools.value) | reinterpret_cast<uintptr_t>(pools.key_scales) |
       reinterpret_cast<uintptr_t>(pools.value_scales) | reinterpret_cast<uintptr_t>(slots)) % 4)
    return fail(PBE_ERR_INVALID, "MXFP4 pools, scale pools and slots must be 4-byte aligned");
  const uint64_t row_bytes = (uint64_t)n_tokens * kv_heads * head_dim * elem;
  const Span k{keys, row_bytes}, v{values, row_bytes}, s{slots, (uint64_t)n_tokens * 4};
  const std::initializer_list<Span> pages = {{pools.key, pools.key_bytes}, {pools.value, pools.value_bytes},
                                             {pools.key_scales, pools.key_scale_bytes}, {pools.value_scales, pools.value_scale_bytes}};
  // Workgroups read rows, pages and slots while others write.
  if (any_meet({k, v}, pages) || (rows_written ? meet(k, v) || any_meet({k, v}, {s}) : any_meet({s}, pages)))
    return fail(PBE_ERR_INVALID, "what is written must lie apart from what is read, and key rows from value rows");
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    auto ok = [&](const void* ptr, uint64_t bytes) { return bytes == 0 || accessible(ptr, bytes, device, &known); };
    if (!ok(keys, row_bytes) || !ok(values, row_bytes) || !ok(slots, (uint64_t)n_tokens * 4) || !ok(pools.key, pools.key_bytes) ||
        !ok(pools.value, pools.value_bytes) || !ok(pools.key_scales, pools.key_scale_bytes) ||
        !ok(pools.value_scales, pools.value_scale_bytes))
      return fail(PBE_ERR_INVALID, "MXFP4 operands must be memory of device %d", device);
  }
  // A block counts where all four pools hold it whole; slots are 31 bits.
  const uint64_t blocks = std::min(std::min(pools.key_bytes, pools.value_bytes) / half,
                                   std::min(pools.key_scale_bytes, pools.value_scale_bytes) / (half / 16));
  p->key_pool = static_cast<uint8_t*>(const_cast<void*>(pools.key));
  p->value_pool = static_cast<uint8_t*>(const_cast<void*>(pools.value));
  p->key_scales = const_cast<uint8_t*>(pools.key_scales);
  p->value_scales = const_cast<uint8_t*>(pools.value_scales);
  p->slots = slots;
  p->blocks = (uint32_t)std::min<uint64_t>(blocks, 0x7fffffffu);
  p->n_tokens = (uint32_t)n_tokens;
  p->units = (uint32_t)units;
  p->kv_heads = (uint32_t)kv_heads;
  p->half = (uint32_t)half;
  p->by_heads = pbe::make_fast_div((uint32_t)kv_heads);
  return PBE_OK;
}

}  // namespace

extern "C" {

int pbe_scatter_kv_mxfp4(const void* keys, const void* values, int32_t in_dtype, int32_t n_tokens,
                         const int32_t* slot_mapping, int32_t kv_heads, int32_t head_dim,
                         void* key_pool, uint64_t key_pool_bytes, void* value_pool,
                         uint64_t value_pool_bytes, uint8_t* key_scales, uint64_t key_scale_bytes,
                         uint8_t* value_scales, uint64_t value_scale_bytes, int device,
                         void* stream) {
  if (in_dtype != PBE_IN_BF16 && in_dtype != PBE_IN_F32) return fail(PBE_ERR_INVALID, "unknown input dtype %d", (int)in_dtype);
  if (n_tokens < 0 || kv_heads <= 0 || head_dim <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "n_tokens >= 0, kv_heads, head_dim > 0 and a device");
  if (n_tokens == 0) return PBE_OK;
  const bool f32 = in_dtype == PBE_IN_F32;
  pbe::Mxfp4RowsParams p{};
  const int rc = rows_params({key_pool, key_pool_bytes, value_pool, value_pool_bytes, key_scales, key_scale_bytes, value_scales, value_scale_bytes},
                             slot_mapping, n_tokens, kv_heads, head_dim, keys, values, f32 ? 4 : 2, false, device, &p);
  if (rc != PBE_OK) return rc;
  p.keys = static_cast<const uint8_t*>(keys);
  p.values = static_cast<const uint8_t*>(values);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_scatter_kv_mxfp4(p, head_dim, f32, static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

int pbe_gather_kv_mxfp4(const void* key_pool, uint64_t key_pool_bytes, const void* value_pool,
                        uint64_t value_pool_bytes, const uint8_t* key_scales,
                        uint64_t key_scale_bytes, const uint8_t* value_scales,
                        uint64_t value_scale_bytes, const int32_t* slot_mapping, int32_t n_tokens,
                        int32_t kv_heads, int32_t head_dim, void* keys, void* values, int device,
                        void* stream) {
  if (n_tokens < 0 || kv_heads <= 0 || head_dim <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "n_tokens >= 0, kv_heads, head_dim > 0 and a device");
  if (n_tokens == 0) return PBE_OK;
  pbe::Mxfp4RowsParams p{};
  const int rc = rows_params({key_pool, key_pool_bytes, value_pool, value_pool_bytes, key_scales, key_scale_bytes, value_scales, value_scale_bytes},
                             slot_mapping, n_tokens, kv_heads, head_dim, keys, values, 2, true, device, &p);
  if (rc != PBE_OK) return rc;
  p.keys_out = static_cast<uint8_t*>(keys);
  p.values_out = static_cast<uint8_t*>(values);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_gather_kv_mxfp4(p, head_dim, static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

int32_t pbe_paged_decode_mxfp4_splits(int32_t batch, int32_t kv_heads, int32_t max_blocks_per_seq) {
  if (batch <= 0 || kv_heads <= 0 || max_blocks_per_seq <= 0) return 1;
  return pbe::mxfp4_decode_splits(batch, kv_heads, max_blocks_per_seq, compute_units());
}

uint64_t pbe_paged_decode_mxfp4_workspace_bytes(int32_t batch, int32_t q_heads, int32_t head_dim,
                                                int32_t splits) {
  if (batch <= 0 || q_heads <= 0 || head_dim <= 0 || splits <= 0) return 0;
  return pbe::mxfp4_decode_workspace_bytes(batch, q_heads, head_dim, splits);
}

int pbe_paged_decode_mxfp4(const void* key_pool, const void* value_pool, uint64_t pool_bytes,
                           const uint8_t* key_scales, const uint8_t* value_scales,
                           uint64_t scale_pool_bytes, int32_t kv_heads, int32_t head_dim,
                           const void* queries, void* outputs, int32_t batch, int32_t q_heads,
                           const int32_t* block_tables, const int32_t* seq_lens,
                           int32_t max_blocks_per_seq, int32_t splits, void* workspace,
                           uint64_t workspace_bytes, int device, void* stream) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || max_blocks_per_seq <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "batch, q_heads, kv_heads, max_blocks_per_seq > 0 and a device");
  if (head_dim != 64 && head_dim != 128) return fail(PBE_ERR_UNSUPPORTED, "MXFP4 pages hold heads of 64 or 128 dims");
  if (q_heads % kv_heads != 0 || q_heads / kv_heads > pbe::kMxDecodeMaxGroup)
    return fail(PBE_ERR_UNSUPPORTED, "q_heads must be 1..%d times kv_heads", pbe::kMxDecodeMaxGroup);
  if (!key_pool || !value_pool || !key_scales || !value_scales || !queries || !outputs || !block_tables || !seq_lens)
    return fail(PBE_ERR_INVALID, "null decode operand");
  auto at = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
  if ((at(queries) | at(outputs) | at(key_pool) | at(value_pool) | at(workspace)) % 16 || (at(key_scales) | at(value_scales)) % 4 ||
      (at(block_tables) | at(seq_lens)) % 4)
    return fail(PBE_ERR_INVALID, "queries, outputs, pools and workspace must be 16-byte aligned, scale pools and tables 4-byte aligned");
  if (splits < 0 || splits > pbe::kMxDecodeMaxSplits) return fail(PBE_ERR_INVALID, "splits must be 0..%d", pbe::kMxDecodeMaxSplits);
  // so that no product below passes 64 bits
  if ((int64_t)batch * q_heads > INT32_MAX || (int64_t)batch * max_blocks_per_seq > (1ll << 40))
    return fail(PBE_ERR_INVALID, "batch * q_heads must be at most INT32_MAX and batch * max_blocks_per_seq at most 2^40");
  const uint64_t half = kTokens * (uint64_t)kv_heads * (uint64_t)head_dim / 2;
  if (half > 0xffffffffull) return fail(PBE_ERR_INVALID, "a block of one plane must be smaller than 4 GiB");
  if (pool_bytes < half || scale_pool_bytes < half / 16) return fail(PBE_ERR_INVALID, "pools and scale pools must hold at least one block");
  if (splits == 0) {
    splits = pbe_paged_decode_mxfp4_splits(batch, kv_heads, max_blocks_per_seq);
    const uint64_t two = pbe::mxfp4_decode_workspace_bytes(batch, q_heads, head_dim, 2);  // linear in the splits
    splits = (int32_t)std::max<uint64_t>(1, std::min<uint64_t>((uint64_t)splits, workspace ? workspace_bytes / (two / 2) : 1));
  }
  const uint64_t need = pbe::mxfp4_decode_workspace_bytes(batch, q_heads, head_dim, splits);
  if (need && !workspace) return fail(PBE_ERR_INVALID, "more than one split needs a workspace");
  if (workspace_bytes < need)
    return fail(PBE_ERR_INVALID, "decode workspace holds %llu of %llu bytes", (unsigned long long)workspace_bytes, (unsigned long long)need);
  const uint64_t rows = (uint64_t)batch * (uint64_t)q_heads * (uint64_t)head_dim * 2;
  const Span q{queries, rows}, out{outputs, rows}, partials{workspace, need};
  // The outputs may take the queries' place, row for row: a KV head's are written when all that read its queries have.
  if (any_meet({out, partials}, {{key_pool, pool_bytes}, {value_pool, pool_bytes}, {key_scales, scale_pool_bytes}, {value_scales, scale_pool_bytes},
                                 {block_tables, (uint64_t)batch * (uint64_t)max_blocks_per_seq * 4}, {seq_lens, (uint64_t)batch * 4}}) ||
      meet(out, partials) || meet(q, partials) || (queries != outputs && meet(q, out)))
    return fail(PBE_ERR_INVALID, "decode outputs and workspace must lie apart from each other and from what is read");
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    auto ok = [&](const void* ptr, uint64_t bytes) { return bytes == 0 || accessible(ptr, bytes, device, &known); };
    if (!ok(key_pool, pool_bytes) || !ok(value_pool, pool_bytes) || !ok(key_scales, scale_pool_bytes) || !ok(value_scales, scale_pool_bytes) ||
        !ok(queries, rows) || !ok(outputs, rows) || !ok(block_tables, (uint64_t)batch * (uint64_t)max_blocks_per_seq * 4) ||
        !ok(seq_lens, (uint64_t)batch * 4) || !ok(workspace, need))
      return fail(PBE_ERR_INVALID, "decode operands must be memory of device %d", device);
    // Arrival tickets are device atomics, which not every link carries to host memory.
    if (need && on_host(workspace, known)) return fail(PBE_ERR_INVALID, "the decode workspace must be device memory");
  }
  pbe::Mxfp4DecodeParams p{};
  p.key_pool = static_cast<const uint8_t*>(key_pool);
  p.value_pool = static_cast<const uint8_t*>(value_pool);
  p.key_scales = key_scales;
  p.value_scales = value_scales;
  p.q = static_cast<const uint16_t*>(queries);
  p.out = static_cast<uint16_t*>(outputs);
  p.tables = block_tables;
  p.seq_lens = seq_lens;
  p.half = (uint32_t)half;
  p.batch = batch;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.group = q_heads / kv_heads;
  p.max_blocks = max_blocks_per_seq;
  p.blocks = (int32_t)std::min<uint64_t>(std::min(pool_bytes / half, scale_pool_bytes / (half / 16)), INT32_MAX);
  p.scale = (1.f / std::sqrt((float)head_dim)) * 1.4426950408889634f;
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_paged_decode_mxfp4(p, head_dim, splits, workspace, compute_units(device), static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

}  // extern "C"
