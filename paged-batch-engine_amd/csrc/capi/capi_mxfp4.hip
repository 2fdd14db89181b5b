// C ABI: MXFP4 pages (their writer and the gather that reads rows back).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <vector>

#include "capi_internal.h"
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
                const void* values, uint64_t elem, int device, pbe::Mxfp4RowsParams* p) {
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
       reinterpret_cast<uintptr_t>(pools.value_scales)) % 4)
    return fail(PBE_ERR_INVALID, "MXFP4 pools and scale pools must be 4-byte aligned");
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    const uint64_t row_bytes = (uint64_t)n_tokens * kv_heads * head_dim * elem;
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
                             slot_mapping, n_tokens, kv_heads, head_dim, keys, values, f32 ? 4 : 2, device, &p);
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
                             slot_mapping, n_tokens, kv_heads, head_dim, keys, values, 2, device, &p);
  if (rc != PBE_OK) return rc;
  p.keys_out = static_cast<uint8_t*>(keys);
  p.values_out = static_cast<uint8_t*>(values);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_gather_kv_mxfp4(p, head_dim, static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

}  // extern "C"
