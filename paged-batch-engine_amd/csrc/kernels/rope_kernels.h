// Internal interface of the page writer that norms and rotates heads first.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernels.h"  // FastDiv

namespace pbe {

enum class PageKind : int { kBf16, kFp8, kMxfp4 };

struct RopeParams {
  const uint8_t* q;          // row t at t * q_stride bytes, 16-byte aligned
  const uint8_t* k;
  const uint8_t* v;
  uint64_t q_stride, k_stride, v_stride;
  const uint8_t* q_weight;   // [dim] of the input's type, or null
  const uint8_t* k_weight;
  const int32_t* positions;  // [tokens], or null: no token is padding
  const float* cos_sin;      // [max_position][rotary]: cosines, then sines
  const int32_t* slots;      // [tokens]
  uint8_t* q_out;            // bf16 [tokens][q_heads][dim]
  uint8_t* key_pool;
  uint8_t* value_pool;
  uint8_t* key_scales;       // FP8: fp32 [slot][kv_head]; MXFP4: bytes by block
  uint8_t* value_scales;
  uint32_t slots_in_pools;   // slots at or beyond it are not written
  uint32_t n_tokens, q_heads, kv_heads;
  uint32_t max_position, rotary;
  float eps;
  uint32_t runs;             // of heads per token: q_runs + 2 * kv_runs
  uint32_t q_runs, kv_runs;
  uint32_t units;            // lanes (< 2^31)
  FastDiv by_runs;
};

// Sets runs to by_runs; n_tokens * (q_heads + 2 * kv_heads) * dim / 8 < 2^31.
hipError_t launch_qk_norm_rope(RopeParams p, int dim, bool f32_input, bool pairs, PageKind pages, int64_t compute_units, hipStream_t stream);

}  // namespace pbe
