// Internal interface of the MXFP4 page writer and of its inverse.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernels.h"  // FastDiv

namespace pbe {

struct Mxfp4RowsParams {
  const uint8_t* keys;   // writer: [tokens][kv_heads * dim] of BF16 or FP32, 16-byte aligned rows
  const uint8_t* values;
  uint8_t* keys_out;     // gather: the same in BF16
  uint8_t* values_out;
  uint8_t* key_pool;     // block b at b * half
  uint8_t* value_pool;
  uint8_t* key_scales;   // block b at b * half / 16
  uint8_t* value_scales;
  const int32_t* slots;
  uint32_t blocks;       // that fit all four pools: slots of others are out of range
  uint32_t n_tokens;
  uint32_t units;        // lanes: 16-token groups * kv_heads * 16 * dim / 8 (< 2^31)
  uint32_t kv_heads;
  uint32_t half;
  FastDiv by_heads;
};

hipError_t launch_scatter_kv_mxfp4(const Mxfp4RowsParams& p, int dim, bool f32_input, hipStream_t stream);
hipError_t launch_gather_kv_mxfp4(const Mxfp4RowsParams& p, int dim, hipStream_t stream);

}  // namespace pbe
