// gfx950 writer of new tokens' K/V into MXFP4 pages, and the gather that reads
// rows back. Per group of 32 head dims: scale 2^(floor(log2 amax) - 2), codes
// RNE(x / scale) in E2M1; back, value = code * scale, exact in BF16.
//
// Work unit: one lane takes eight head dims of a token's K row and the same of
// its V row; four lanes share a group, head_dim / 8 a row. Units run [16-token
// group][head][token][dims]: a workgroup holds 16 tokens of a head, which in a
// prompt are the tokens of one block, so the four bytes a lane stores fill the
// head's stretch of that block from one compute unit.
//
// Both are bound by memory, and by the launch where there are few rows. 8,192
// tokens of 4 x 128 BF16 (21 MB): writer 5.4 us, 3.9 TB/s, gather 5.9, 3.6 (FP32 rows,
// 38 MB, on rows that stay: writer 7.8, and 4.6 of BF16); 64 tokens of 2 x 64: 2.5 and 2.4. The writer fetches and writes what it must (17.1
// and 4.5 MB), so whole lines leave a compute unit although a lane stores four bytes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxfp4_device.h"
#include "mxfp4_kernels.h"

namespace pbe {
namespace {

constexpr uint32_t kThreads = 256;

// Where unit u works: its token, head, eight dims, and the block and place of
// the token's slot.
template <int D>
struct Place {
  uint32_t token, head, vec;
  __device__ __forceinline__ Place(uint32_t u, const Mxfp4RowsParams& p) {
    constexpr uint32_t kVecs = D / 8;
    vec = u % kVecs;
    const uint32_t row = u / (kVecs * kMxTokens);
    const uint32_t group = (__umulhi(row, p.by_heads.mul) + row) >> p.by_heads.shift;
    head = row - group * p.kv_heads;
    token = group * kMxTokens + u / kVecs % kMxTokens;
  }
};

template <int D, bool kF32>
__global__ __launch_bounds__(kThreads) void scatter_kv_mxfp4_kernel(const Mxfp4RowsParams p) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  const Place<D> at(u, p);
  // The lanes of a group share one token, so they leave together.
  if (u >= p.units || at.token >= p.n_tokens) return;
  constexpr uint32_t E = kF32 ? 4 : 2;
  const uint64_t in = ((uint64_t)at.token * p.kv_heads + at.head) * (D * E) + at.vec * (8 * E);
  const u32x4* k_in = reinterpret_cast<const u32x4*>(p.keys + in);
  const u32x4* v_in = reinterpret_cast<const u32x4*>(p.values + in);
  const u32x4 k = __builtin_nontemporal_load(k_in), v = __builtin_nontemporal_load(v_in);
  u32x4 k2 = k, v2 = v;
  if constexpr (kF32) k2 = __builtin_nontemporal_load(k_in + 1), v2 = __builtin_nontemporal_load(v_in + 1);
  const int32_t slot = p.slots[at.token];
  const uint32_t block = (uint32_t)slot / kMxTokens, t = (uint32_t)slot % kMxTokens;
  if (slot < 0 || block >= p.blocks) return;
  uint32_t ka, va;
  if constexpr (kF32) ka = max(mx_amax_f32(k), mx_amax_f32(k2)), va = max(mx_amax_f32(v), mx_amax_f32(v2));
  else ka = mx_amax_bf16(k), va = mx_amax_bf16(v);
  const uint32_t ks = mx_scale_byte(quad_max(ka)), vs = mx_scale_byte(quad_max(va));
  uint32_t kc, vc;
  if constexpr (kF32) kc = mx_codes_f32(k, k2, mx_scale(ks)), vc = mx_codes_f32(v, v2, mx_scale(vs));
  else kc = mx_codes_bf16(k, mx_scale(ks)), vc = mx_codes_bf16(v, mx_scale(vs));
  const uint64_t base = (uint64_t)block * p.half + at.head * mx_head_bytes(D);
  *reinterpret_cast<uint32_t*>(p.key_pool + base + mx_key_at(D, t, at.vec)) = kc;
  uint8_t* v_out = p.value_pool + base + mx_value_at(D, t, at.vec);
  if constexpr (D == 128) {
    *reinterpret_cast<uint32_t*>(v_out) = vc;
  } else {
    *reinterpret_cast<uint16_t*>(v_out) = (uint16_t)vc;
    *reinterpret_cast<uint16_t*>(v_out + mx_column(D)) = (uint16_t)(vc >> 16);
  }
  if (at.vec % 4 == 0) {
    const uint64_t sc = (uint64_t)block * (p.half / 16) + at.head * mx_head_scales(D) + mx_scale_at(t, at.vec);
    p.key_scales[sc] = (uint8_t)ks;
    p.value_scales[sc] = (uint8_t)vs;
  }
}

template <int D>
__global__ __launch_bounds__(kThreads) void gather_kv_mxfp4_kernel(const Mxfp4RowsParams p) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  const Place<D> at(u, p);
  if (u >= p.units || at.token >= p.n_tokens) return;
  const int32_t slot = p.slots[at.token];
  if (slot < 0) return;
  const uint32_t block = (uint32_t)slot / kMxTokens, t = (uint32_t)slot % kMxTokens;
  u32x4 k, v;
  if (block >= p.blocks) {
    k = v = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  } else {
    const uint64_t base = (uint64_t)block * p.half + at.head * mx_head_bytes(D);
    const uint64_t sc = (uint64_t)block * (p.half / 16) + at.head * mx_head_scales(D) + mx_scale_at(t, at.vec);
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(p.key_pool + base + mx_key_at(D, t, at.vec));
    const uint8_t* v_at = p.value_pool + base + mx_value_at(D, t, at.vec);
    uint32_t vc;
    if constexpr (D == 128)
      vc = *reinterpret_cast<const uint32_t*>(v_at);
    else
      vc = *reinterpret_cast<const uint16_t*>(v_at) | (uint32_t) * reinterpret_cast<const uint16_t*>(v_at + mx_column(D)) << 16;
    k = mx_values(kc, mx_scale(p.key_scales[sc]));
    v = mx_values(vc, mx_scale(p.value_scales[sc]));
  }
  const uint64_t out = ((uint64_t)at.token * p.kv_heads + at.head) * (D * 2) + at.vec * 16;
  *reinterpret_cast<u32x4*>(p.keys_out + out) = k;
  *reinterpret_cast<u32x4*>(p.values_out + out) = v;
}

}  // namespace

hipError_t launch_scatter_kv_mxfp4(const Mxfp4RowsParams& p, int dim, bool f32_input, hipStream_t stream) {
  const dim3 grid((p.units + kThreads - 1) / kThreads), block(kThreads);
  if (dim == 128) {
    if (f32_input) hipLaunchKernelGGL((scatter_kv_mxfp4_kernel<128, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((scatter_kv_mxfp4_kernel<128, false>), grid, block, 0, stream, p);
  } else if (dim == 64) {
    if (f32_input) hipLaunchKernelGGL((scatter_kv_mxfp4_kernel<64, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((scatter_kv_mxfp4_kernel<64, false>), grid, block, 0, stream, p);
  } else {
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_gather_kv_mxfp4(const Mxfp4RowsParams& p, int dim, hipStream_t stream) {
  const dim3 grid((p.units + kThreads - 1) / kThreads), block(kThreads);
  if (dim == 128) hipLaunchKernelGGL((gather_kv_mxfp4_kernel<128>), grid, block, 0, stream, p);
  else if (dim == 64) hipLaunchKernelGGL((gather_kv_mxfp4_kernel<64>), grid, block, 0, stream, p);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace pbe
