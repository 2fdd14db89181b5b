// Device helpers of MXFP4 pages: E2M1 codes with an E8M0 scale per 32 head
// dims, and where a token's codes and scales lie in a block of 16 tokens.
#pragma once
#include "fp8_device.h"

namespace pbe {
namespace {

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kMxGroup = 32;   // head dims that share a scale
constexpr uint32_t kMxTokens = 16;  // of a block

// Bytes of one KV head's codes (K or V) and scales in a block.
constexpr uint32_t mx_head_bytes(uint32_t dim) { return kMxTokens * dim / 2; }
constexpr uint32_t mx_head_scales(uint32_t dim) { return kMxTokens * dim / kMxGroup; }

// Offsets within a head's stretch of token `t`'s dims [8*vec, 8*vec + 8). Four
// bytes of K; of V, four bytes (dim 128) or two pairs of bytes, the second
// mx_column(dim) after the first (dim 64: columns of four dims).
constexpr uint32_t mx_column(uint32_t dim) { return 4 * (dim / 32); }
__device__ __forceinline__ uint32_t mx_key_at(uint32_t dim, uint32_t t, uint32_t vec) {
  const uint32_t quarter = 8 * vec / (dim / 4);
  return (quarter * kMxTokens + t) * (dim / 8) + 4 * (vec - quarter * (dim / 32));
}
__device__ __forceinline__ uint32_t mx_value_at(uint32_t dim, uint32_t t, uint32_t vec) {
  return (t / 4) * 16 * mx_column(dim) + 8 * vec / (dim / 16) * mx_column(dim) + (t % 4) * (dim / 32);
}
__device__ __forceinline__ uint32_t mx_scale_at(uint32_t t, uint32_t vec) { return vec / 4 * kMxTokens + t; }

// The E8M0 byte of a group whose largest magnitude has FP32 bits `amax`: its
// exponent less two, that of the largest code. Magnitudes are compared as
// integers, so an infinity or a NaN wins and gives 255, the NaN scale.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// A scale byte as the scaled converters take it: they read the eight exponent
// bits of a float and nothing else of it, 255 as NaN, 0 as 2^-127.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Largest of four lanes' values in each of them (the lanes of one group).
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));
}
__device__ __forceinline__ uint32_t mx_amax_f32(u32x4 x) {
  return max(max(x.x & 0x7fffffffu, x.y & 0x7fffffffu), max(x.z & 0x7fffffffu, x.w & 0x7fffffffu));
}
__device__ __forceinline__ uint32_t mx_amax_bf16(u32x4 x) {  // as FP32 bits
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(x[i] & 0x7fff0000u, (x[i] << 16) & 0x7fff0000u));
  return m;
}

// Eight values over `scale` as codes, even dims low: the converter rounds to
// nearest, ties to the even code, and keeps to 6 in magnitude.
__device__ __forceinline__ uint32_t mx_codes_bf16(u32x4 x, float scale) {
  auto pair = [&](int i) {
    const uint32_t w = x[i];  // a bit cast of the vector's element itself takes the first one's bits
    return __builtin_bit_cast(mx_bf16x2, w);
  };
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, pair(0), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair(1), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair(2), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair(3), scale, 3);
}
__device__ __forceinline__ uint32_t mx_codes_f32(u32x4 a, u32x4 b, float scale) {
  auto f = [](uint32_t u) { return __uint_as_float(u); };
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f(a.x), f(a.y), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(a.z), f(a.w), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(b.x), f(b.y), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(b.z), f(b.w), scale, 3);
}

// Two values of byte kByte of `codes` as a BF16 pair (exact).
template <int kByte>
__device__ __forceinline__ uint32_t mx_pair(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kByte));
}
__device__ __forceinline__ u32x4 mx_values(uint32_t codes, float scale) {
  return u32x4{mx_pair<0>(codes, scale), mx_pair<1>(codes, scale), mx_pair<2>(codes, scale), mx_pair<3>(codes, scale)};
}

}  // namespace
}  // namespace pbe
