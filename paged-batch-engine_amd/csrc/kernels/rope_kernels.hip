// gfx950 page writer that norms and rotates first: from a layer's query, key and
// value rows to the reader's queries and the page slots, in one pass.
//   norm      x <- x / sqrt(mean(x^2) + eps) * w, per head, queries and keys
//   rotation  (a, b) <- (a c - b s, b c + a s), c and s of the token's position;
//             a, b are dims i and i + rotary/2, or 2i and 2i + 1 (pairs)
// All of it in FP32, rounded once, to BF16: the type the reader's queries and
// the page writers' rows have. FP8 and MXFP4 pages are made from those rounded
// keys and values, so they hold what the page writers make of the same rows.
//
// Work unit: a lane holds eight dims, head_dim / 8 lanes a head. They take one
// head of a token, or several in turn (a run): cosines, sines and weights are
// then read once for the run, and all of its rows are in flight together.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxfp4_device.h"
#include "rope_kernels.h"

namespace pbe {
namespace {

constexpr int kThreads = 256;

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x2v __attribute__((ext_vector_type(2)));

// Sum over aligned groups of kLanes lanes (8 or 16: within a DPP row), the same
// in every lane.
template <int kLanes>
__device__ __forceinline__ float group_sum(float x) {
  x += dpp_f<0xb1>(x);
  x += dpp_f<0x4e>(x);
  x += dpp_f<0x141>(x);
  if constexpr (kLanes == 16) x += dpp_f<0x140>(x);
  return x;
}

template <bool kF32>
struct Row8 {  // eight input values of a lane
  u32x4 a, b;
  __device__ __forceinline__ void load(const uint8_t* at) {
    a = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
    if constexpr (kF32) b = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at + 16));
  }
  __device__ __forceinline__ void load_kept(const uint8_t* at) {  // other lanes read it too
    a = *reinterpret_cast<const u32x4*>(at);
    if constexpr (kF32) b = *reinterpret_cast<const u32x4*>(at + 16);
  }
  __device__ __forceinline__ void to_f32(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kF32) {
        x[i] = __uint_as_float(a[i]);
        x[4 + i] = __uint_as_float(b[i]);
      } else {
        x[2 * i] = bf16_lo(a[i]);
        x[2 * i + 1] = bf16_hi(a[i]);
      }
    }
  }
};

__device__ __forceinline__ uint32_t round_pair(float x, float y) {  // to nearest even
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v{x, y}), mx_bf16x2));
}

template <int D, bool kF32, PageKind kPages, int kRun>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(const RopeParams p, const bool pairs) {
  constexpr uint32_t L = D / 8, E = kF32 ? 4 : 2;
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= p.units) return;
  const uint32_t vec = u % L, job = u / L;
  const uint32_t token = (__umulhi(job, p.by_runs.mul) + job) >> p.by_runs.shift;
  const uint32_t head0 = (job - token * p.runs) * kRun, heads = p.q_heads + 2 * p.kv_heads;
  const uint32_t d0 = 8 * vec, half = p.rotary / 2;
  // The rows, the table's line and the weights do not wait for each other.
  Row8<kF32> rows[kRun];
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const uint32_t h = min(head0 + i, heads - 1);
    const uint8_t* from = h < p.q_heads ? p.q + token * p.q_stride + h * (D * E)
                          : h < p.q_heads + p.kv_heads ? p.k + token * p.k_stride + (h - p.q_heads) * (D * E)
                                                       : p.v + token * p.v_stride + (h - p.q_heads - p.kv_heads) * (D * E);
    rows[i].load(from + d0 * E);
  }
  const int32_t slot = p.slots[token];
  const int32_t pos = p.positions ? p.positions[token] : 0;
  if (pos < 0) return;
  const bool turns = d0 < p.rotary, placed = p.rotary == 0 || (uint32_t)pos < p.max_position;
  // Cosines and sines of the lane's dims: eight, or (pairs) the first four.
  float c[8], s[8];
  if (turns && placed) {
    const float* line = p.cos_sin + (uint64_t)(uint32_t)pos * p.rotary;
    const float* at = line + (pairs ? d0 / 2 : d0 < half ? d0 : d0 - half);
    const f32x4v c0 = *reinterpret_cast<const f32x4v*>(at), s0 = *reinterpret_cast<const f32x4v*>(at + half);
    f32x4v c1 = c0, s1 = s0;
    if (!pairs) c1 = *reinterpret_cast<const f32x4v*>(at + 4), s1 = *reinterpret_cast<const f32x4v*>(at + half + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = c0[i], s[i] = s0[i], c[4 + i] = c1[i], s[4 + i] = s1[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  }
  float qw[8], kw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qw[i] = kw[i] = 1.f;
  Row8<kF32> w;
  if (p.q_weight && head0 < p.q_heads) w.load_kept(p.q_weight + d0 * E), w.to_f32(qw);
  if (p.k_weight && head0 + kRun > p.q_heads) w.load_kept(p.k_weight + d0 * E), w.to_f32(kw);
  // The lane with the other half of this lane's pairs.
  const uint32_t lane = threadIdx.x & 63, away = p.rotary / 16;
  const uint32_t partner = !turns || pairs ? lane : d0 < half ? lane + away : lane - away;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const uint32_t head = head0 + i;
    const bool is_q = head < p.q_heads, is_v = head >= p.q_heads + p.kv_heads;
    float x[8];
    rows[i].to_f32(x);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
    const float r = __builtin_amdgcn_rsqf(group_sum<L>(ss) * (1.f / D) + p.eps);
    const bool normed = !is_v && (is_q ? p.q_weight : p.k_weight) != nullptr;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = normed ? x[e] * r * (is_q ? qw[e] : kw[e]) : x[e];
    u32x4 y;
    if (pairs) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = x[2 * e], b = x[2 * e + 1];
        y[e] = turns && !is_v ? round_pair(a * c[e] - b * s[e], b * c[e] + a * s[e]) : round_pair(a, b);
      }
    } else {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl(x[e], (int)partner, 64);
        z[e] = turns && !is_v ? x[e] * c[e] + (d0 < half ? -other : other) * s[e] : x[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = round_pair(z[2 * e], z[2 * e + 1]);
    }
    if (!kF32 && is_v) y = rows[i].a;  // the bits as they came, a NaN's too
    if (head >= heads) continue;
    if (is_q) {
      if (!placed) y = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
      *reinterpret_cast<u32x4*>(p.q_out + (((uint64_t)token * p.q_heads + head) * D + d0) * 2) = y;
      continue;
    }
    if (slot < 0 || (uint32_t)slot >= p.slots_in_pools || !placed) continue;
    const uint32_t h = head - p.q_heads - (is_v ? p.kv_heads : 0);
    uint8_t* pool = is_v ? p.value_pool : p.key_pool;
    uint8_t* scales = is_v ? p.value_scales : p.key_scales;
    const uint64_t row = (uint64_t)(uint32_t)slot * p.kv_heads + h;  // of token-major pages
    if constexpr (kPages == PageKind::kBf16) {
      *reinterpret_cast<u32x4*>(pool + (row * D + d0) * 2) = y;
    } else if constexpr (kPages == PageKind::kFp8) {
      const float m = group_max<L>(amax8(y));
      const u32x2 codes = quantise8(y, m > 0.f ? 448.f / m : 0.f);
      *reinterpret_cast<u32x2*>(pool + row * D + d0) = codes;
      if (vec == 0) reinterpret_cast<float*>(scales)[row] = m > 0.f ? m / 448.f : 1.f;
    } else {
      const uint32_t block = (uint32_t)slot / kMxTokens, t = (uint32_t)slot % kMxTokens;
      const uint32_t byte = mx_scale_byte(quad_max(mx_amax_bf16(y)));
      const uint32_t codes = mx_codes_bf16(y, mx_scale(byte));
      uint8_t* at = pool + ((uint64_t)block * p.kv_heads + h) * mx_head_bytes(D);
      if (!is_v || D == 128) {
        *reinterpret_cast<uint32_t*>(at + (is_v ? mx_value_at(D, t, vec) : mx_key_at(D, t, vec))) = codes;
      } else {
        at += mx_value_at(D, t, vec);
        *reinterpret_cast<uint16_t*>(at) = (uint16_t)codes;
        *reinterpret_cast<uint16_t*>(at + mx_column(D)) = (uint16_t)(codes >> 16);
      }
      if (vec % 4 == 0) scales[((uint64_t)block * p.kv_heads + h) * mx_head_scales(D) + mx_scale_at(t, vec)] = (uint8_t)byte;
    }
  }
}

template <int D, bool kF32, PageKind kPages>
hipError_t launch_run(const RopeParams& p, bool pairs, int run, hipStream_t stream) {
  const dim3 grid((p.units + kThreads - 1) / kThreads), block(kThreads);
  if (run == 4) hipLaunchKernelGGL((qk_norm_rope_kernel<D, kF32, kPages, 4>), grid, block, 0, stream, p, pairs);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<D, kF32, kPages, 1>), grid, block, 0, stream, p, pairs);
  return hipGetLastError();
}

template <int D, bool kF32>
hipError_t launch_pages(const RopeParams& p, bool pairs, PageKind pages, int run, hipStream_t stream) {
  switch (pages) {
    case PageKind::kBf16: return launch_run<D, kF32, PageKind::kBf16>(p, pairs, run, stream);
    case PageKind::kFp8: return launch_run<D, kF32, PageKind::kFp8>(p, pairs, run, stream);
    default: return launch_run<D, kF32, PageKind::kMxfp4>(p, pairs, run, stream);
  }
}

}  // namespace

hipError_t launch_qk_norm_rope(RopeParams p, int dim, bool f32_input, bool pairs, PageKind pages, int64_t compute_units, hipStream_t stream) {
  const uint32_t heads = p.q_heads + 2 * p.kv_heads, lanes = (uint32_t)dim / 8;
  const int run = (uint64_t)p.n_tokens * heads * lanes >= (uint64_t)compute_units * 16 * kThreads ? 4 : 1;
  p.runs = (heads + run - 1) / run;
  p.units = p.n_tokens * p.runs * lanes;
  p.by_runs = make_fast_div(p.runs);
  if (dim == 128) return f32_input ? launch_pages<128, true>(p, pairs, pages, run, stream) : launch_pages<128, false>(p, pairs, pages, run, stream);
  if (dim == 64) return f32_input ? launch_pages<64, true>(p, pairs, pages, run, stream) : launch_pages<64, false>(p, pairs, pages, run, stream);
  return hipErrorInvalidValue;
}

}  // namespace pbe
