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
// head of a token, or (a run) up to four of its query, key or value heads in
// turn: cosines, sines and weights are then read once for the run, and all of
// its rows are in flight together.
//
// What bounds it: the rows' bytes in large calls (8,191 tokens of (28 + 2 x 4) x
// 128: BF16 28.7 us, 5.4 TB/s; FP32 in, half of the dims turned in pairs 40.5 us,
// 5.6 TB/s), the launch and one chain of arguments, position, line of the table
// and rows in small ones (one token 2.5 us in a graph). The pages' kind changes
// little: 8,192 tokens as above into BF16, FP8 and MXFP4 pages 29.6 / 30.9 / 30.4 us,
// 5,040 of (12 + 2 x 2) x 128 10.6 / 11.2 / 10.9, 64 of these 2.9 / 3.2 / 3.1; without
// norms up to 0.6 less, or 0.9 more. A token's few bytes of an MXFP4 page leave a
// compute unit by themselves, so that those pages' 4.5 MB (of 63.2 written) count as
// 10.8. Halves of a whole head
// change lanes by DPP; through LDS, as parts of a head's dims do, with kinds of
// heads mixed in a run, the BF16 call took 33.4.
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

// x of the lane half a head away: 8 of 16 lanes, or 4 of 8 (mirrored within the
// eight, then within each four).
template <int kLanes>
__device__ __forceinline__ float half_away(float x) {
  if constexpr (kLanes == 16) return dpp_f<0x128>(x);  // row_ror 8
  return dpp_f<0x1b>(dpp_f<0x141>(x));
}

enum class Turn { kNone, kPairs, kHead, kPart };  // kHead: halves of the whole head, kPart: of its first dims

// K or V row `y` (BF16) of a token's head into its slot.
template <int D, PageKind kPages>
__device__ __forceinline__ void store_row(const RopeParams& p, bool is_v, uint32_t slot, uint32_t h, uint32_t vec, u32x4 y) {
  uint8_t* pool = is_v ? p.value_pool : p.key_pool;
  uint8_t* scales = is_v ? p.value_scales : p.key_scales;
  const uint64_t row = (uint64_t)slot * p.kv_heads + h;  // of token-major pages
  if constexpr (kPages == PageKind::kBf16) {
    *reinterpret_cast<u32x4*>(pool + (row * D + 8 * vec) * 2) = y;
  } else if constexpr (kPages == PageKind::kFp8) {
    const float m = group_max<D / 8>(amax8(y));
    const u32x2 codes = quantise8(y, m > 0.f ? 448.f / m : 0.f);
    *reinterpret_cast<u32x2*>(pool + row * D + 8 * vec) = codes;
    if (vec == 0) reinterpret_cast<float*>(scales)[row] = m > 0.f ? m / 448.f : 1.f;
  } else {
    const uint32_t block = slot / kMxTokens, t = slot % kMxTokens;
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

template <int D, bool kF32, PageKind kPages, int kRun>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(const RopeParams p, const Turn turn) {
  constexpr uint32_t L = D / 8, E = kF32 ? 4 : 2;
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= p.units) return;
  const uint32_t vec = u % L, job = u / L, d0 = 8 * vec, half = p.rotary / 2;
  const uint32_t token = (__umulhi(job, p.by_runs.mul) + job) >> p.by_runs.shift, run = job - token * p.runs;
  const bool is_q = run < p.q_runs, is_v = run >= p.q_runs + p.kv_runs;
  const uint32_t head0 = (is_q ? run : is_v ? run - p.q_runs - p.kv_runs : run - p.q_runs) * kRun;
  const uint32_t count = min((uint32_t)kRun, (is_q ? p.q_heads : p.kv_heads) - head0);
  // The rows, the table's line and the weights do not wait for each other.
  const uint8_t* from = (is_q ? p.q + token * p.q_stride : is_v ? p.v + token * p.v_stride : p.k + token * p.k_stride) + (head0 * D + d0) * E;
  Row8<kF32> rows[kRun];
#pragma unroll
  for (int i = 0; i < kRun; ++i) rows[i].load(from + (i < (int)count ? i * (D * E) : 0));
  const int32_t pos = p.positions ? p.positions[token] : 0;
  const int32_t slot = p.slots[token];
  const uint8_t* weight = is_v ? nullptr : is_q ? p.q_weight : p.k_weight;
  Row8<kF32> weights;
  if (weight) weights.load_kept(weight + d0 * E);
  if (pos < 0) return;
  const bool placed = turn == Turn::kNone || (uint32_t)pos < p.max_position, turns = d0 < p.rotary && placed && !is_v;
  // Cosines and sines of the lane's dims: eight, or (pairs) the first four. In
  // the first half of a head's dims the sine counts negative.
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  if (turns) {
    const float* at = p.cos_sin + (uint64_t)(uint32_t)pos * p.rotary + (turn == Turn::kPairs ? d0 / 2 : d0 < half ? d0 : d0 - half);
    const f32x4v c0 = *reinterpret_cast<const f32x4v*>(at), s0 = *reinterpret_cast<const f32x4v*>(at + half);
    f32x4v c1 = c0, s1 = s0;
    if (turn != Turn::kPairs) c1 = *reinterpret_cast<const f32x4v*>(at + 4), s1 = *reinterpret_cast<const f32x4v*>(at + half + 4);
    const bool minus = turn != Turn::kPairs && d0 < half;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = c0[i], s[i] = minus ? -s0[i] : s0[i], c[4 + i] = c1[i], s[4 + i] = minus ? -s1[i] : s1[i];
  }
  float w[8];
  if (weight) weights.to_f32(w);
  const bool stored = placed && slot >= 0 && (uint32_t)slot < p.slots_in_pools;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    if (i >= (int)count) break;
    float x[8];
    u32x4 y;
    rows[i].to_f32(x);
    if (is_v) {
      if constexpr (kF32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = round_pair(x[2 * e], x[2 * e + 1]);
      } else {
        y = rows[i].a;  // the bits as they came, a NaN's too
      }
    } else {
      if (weight) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
        const float r = __builtin_amdgcn_rsqf(group_sum<L>(ss) * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
      }
      float z[8];
      if (turn == Turn::kHead) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = x[e] * c[e] + half_away<L>(x[e]) * s[e];
      } else if (turn == Turn::kPairs) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = x[2 * e], b = x[2 * e + 1];
          z[2 * e] = a * c[e] - b * s[e];
          z[2 * e + 1] = b * c[e] + a * s[e];
        }
      } else if (turn == Turn::kPart) {
        // the lane with the other half of this lane's pairs
        const uint32_t lane = threadIdx.x & 63, away = p.rotary / 16;
        const uint32_t partner = d0 >= p.rotary ? lane : d0 < half ? lane + away : lane - away;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float other = __shfl(x[e], (int)partner, 64);
          z[e] = d0 < p.rotary ? x[e] * c[e] + other * s[e] : x[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = x[e];
      }
      // Past the turned dims a pair's c = 1 and s = 0 leave a finite value as it
      // is, but 0 times an infinity is none.
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = turn == Turn::kPairs && d0 >= p.rotary ? round_pair(x[2 * e], x[2 * e + 1]) : round_pair(z[2 * e], z[2 * e + 1]);
    }
    if (is_q) {
      if (!placed) y = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
      *reinterpret_cast<u32x4*>(p.q_out + (((uint64_t)token * p.q_heads + head0 + i) * D + d0) * 2) = y;
    } else if (stored) {
      store_row<D, kPages>(p, is_v, (uint32_t)slot, head0 + i, vec, y);
    }
  }
}

template <int D, bool kF32, PageKind kPages>
hipError_t launch_run(const RopeParams& p, Turn turn, int run, hipStream_t stream) {
  const dim3 grid((p.units + kThreads - 1) / kThreads), block(kThreads);
  if (run == 4) hipLaunchKernelGGL((qk_norm_rope_kernel<D, kF32, kPages, 4>), grid, block, 0, stream, p, turn);
  else if (run == 2) hipLaunchKernelGGL((qk_norm_rope_kernel<D, kF32, kPages, 2>), grid, block, 0, stream, p, turn);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<D, kF32, kPages, 1>), grid, block, 0, stream, p, turn);
  return hipGetLastError();
}

template <int D, bool kF32>
hipError_t launch_pages(const RopeParams& p, Turn turn, PageKind pages, int run, hipStream_t stream) {
  switch (pages) {
    case PageKind::kBf16: return launch_run<D, kF32, PageKind::kBf16>(p, turn, run, stream);
    case PageKind::kFp8: return launch_run<D, kF32, PageKind::kFp8>(p, turn, run, stream);
    default: return launch_run<D, kF32, PageKind::kMxfp4>(p, turn, run, stream);
  }
}

}  // namespace

hipError_t launch_qk_norm_rope(RopeParams p, int dim, bool f32_input, bool pairs, PageKind pages, int64_t compute_units, hipStream_t stream) {
  const uint32_t lanes = (uint32_t)dim / 8;
  const Turn turn = p.rotary == 0 ? Turn::kNone : pairs ? Turn::kPairs : (int)p.rotary == dim ? Turn::kHead : Turn::kPart;
  // Runs pay where one head at a time is many workgroups per compute unit. us in
  // a graph, 1 / 2 / 4 heads: 8,191 tokens of (28 + 2 x 4) x 128 BF16 (72 of them)
  // 36.7 / 31.9 / 28.7 (floor 23.5), 16,384 of (12 + 2 x 2) x 128 (64) 36.1 / 31.5 /
  // 28.9; 5,040 of these (20) 12.2 / 10.8 / 10.8, 5,040 of (14 + 2 x 2) x 64 (11) 7.8
  // / 6.9 / 7.6, 2,000 of (12 + 2 x 2) x 128 (8) 5.3 / 5.1 / 5.8; 512 (2) 3.3 / 3.5 /
  // 4.2, 1 2.5 / 2.8 / 3.4. Other pages turn at the same places: 8,192 of (28 + 2 x 4)
  // x 128, FP8 36.2 / 31.8 / 30.4, MXFP4 38.7 / 34.3 / 30.6; 5,040 of (12 + 2 x 2) x 128
  // 12.2 / 11.1 / 12.5 and 12.6 / 10.9 / 11.5; 64 3.2 / 3.7 / 4.4 and 3.1 / 3.5 / 4.2.
  const uint64_t each = (uint64_t)p.n_tokens * (p.q_heads + 2 * p.kv_heads) * lanes / ((uint64_t)compute_units * kThreads);
  const int run = each >= 24 ? 4 : each >= 8 ? 2 : 1;
  p.q_runs = (p.q_heads + run - 1) / run;
  p.kv_runs = (p.kv_heads + run - 1) / run;
  p.runs = p.q_runs + 2 * p.kv_runs;
  p.units = p.n_tokens * p.runs * lanes;
  p.by_runs = make_fast_div(p.runs);
  if (dim == 128) return f32_input ? launch_pages<128, true>(p, turn, pages, run, stream) : launch_pages<128, false>(p, turn, pages, run, stream);
  if (dim == 64) return f32_input ? launch_pages<64, true>(p, turn, pages, run, stream) : launch_pages<64, false>(p, turn, pages, run, stream);
  return hipErrorInvalidValue;
}

}  // namespace pbe
