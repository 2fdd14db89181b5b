// Prompt reader: causal attention of many query tokens a sequence over its keys.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "decode_device.h"
#include "mxfp4_device.h"
#include "prompt_kernels.h"

namespace pbe {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));

#define PBE_LDS __attribute__((address_space(3)))

constexpr int kKeys = 64;        // keys of a tile
constexpr int kMinPiece = 8;     // key tiles of a piece that joining is worth
constexpr int kMaxPieces = 256;  // of a tile
constexpr float kLazy = 8.f;     // how far (in base 2) scores may pass the maximum that weights refer to

// ---- which rows and keys a workgroup has ----
struct Unit {
  int b = -1;              // sequence; -1: none for this workgroup
  int tile = 0;            // of its rows
  int s = 0, k = 1;        // which piece of the tile's keys, of how many
  int begin = 0, rows = 0; // first row of q, tokens
  int shown = 0;           // of those, the ones within n_q
  int first = 0;           // first row of k (rows)
  int len = 0;             // keys
  bool bad = false;        // starts or length make no sense
};

template <KeyKind kKind>
__device__ __forceinline__ Unit unit_of(const PromptParams& p, int b) {
  Unit u;
  u.b = b;
  const int lo = p.q_starts[b], hi = p.q_starts[b + 1];
  u.begin = min(max(lo, 0), p.n_q);
  u.bad = lo < 0 || hi < lo || hi > p.n_q;
  u.shown = max(0, min(hi, p.n_q) - u.begin);
  u.rows = u.shown;
  if constexpr (kKind == KeyKind::kRows) {
    const int from = p.lens[b], to = p.lens[b + 1];
    u.bad |= from < 0 || to < from || to > p.n_k;
    u.first = from;
    u.len = u.bad ? 0 : to - from;
  } else {
    const int len = p.lens[b];
    u.bad |= len < 0 || len > 0x7fffff00 || (uint32_t)len > (uint32_t)p.max_blocks * (uint64_t)kBlockTokens;
    u.len = u.bad ? 0 : len;
  }
  return u;
}

__device__ __forceinline__ int key_tiles(int len) { return (int)(((uint32_t)len + kKeys - 1) / kKeys); }

// Unit z of the batch. Every tile of a sequence is cut into as many pieces as its
// whole length gives.
template <KeyKind kKind, int kRows>
__device__ __forceinline__ Unit find_unit(const PromptParams& p, int z, int lane) {
  int c = 0x7fffffff;
  auto tiles_of = [&](const Unit& u) { return (int)(((uint32_t)u.shown * (uint32_t)p.group + kRows - 1) / kRows); };
  if (p.wanted) {
    int64_t sum = 0;
    for (int i = lane; i < p.batch; i += 64) {
      const Unit u = unit_of<kKind>(p, i);
      sum += (int64_t)tiles_of(u) * key_tiles(u.len);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
    c = (int)min((int64_t)0x7fffffff, max((int64_t)kMinPiece, (sum + p.wanted - 1) / p.wanted));
  }
  int before = 0;
  for (int i = 0; i < p.batch; i += 64) {
    Unit u;
    int n = 0, k = 1;
    if (i + lane < p.batch) {
      u = unit_of<kKind>(p, i + lane);
      const int kt = key_tiles(u.len);
      k = p.wanted ? min(kMaxPieces, max(1, (kt + c - 1) / c)) : 1;
      n = tiles_of(u) * k;
    }
    const int upto = wave_scan(n) + before;
    const uint64_t past = __ballot(upto > z);
    if (past) {
      const int at = __builtin_ctzll(past);
      Unit r;
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      r.b = i + at;
      r.k = of(k);
      r.begin = of(u.begin);
      r.rows = r.shown = of(u.shown);
      r.first = of(u.first);
      r.len = of(u.len);
      r.bad = of(u.bad);
      const int w = z - of(upto - n), tiles = of(n) / r.k;
      r.tile = tiles - 1 - w / r.k;  // those that see the most keys first
      r.s = w % r.k;
      return r;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return Unit{};
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const f32x2 v{a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The sum of a word's two BF16 values and c, in FP32.
typedef short s16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float sum_bf16(uint32_t x, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2, x), s16x2{0x3f80, 0x3f80}, c, false);
}

// Where the 16-byte chunk c of row r of a K or V tile lies in LDS (in bytes): the
// chunks of a row change places so that the lanes of a read hit different banks.
template <int D>
__device__ __forceinline__ uint32_t k_at(uint32_t r, uint32_t c) {
  return r * (2 * D) + ((c ^ (r & (D / 8 - 1))) * 16);
}
template <int D>
__device__ __forceinline__ uint32_t v_at(uint32_t r, uint32_t c) {
  return r * (2 * D) + ((c ^ ((2 * r) & (D / 8 - 1))) * 16);
}

// ---- keys and values into LDS ----
// 16 bytes a lane from `from` to LDS, lane after lane from `to` on, past the
// registers. Written as an instruction because the compiler would wait for the
// builtin's result before any read of LDS; here arrived() says when it is there.
// It writes no register but m0, which nothing else here uses.
__device__ __forceinline__ void load_to_lds(const uint8_t* from, PBE_LDS uint8_t* to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"((uint32_t)(uintptr_t)to) : "memory");
}
// Waits for all that this wave has asked global memory for (vmcnt 0, no other counter).
__device__ __forceinline__ void arrived() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);
  asm volatile("" ::: "memory");
}

template <int D, KeyKind kKind, int kWaves>
struct Stage {
  static constexpr int T = 64 * kWaves;
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kRowsAnInstr = 1024 / (2 * D), kInstrs = kKeys / kRowsAnInstr / kWaves;
  static constexpr int kFp8Units = kKeys * D / 16, kFp8Each = (kFp8Units + T - 1) / T;
  static constexpr int kMxEach = (256 + T - 1) / T;
  static constexpr bool kDirect = kKind == KeyKind::kRows || kKind == KeyKind::kBf16;

  const PromptParams& p;
  const Unit& u;
  int head, lane, wave, nblocks;
  int32_t ids = 0, next_ids = 0;  // of 64 blocks from `chunk` on, a lane each, and of the next 64
  uint64_t bad = 0, next_bad = 0;
  int chunk = -1;
  // FP8, MXFP4: what waits in registers to be converted
  u32x4 kr[kKind == KeyKind::kFp8 ? kFp8Each : kMxEach], vr[kKind == KeyKind::kFp8 ? kFp8Each : kMxEach];
  uint32_t sk[kMxEach], sv[kMxEach];

  __device__ __forceinline__ Stage(const PromptParams& p_, const Unit& u_, int head_, int lane_, int wave_)
      : p(p_), u(u_), head(head_), lane(lane_), wave(wave_), nblocks((int)(((uint32_t)u_.len + kBlockTokens - 1) / kBlockTokens)) {}

  __device__ __forceinline__ void load_ids(int first, int32_t* to, uint64_t* wrong) {
    const int i = min(first + lane, nblocks - 1);
    int32_t id = p.tables[(int64_t)u.b * p.max_blocks + i];
    const bool off = id < 0 || id >= p.blocks;
    *wrong = __ballot(off);
    *to = off ? 0 : id;
  }
  // Makes the ids of key tile kt's blocks (kt counts up by one) ready.
  __device__ __forceinline__ void ids_for(int kt) {
    if constexpr (kKind != KeyKind::kRows) {
      const int c = kt / 16 * 64;
      if (c == chunk) return;
      if (chunk < 0) {
        load_ids(c, &ids, &bad);
      } else {
        ids = next_ids;
        bad = next_bad;
      }
      chunk = c;
      load_ids(c + 64, &next_ids, &next_bad);
    }
  }
  // Which of a key tile's four blocks are not in the pools.
  __device__ __forceinline__ uint32_t wrong_blocks(int kt) const { return (uint32_t)(bad >> (kt % 16 * 4)) & 15u; }

  // Byte offset of the K (or V) row of key j, of this head.
  __device__ __forceinline__ uint64_t row_at(int j, uint64_t stride) const {
    if constexpr (kKind == KeyKind::kRows) {
      return (uint64_t)(u.first + j) * stride;
    } else {
      const uint32_t id = (uint32_t)__shfl(ids, (j / kBlockTokens) & 63, 64);
      return (uint64_t)id * p.half + (uint64_t)(j % kBlockTokens) * stride;
    }
  }

  // Asks for key tile kt.
  __device__ __forceinline__ void load(int kt, PBE_LDS uint8_t* ks, PBE_LDS uint8_t* vs) {
    ids_for(kt);
    const int last = u.len - 1;
    if constexpr (kDirect) {
#pragma unroll
      for (int i = 0; i < kInstrs; ++i) {
        const int r0 = (wave * kInstrs + i) * kRowsAnInstr;
        const uint32_t r = (uint32_t)r0 + (uint32_t)lane / (D / 8), c = (uint32_t)lane % (D / 8);
        const int j = min(kt * kKeys + (int)r, last);
        const uint64_t at = (uint64_t)head * (2 * D);
        const uint8_t* kp = p.k + row_at(j, p.k_stride) + at + (c ^ (r & (D / 8 - 1))) * 16;
        const uint8_t* vp = p.v + row_at(j, p.v_stride) + at + (c ^ ((2 * r) & (D / 8 - 1))) * 16;
        load_to_lds(kp, ks + r0 * (2 * D));
        load_to_lds(vp, vs + r0 * (2 * D));
      }
    } else if constexpr (kKind == KeyKind::kFp8) {
#pragma unroll
      for (int i = 0; i < kFp8Each; ++i) {
        const int unit = min((int)threadIdx.x + i * T, kFp8Units - 1);
        const int j = min(kt * kKeys + unit / (D / 16), last);
        const uint64_t at = row_at(j, p.k_stride) + (uint64_t)head * D + (uint64_t)(unit % (D / 16)) * 16;
        kr[i] = *(PBE_GLOBAL const u32x4*)(uintptr_t)(p.k + at);
        vr[i] = *(PBE_GLOBAL const u32x4*)(uintptr_t)(p.v + at);
      }
      const int j = min(kt * kKeys + lane, last);
      const uint32_t id = (uint32_t)__shfl(ids, (j / kBlockTokens) & 63, 64);
      const uint64_t at = (((uint64_t)id * kBlockTokens + (uint64_t)(j % kBlockTokens)) * (uint64_t)p.kv_heads + (uint64_t)head) * 4;
      if (wave == 0) sk[0] = *(PBE_GLOBAL const uint32_t*)(uintptr_t)(p.k_scales + at);
      if (wave == 1) sk[0] = *(PBE_GLOBAL const uint32_t*)(uintptr_t)(p.v_scales + at);
    } else {
      const int last_block = nblocks - 1;
#pragma unroll
      for (int i = 0; i < kMxEach; ++i) {
        const int unit = min((int)threadIdx.x + i * T, 255);
        {  // K: 64 tokens, four quarters of the dims each
          const int tok = unit / 4, quarter = unit % 4, block = min(kt * 4 + tok / kBlockTokens, last_block);
          const uint64_t id = (uint64_t)(uint32_t)__shfl(ids, block & 63, 64);
          const uint64_t at = id * p.half + (uint64_t)head * mx_head_bytes(D) + (uint64_t)(quarter * kBlockTokens + tok % kBlockTokens) * (D / 8);
          if constexpr (D == 128) kr[i] = *(PBE_GLOBAL const u32x4*)(uintptr_t)(p.k + at);
          else kr[i].xy = *(PBE_GLOBAL const u32x2*)(uintptr_t)(p.k + at);
          sk[i] = *(PBE_GLOBAL const uint8_t*)(uintptr_t)(p.k_scales + id * (p.half / 16) + (uint64_t)head * mx_head_scales(D) +
                                                          (D == 128 ? quarter : quarter / 2) * kBlockTokens + tok % kBlockTokens);
        }
        {  // V: 16 quads of tokens, 16 columns of dims each
          const int quad = unit / 16, column = unit % 16, block = min(kt * 4 + quad / 4, last_block);
          const uint64_t id = (uint64_t)(uint32_t)__shfl(ids, block & 63, 64);
          const uint64_t at = id * p.half + (uint64_t)head * mx_head_bytes(D) + (uint64_t)(quad % 4) * (2 * D) + (uint64_t)column * (D / 8);
          if constexpr (D == 128) vr[i] = *(PBE_GLOBAL const u32x4*)(uintptr_t)(p.v + at);
          else vr[i].xy = *(PBE_GLOBAL const u32x2*)(uintptr_t)(p.v + at);
          sv[i] = *(PBE_GLOBAL const uint32_t*)(uintptr_t)(p.v_scales + id * (p.half / 16) + (uint64_t)head * mx_head_scales(D) +
                                                           (D == 128 ? column / 4 : column / 8) * kBlockTokens + quad % 4 * 4);
        }
      }
    }
  }

  // Puts what load() asked for into the tiles (a direct load does so by itself).
  __device__ __forceinline__ void store(PBE_LDS uint8_t* ks, PBE_LDS uint8_t* vs, PBE_LDS float* scales) {
    if constexpr (kKind == KeyKind::kFp8) {
#pragma unroll
      for (int i = 0; i < kFp8Each; ++i) {
        const int unit = (int)threadIdx.x + i * T;
        if (kFp8Units % T && unit >= kFp8Units) break;
        const uint32_t r = (uint32_t)unit / (D / 16), c = 2 * ((uint32_t)unit % (D / 16));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x2 a = e4m3x4_to_bf16x4_cvt(kr[i][2 * e]), b = e4m3x4_to_bf16x4_cvt(kr[i][2 * e + 1]);
          *(PBE_LDS u32x4*)(ks + k_at<D>(r, c + e)) = u32x4{a.x, a.y, b.x, b.y};
          const u32x2 x = e4m3x4_to_bf16x4_cvt(vr[i][2 * e]), y = e4m3x4_to_bf16x4_cvt(vr[i][2 * e + 1]);
          *(PBE_LDS u32x4*)(vs + v_at<D>(r, c + e)) = u32x4{x.x, x.y, y.x, y.y};
        }
      }
      if (wave == 0) scales[lane] = __uint_as_float(sk[0]);
      if (wave == 1) scales[kKeys + lane] = __uint_as_float(sk[0]);
    } else if constexpr (kKind == KeyKind::kMxfp4) {
#pragma unroll
      for (int i = 0; i < kMxEach; ++i) {
        const int unit = (int)threadIdx.x + i * T;
        if (256 % T && unit >= 256) break;
        const uint32_t tok = (uint32_t)unit / 4, quarter = (uint32_t)unit % 4;
        const float scale = mx_scale(sk[i]);
#pragma unroll
        for (uint32_t e = 0; e < D / 32; ++e) *(PBE_LDS u32x4*)(ks + k_at<D>(tok, quarter * (D / 32) + e)) = mx_values(kr[i][e], scale);
        const uint32_t quad = (uint32_t)unit / 16, column = (uint32_t)unit % 16;
#pragma unroll
        for (uint32_t t = 0; t < 4; ++t) {
          const float s = mx_scale((sv[i] >> (8 * t)) & 255u);
          if constexpr (D == 128) {
            *(PBE_LDS u32x4*)(vs + v_at<D>(4 * quad + t, column)) = mx_values(vr[i][t], s);
          } else {
            const uint32_t codes = vr[i][t / 2] >> (16 * (t % 2));
            *(PBE_LDS u32x2*)(vs + v_at<D>(4 * quad + t, column / 2) + 8 * (column % 2)) = u32x2{mx_pair<0>(codes, s), mx_pair<1>(codes, s)};
          }
        }
      }
    }
  }
};

// Non-zero where one of a word's two BF16 values is an infinity or a NaN.
__device__ __forceinline__ uint32_t special(uint32_t x) { return ((x & 0x7fff7fffu) + 0x00800080u) & 0x80008000u; }

template <int D, KeyKind kKind, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves / 2) void prompt_attention_kernel(const PromptParams p) {
  constexpr int kRows = 32 * kWaves, kTile = kKeys * D * 2, kDims = D / 32;
  using S = Stage<D, kKind, kWaves>;
  // two turns of a tile's keys and values; of FP8 ones, their scales
  __shared__ __align__(1024) uint8_t tile_mem[4 * kTile];
  __shared__ __align__(16) float scale_mem[kKind == KeyKind::kFp8 ? 4 * kKeys : 4];
  __shared__ uint32_t special_mem[kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int z = blockIdx.x / p.kv_heads, head = blockIdx.x - z * p.kv_heads;
  const Unit u = find_unit<kKind, kRows>(p, z, lane);
  if (u.b < 0) return;
  const int h = lane >> 5, col = lane & 31;
  const int stacked = u.rows * p.group;                       // rows of the sequence and this head
  const int row0 = u.tile * kRows + wave * 32;                // of the wave
  auto token_of = [&](int r) { return (int)fast_div((uint32_t)min(r, stacked - 1), p.by_group); };
  const int token = token_of(row0 + col), g = min(row0 + col, stacked - 1) - token * p.group;
  const int q_heads = p.kv_heads * p.group;
  const int64_t q_row = (int64_t)u.begin + token;
  const int q_head = head * p.group + g;
  auto seen_by = [&](int tok) { return max(0, u.len - u.rows + tok + 1); };
  const int seen = seen_by(token);
  const int wave_least = seen_by(token_of(row0)), wave_most = row0 < stacked ? seen_by(token_of(row0 + 31)) : 0;
  const int tile_least = seen_by(token_of(u.tile * kRows)), tile_most = seen_by(token_of(u.tile * kRows + kRows - 1));
  const int all = key_tiles(tile_most);
  const int kt0 = (int)((int64_t)all * u.s / u.k), kt1 = (int)((int64_t)all * (u.s + 1) / u.k);

  bf16x8 q[D / 16];
  {
    const uint8_t* at = p.q + (uint64_t)q_row * p.q_stride + (uint64_t)q_head * (2 * D) + h * 16;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = *(PBE_GLOBAL const bf16x8*)(uintptr_t)(at + i * 32);
  }
  f32x16 o[kDims];
#pragma unroll
  for (int i = 0; i < kDims; ++i) o[i] = f32x16{};
  float m = -INFINITY, l = 0.f;

  S stage(p, u, head, lane, wave);
  PBE_LDS uint8_t* const tiles = (PBE_LDS uint8_t*)tile_mem;
  PBE_LDS float* const tile_scales = (PBE_LDS float*)scale_mem;
  auto keys_at = [&](int turn) { return tiles + turn * (2 * kTile); };
  auto values_at = [&](int turn) { return tiles + turn * (2 * kTile) + kTile; };
  uint32_t wrong = 0, next_wrong = 0;
  if (kt0 < kt1) {
    stage.load(kt0, keys_at(0), values_at(0));
    stage.store(keys_at(0), values_at(0), tile_scales);
    next_wrong = stage.wrong_blocks(kt0);
  }
  for (int kt = kt0; kt < kt1; ++kt) {
    const int turn = (kt - kt0) & 1;
    const int first = kt * kKeys;
    if constexpr (S::kDirect) arrived();
    __syncthreads();
    wrong = next_wrong;
    PBE_LDS const uint8_t* kb = keys_at(turn);
    PBE_LDS const uint8_t* vb = values_at(turn);
    const bool more = kt + 1 < kt1;
    if (more) {
      stage.load(kt + 1, keys_at(turn ^ 1), values_at(turn ^ 1));
      if constexpr (kKind != KeyKind::kRows) next_wrong = stage.wrong_blocks(kt + 1);
    }
    // Values that some of the tile's rows do not see may be anything: an infinity
    // or a NaN times a weight of zero would reach those rows.
    bool odd = false;
    if (first + kKeys > tile_least) {
      uint32_t some = 0;
#pragma unroll
      for (int i = 0; i < kTile / (64 * kWaves * 16); ++i) {
        const u32x4 x = *(PBE_LDS const u32x4*)(vb + (i * 64 * kWaves + threadIdx.x) * 16);
        some |= special(x.x) | special(x.y) | special(x.z) | special(x.w);
      }
      const bool any = __ballot(some != 0) != 0;
      if (lane == 0) special_mem[wave] = any;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWaves; ++i) odd |= special_mem[i] != 0;
    }
    if (first < wave_most) {
      f32x16 s[2];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        s[sub] = f32x16{};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const bf16x8 a = *(PBE_LDS const bf16x8*)(kb + k_at<D>(sub * 32 + col, 2 * i + h));
          s[sub] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, q[i], s[sub], 0, 0, 0);
        }
      }
      auto key_of = [&](int sub, int i) { return first + sub * 32 + 8 * (i / 4) + 4 * h + i % 4; };
      PBE_LDS const float* scales = tile_scales + turn * (2 * kKeys);
      if constexpr (kKind == KeyKind::kFp8) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 f = *(PBE_LDS const f32x4*)(scales + sub * 32 + 8 * i + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[sub][4 * i + e] *= f[e];
          }
      }
      if (kKind != KeyKind::kRows && wrong) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (wrong >> (2 * sub + i / 8) & 1) s[sub][i] = NAN;
      }
      const bool masked = first + kKeys > wave_least;
      if (masked) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[sub][i] = key_of(sub, i) < seen ? s[sub][i] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[0][i]);
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[1][i]);
      top = halves_max(top);
      // The maximum that weights refer to follows the largest score only when that
      // has passed it by 2^kLazy: sums then need no scaling for most tiles.
      if (__any((top - m) * p.scale > kLazy || (m == -INFINITY && top > m))) {
        const float now = fmaxf(m, top);
        const float fade = m == now ? 1.f : __builtin_amdgcn_exp2f((m - now) * p.scale);
        m = now;
        l *= fade;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= fade;
      }
      const float base = m == -INFINITY ? 0.f : m;
      bf16x8 w[4];
      float sum = 0.f;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[sub][i] = __builtin_amdgcn_exp2f((s[sub][i] - base) * p.scale);
          if constexpr (kKind == KeyKind::kFp8) sum += s[sub][i];
        }
      if constexpr (kKind == KeyKind::kFp8) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 f = *(PBE_LDS const f32x4*)(scales + kKeys + sub * 32 + 8 * i + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[sub][4 * i + e] *= f[e];
          }
        if (masked) {
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[sub][i] = key_of(sub, i) < seen ? s[sub][i] : 0.f;
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        u32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = pack_bf16(s[n / 2][8 * (n % 2) + 2 * e], s[n / 2][8 * (n % 2) + 2 * e + 1]);
        w[n] = __builtin_bit_cast(bf16x8, x);
        if constexpr (kKind != KeyKind::kFp8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sum = sum_bf16(x[e], sum);
        }
      }
      l += sum;
      // lane l of 16: four dims of key l / 4; it gets dim l of four keys
      auto values = [&](int d, int n) {
        const uint32_t i = lane & 15, chunk = 4 * d + 2 * ((lane >> 4) & 1) + (i % 4) / 2;
        s16x4 a, b;
        const uint32_t r = 16 * n + 4 * h + i / 4;
        a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PBE_LDS s16x4*)(vb + v_at<D>(r, chunk) + 8 * (i % 2)));
        b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PBE_LDS s16x4*)(vb + v_at<D>(r + 8, chunk) + 8 * (i % 2)));
        const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
        return u32x4{x.x, x.y, y.x, y.y};
      };
      if (!odd) {
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int n = 0; n < 4; ++n)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values(d, n)), w[n], o[d], 0, 0, 0);
      } else {
        // Infinities and NaN are counted apart, for the rows that see them.
        bf16x8 sees[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          u32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = (key_of(n / 2, 8 * (n % 2) + 2 * e) < seen ? 0x3f80u : 0u) | (key_of(n / 2, 8 * (n % 2) + 2 * e + 1) < seen ? 0x3f800000u : 0u);
          sees[n] = __builtin_bit_cast(bf16x8, x);
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          f32x16 up = {}, down = {};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const u32x4 x = values(d, n);
            u32x4 fine, plus, minus;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t lo = x[e] & 0xffffu, hi = x[e] >> 16;
              const bool lo_off = (lo & 0x7f80u) == 0x7f80u, hi_off = (hi & 0x7f80u) == 0x7f80u;
              fine[e] = (lo_off ? 0u : lo) | (hi_off ? 0u : hi << 16);
              // a NaN counts as both infinities
              plus[e] = (lo_off && lo != 0xff80u ? 0x3f80u : 0u) | (hi_off && hi != 0xff80u ? 0x3f800000u : 0u);
              minus[e] = (lo_off && lo != 0x7f80u ? 0x3f80u : 0u) | (hi_off && hi != 0x7f80u ? 0x3f800000u : 0u);
            }
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fine), w[n], o[d], 0, 0, 0);
            up = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, plus), sees[n], up, 0, 0, 0);
            down = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, minus), sees[n], down, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (up[i] > 0.f) o[d][i] += INFINITY;
            if (down[i] > 0.f) o[d][i] -= INFINITY;
          }
        }
      }
    }
    if (more) stage.store(keys_at(turn ^ 1), values_at(turn ^ 1), tile_scales + (turn ^ 1) * (2 * kKeys));
  }

  l = halves_sum(l);
  if (row0 + col >= stacked) return;
  if (u.k == 1) {
    const float over = u.bad ? NAN : seen > 0 ? 1.f / l : 0.f;
    uint8_t* at = p.out + ((uint64_t)q_row * (uint64_t)q_heads + (uint64_t)q_head) * (2 * D) + h * 8;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(PBE_GLOBAL u32x2*)(uintptr_t)(at + d * 64 + i * 16) =
            u32x2{pack_bf16(o[d][4 * i] * over, o[d][4 * i + 1] * over), pack_bf16(o[d][4 * i + 2] * over, o[d][4 * i + 3] * over)};
  } else {
    const uint64_t row = ((uint64_t)z * (uint64_t)p.kv_heads + (uint64_t)head) * kRows + (uint64_t)(wave * 32 + col);
    float* acc = p.part_acc + row * D + 4 * h;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) *(PBE_GLOBAL f32x4*)(uintptr_t)(acc + d * 32 + i * 8) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (h == 0) *(PBE_GLOBAL f32x2*)(uintptr_t)(p.part_ml + row * 2) = f32x2{m, l};
  }
}

// Joins the pieces of the tiles that were cut: piece s of k takes the s-th part of
// the tile's rows.
template <int D, KeyKind kKind, int kWaves>
__global__ __launch_bounds__(256) void prompt_join_kernel(const PromptParams p) {
  constexpr int kRows = 32 * kWaves, kLanes = D / 4;
  const int lane = threadIdx.x & 63;
  const int z = blockIdx.x / p.kv_heads, head = blockIdx.x - z * p.kv_heads;
  const Unit u = find_unit<kKind, kRows>(p, z, lane);
  if (u.b < 0 || u.k == 1) return;
  const int stacked = u.rows * p.group;
  const int from = kRows * u.s / u.k, to = kRows * (u.s + 1) / u.k;
  const int q_heads = p.kv_heads * p.group;
  const uint64_t z0 = (uint64_t)(z - u.s);
  for (int r = from + (int)threadIdx.x / kLanes; r < to; r += 256 / kLanes) {
    const int row = u.tile * kRows + r;
    if (row >= stacked) break;
    const int token = (int)fast_div((uint32_t)row, p.by_group), g = row - token * p.group, d = 4 * (threadIdx.x % kLanes);
    const int seen = max(0, u.len - u.rows + token + 1);
    auto place = [&](int s) { return ((z0 + (uint64_t)s) * (uint64_t)p.kv_heads + (uint64_t)head) * kRows + (uint64_t)r; };
    float m = -INFINITY;
    for (int s = 0; s < u.k; ++s) m = fmaxf(m, p.part_ml[place(s) * 2]);
    const float base = m == -INFINITY ? 0.f : m;
    f32x4 acc = {};
    float l = 0.f;
    for (int s = 0; s < u.k; ++s) {
      const uint64_t at = place(s);
      const float f = __builtin_amdgcn_exp2f((p.part_ml[at * 2] - base) * p.scale);
      l += p.part_ml[at * 2 + 1] * f;
      const f32x4 x = *(PBE_GLOBAL const f32x4*)(uintptr_t)(p.part_acc + at * D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += x[e] * f;
    }
    const float over = seen > 0 ? 1.f / l : 0.f;
    *(PBE_GLOBAL u32x2*)(uintptr_t)(p.out + (((uint64_t)u.begin + token) * (uint64_t)q_heads + (uint64_t)(head * p.group + g)) * (2 * D) + 2 * d) =
        u32x2{pack_bf16(acc[0] * over, acc[1] * over), pack_bf16(acc[2] * over, acc[3] * over)};
  }
}

template <int D, KeyKind kKind, int kWaves>
hipError_t launch(const PromptParams& p, hipStream_t stream) {
  const dim3 grid((uint32_t)(p.units * p.kv_heads));
  hipLaunchKernelGGL((prompt_attention_kernel<D, kKind, kWaves>), grid, dim3(64 * kWaves), 0, stream, p);
  if (p.wanted) hipLaunchKernelGGL((prompt_join_kernel<D, kKind, kWaves>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int D, KeyKind kKind>
hipError_t launch_rows(const PromptParams& p, int rows, hipStream_t stream) {
  return rows == 64 ? launch<D, kKind, 2>(p, stream) : launch<D, kKind, 4>(p, stream);
}

template <int D>
hipError_t launch_kind(const PromptParams& p, KeyKind kind, int rows, hipStream_t stream) {
  switch (kind) {
    case KeyKind::kRows: return launch_rows<D, KeyKind::kRows>(p, rows, stream);
    case KeyKind::kBf16: return launch_rows<D, KeyKind::kBf16>(p, rows, stream);
    case KeyKind::kFp8: return launch_rows<D, KeyKind::kFp8>(p, rows, stream);
    default: return launch_rows<D, KeyKind::kMxfp4>(p, rows, stream);
  }
}

}  // namespace

int prompt_tile_rows(int64_t n_q, int64_t batch, int32_t group) { return n_q * group <= 64 * batch ? 64 : 128; }

int64_t prompt_units(int64_t n_q, int64_t batch, int32_t group, int rows, int64_t wanted) {
  return n_q * group / rows + std::min(batch, n_q) + wanted;
}

uint64_t prompt_workspace_bytes(int64_t units, int32_t kv_heads, int32_t head_dim, int rows) {
  return (uint64_t)units * (uint64_t)kv_heads * (uint64_t)rows * (uint64_t)(head_dim + 2) * 4;
}

hipError_t launch_prompt_attention(const PromptParams& p, int dim, KeyKind kind, int rows, hipStream_t stream) {
  if (dim == 128) return launch_kind<128>(p, kind, rows, stream);
  if (dim == 64) return launch_kind<64>(p, kind, rows, stream);
  return hipErrorInvalidValue;
}

}  // namespace pbe
