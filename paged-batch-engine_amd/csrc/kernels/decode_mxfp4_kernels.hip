// Decode reader of MXFP4 pages: paged attention for one query token per
// sequence. score = (q . k) * log2(e)/sqrt(D), online softmax in base 2,
// output = sum(p v) / sum(p) in BF16.
//
// A workgroup of four waves reads one piece of a sequence for one KV head, its
// waves tiles of four blocks (64 tokens) in turn.
//  - loads: a block's codes of one head lie in the order of the lanes that
//    take them, so one load instruction reads all of K, and one all of V. The
//    next tile's K is asked for when the scores have used this one's, its V
//    after the values' products.
//  - scores, transposed, on the codes as they are: one scaled 16x16x128 MFMA
//    takes a block's 16 keys (A, E2M1 with the pages' own E8M0 scales) and the
//    query heads of the KV head (B, E4M3, columns). A query is split into two
//    E4M3 numbers of four significant bits, which hold a BF16 number's eight
//    exactly down to 2^-13 of the head's largest, and to 2^-21 of that below;
//    the second pair of MFMA operands adds the lower parts. The MFMA sums a
//    group's products to about 2^-17 of their magnitudes (measured), which is
//    what a score is good for. Lane (g, j) ends with tokens 4g..4g+3 of head j.
//  - values: lane (g, i) holds tokens 4g..4g+3 of column i, the D/16 dims
//    [i*D/16, (i+1)*D/16). The scaled converters make a BF16 pair of a byte, an
//    even and an odd dim of one token, exactly. Both count as terms of one
//    contraction: A row i, of MFMA n, holds dims 2n and 2n + 1 of column i for
//    four tokens a lane, B the probability against the even dims in the
//    columns of heads 0..7 and against the odd ones in columns 8..15 (which
//    carry the same heads again), zero elsewhere. So no two tokens have to be
//    put side by side and no column of B is idle. More than 8 query heads take
//    two such products, of the even and of the odd dims.
//  - probabilities are rounded to BF16 for that product, and the sum they are
//    divided by is of the rounded ones: each weight is off by at most 2^-8 of
//    itself, and they still add up to one.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "decode_device.h"
#include "decode_mxfp4_kernels.h"
#include "mxfp4_device.h"

namespace pbe {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTile = 4;  // blocks of a wave's tile

typedef int i32x8 __attribute__((ext_vector_type(8)));

// A lane's part of one tile.
template <int D>
struct Tile {
  static constexpr int W = D / 32;  // words of codes
  uint32_t k[kTile][W], v[kTile][W];
  uint32_t ks[kTile];  // scale byte of its key's quarter
  uint32_t vs[kTile];  // scale bytes of its four tokens' columns
};

template <int kToken>
__device__ __forceinline__ float token_scale(uint32_t bytes) {  // the converters read the exponent bits alone
  return __uint_as_float(kToken == 3 ? bytes >> 1 : bytes << (23 - 8 * kToken));
}

// Token kT's part of column i as BF16 pairs: c[n] holds dims 2n and 2n + 1.
template <int D, int kT>
__device__ __forceinline__ void token_pairs(const uint32_t (&v)[D / 32], uint32_t scales, uint32_t (&c)[D / 32]) {
  const float s = token_scale<kT>(scales);
  if constexpr (D == 128) {
    c[0] = mx_pair<0>(v[kT], s);
    c[1] = mx_pair<1>(v[kT], s);
    c[2] = mx_pair<2>(v[kT], s);
    c[3] = mx_pair<3>(v[kT], s);
  } else {
    c[0] = mx_pair<2 * (kT % 2)>(v[kT / 2], s);
    c[1] = mx_pair<2 * (kT % 2) + 1>(v[kT / 2], s);
  }
}

// A query head's 32 dims of this lane, BF16 pairs x, as E4M3 numbers hi + lo:
// value = hi * 2^(hi_byte - 127) + lo * 2^(lo_byte - 127). `amax`: FP32 bits of
// the head's largest magnitude, which hi takes to [2^7, 2^8); an infinity or a
// NaN gives byte 255, the NaN scale.
struct SplitQuery {
  i32x8 hi, lo;
  int hi_byte, lo_byte;
};
__device__ __forceinline__ SplitQuery split_query(const u32x4 (&x)[4], uint32_t amax) {
  SplitQuery q;
  const int e = (int)(amax >> 23);
  const int byte = max(e - 7, 4);  // both parts' scales stay within a byte
  q.hi_byte = e == 255 ? 255 : byte;
  q.lo_byte = byte - 4;
  // x * 2^(127 - byte) in two steps, either of them within FP32's exponents
  const int down = 127 - byte, half = down / 2;
  const float s0 = __uint_as_float((uint32_t)(half + 127) << 23), s1 = __uint_as_float((uint32_t)(down - half + 127) << 23);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const uint32_t a = x[w / 2][2 * (w % 2)], b = x[w / 2][2 * (w % 2) + 1];
    const float v[4] = {bf16_lo(a) * s0 * s1, bf16_hi(a) * s0 * s1, bf16_lo(b) * s0 * s1, bf16_hi(b) * s0 * s1};
    uint32_t hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], hi, true);
    const float r[4] = {(v[0] - __builtin_amdgcn_cvt_f32_fp8(hi, 0)) * 16.f, (v[1] - __builtin_amdgcn_cvt_f32_fp8(hi, 1)) * 16.f,
                        (v[2] - __builtin_amdgcn_cvt_f32_fp8(hi, 2)) * 16.f, (v[3] - __builtin_amdgcn_cvt_f32_fp8(hi, 3)) * 16.f};
    uint32_t lo = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], lo, true);
    q.hi[w] = (int)(e == 255 ? 0u : hi);
    q.lo[w] = (int)(e == 255 ? 0u : lo);
  }
  return q;
}

// kWide: more than 8 query heads per KV head.
template <int D, bool kWide>
__global__ __launch_bounds__(kThreads, kWide ? 3 : 4) void paged_decode_mxfp4_kernel(const Mxfp4DecodeParams p) {
  constexpr int W = D / 32;                  // words of K (and of V) codes per lane and block
  constexpr int NT = D / 32;                 // value MFMAs per block (of each parity, kWide)
  constexpr int PARTS = kWide ? 2 : 1;       // accumulators: both parities in one, or even and odd
  constexpr int STEP = kTile * kWaves;       // blocks from a wave's tile to its next
  constexpr int AHEAD = 64 / kTile;          // tiles whose ids a window holds
  constexpr int PITCH = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[kWaves][kWide ? 16 : 8][PITCH];
  __shared__ float lds_m[kWaves][16], lds_l[kWaves][16];

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int h = blockIdx.x, s = blockIdx.y, b = blockIdx.z;
  const int seq = p.seq_lens[b];
  const int nblk = seq > 0 ? (int)(((uint32_t)seq + kBlockTokens - 1) / kBlockTokens) : 0;
  bool bad = seq < 0 || nblk > p.max_blocks;
  const int pieces = bad ? 1 : max(1, (nblk + p.chunk - 1) / p.chunk);
  if (s >= pieces) return;
  const int per = bad ? 0 : (nblk + pieces - 1) / pieces;
  const int c0 = s * per, c1 = bad ? c0 : min(c0 + per, nblk);
  const int first = c0 + w * kTile;
  const int tiles = c1 > first ? (c1 - first + STEP - 1) / STEP : 0;  // of this wave

  // Lane l holds the id of block l % kTile of the wave's tile l / kTile of
  // AHEAD; -1 for one past the piece's end, or outside the pools.
  const int32_t* table = p.tables + (int64_t)b * p.max_blocks;
  int32_t window;
  auto open_window = [&](int tile) {
    const int blk = first + (tile + lane / kTile) * STEP + lane % kTile;
    const int32_t id = table[min(blk, p.max_blocks - 1)];
    const bool ok = id >= 0 && id < p.blocks;
    if (__ballot(blk < c1 && !ok) != 0) bad = true;
    window = blk < c1 && ok ? id : -1;
  };
  open_window(0);
  const uint32_t code_at = lane * (D / 8);
  const uint32_t ks_at = (D == 128 ? g : g / 2) * kMxTokens + j;
  const uint32_t vs_at = (D == 128 ? j / 4 : j / 8) * kMxTokens + 4 * g;
  // Where a tile's blocks lie: a head's codes from the pools' start, a 16th of
  // that for its scales. A block that is none is an empty buffer: its loads
  // return zeros and read no memory.
  uint64_t from[kTile];
  bool live[kTile];
  auto find = [&](int tile) {
    if (tile && tile % AHEAD == 0) open_window(tile);
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      const int32_t id = __builtin_amdgcn_readlane(window, (tile % AHEAD) * kTile + u);
      live[u] = id >= 0;
      from[u] = (uint64_t)(uint32_t)max(id, 0) * p.half + (uint32_t)h * mx_head_bytes(D);
    }
  };
  auto fetch = [&](const uint8_t* pool, const uint8_t* scale_pool, int u, uint32_t (&words)[W], uint32_t& scale, auto wide_scale) {
    const __amdgpu_buffer_rsrc_t codes = __builtin_amdgcn_make_buffer_rsrc((void*)(pool + from[u]), (short)0, live[u] ? mx_head_bytes(D) : 0, 0x00020000);
    const __amdgpu_buffer_rsrc_t scales =
        __builtin_amdgcn_make_buffer_rsrc((void*)(scale_pool + from[u] / 16), (short)0, live[u] ? mx_head_scales(D) : 0, 0x00020000);
    if constexpr (D == 128) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(codes, code_at, 0, 0);
#pragma unroll
      for (int e = 0; e < W; ++e) words[e] = x[e];
    } else {
      const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(codes, code_at, 0, 0);
#pragma unroll
      for (int e = 0; e < W; ++e) words[e] = x[e];
    }
    if constexpr (decltype(wide_scale)::value) scale = __builtin_amdgcn_raw_buffer_load_b32(scales, vs_at, 0, 0);
    else scale = __builtin_amdgcn_raw_buffer_load_b8(scales, ks_at, 0, 0);
  };
  Tile<D> r;
  auto load_keys = [&] {
#pragma unroll
    for (int u = 0; u < kTile; ++u) fetch(p.key_pool, p.key_scales, u, r.k[u], r.ks[u], std::false_type{});
  };
  auto load_values = [&] {
#pragma unroll
    for (int u = 0; u < kTile; ++u) fetch(p.value_pool, p.value_scales, u, r.v[u], r.vs[u], std::true_type{});
  };

  // B of the scores: the scaled MFMA takes terms [16g, 16g + 16) and [64 + 16g,
  // +16) of column j from lane (g, j), where A's lane (g, i) has terms [32g,
  // +32): its key's dims in order, or (D = 64) 16 of them and 16 zeros.
  u32x4 q_in[4] = {};
  const int head = kWide ? j : j % 8;
  {
    const bool has = head < p.group;
    const uint16_t* row = p.q + ((int64_t)b * p.q_heads + (int64_t)h * p.group + (has ? head : 0)) * D;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const uint16_t* at = row + (D == 128 ? 64 * part + 16 * g : 32 * part + 16 * (g / 2));
      const bool mine = has && (D == 128 || g % 2 == 0);
      const u32x4 x = *reinterpret_cast<const u32x4*>(at), y = *reinterpret_cast<const u32x4*>(at + 8);
      q_in[2 * part] = mine ? x : u32x4{0u, 0u, 0u, 0u};
      q_in[2 * part + 1] = mine ? y : u32x4{0u, 0u, 0u, 0u};
    }
  }
  find(0);
  load_keys();
  load_values();
  uint32_t amax = max(max(mx_amax_bf16(q_in[0]), mx_amax_bf16(q_in[1])), max(mx_amax_bf16(q_in[2]), mx_amax_bf16(q_in[3])));
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16, 64));
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32, 64));
  const SplitQuery q = split_query(q_in, amax);
  // Which half of a BF16 pair (p, p) meets this lane's column.
  const uint32_t parity = kWide || j >= 8 ? 0xffff0000u : 0x0000ffffu;

  float m = -INFINITY, l = 0.f;  // of head j: its largest score, and (where parity keeps the upper half) this lane's sum
  f32x4 acc[PARTS][NT];
#pragma unroll
  for (int x = 0; x < PARTS; ++x)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[x][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  // One tile; `part`: fewer than 64 tokens of it count, the piece's last.
  auto compute = [&](int tile, auto part) {
    constexpr bool kPart = decltype(part)::value;
    const int valid = kPart ? min(seq, c1 * kBlockTokens) - (first + tile * STEP) * kBlockTokens : 0;
    f32x4 x[kTile];
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      i32x8 a = {};
#pragma unroll
      for (int e = 0; e < W; ++e) a[e] = (int)r.k[u][e];
      x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      x[u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q.hi, x[u], 4, 0, 0, (int)r.ks[u], 0, q.hi_byte);
      x[u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q.lo, x[u], 4, 0, 0, (int)r.ks[u], 0, q.lo_byte);
    }
    if constexpr (kPart) {
      // Tokens past the end: no score, and zeros for values that may be NaN.
#pragma unroll
      for (int u = 0; u < kTile; ++u) {
        const int mine = min(max(valid - kBlockTokens * u - 4 * g, 0), 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[u][i] = i < mine ? x[u][i] : -INFINITY;
        r.vs[u] &= mine == 4 ? 0xffffffffu : (1u << 8 * mine) - 1u;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if constexpr (D == 128) r.v[u][e] = e < mine ? r.v[u][e] : 0u;
          else r.v[u][e] = 2 * e + 2 <= mine ? r.v[u][e] : 2 * e < mine ? r.v[u][e] & 0xffffu : 0u;
        }
      }
    } else {
      find(tile + 1);
      load_keys();
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kTile; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, x[u][i]);
    const float mn = fmaxf(m, group_max4(top));
    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * p.scale);
    const float base = -mn * p.scale;
    float sum = 0.f;
    uint32_t pb[kTile][4];
#pragma unroll
    for (int u = 0; u < kTile; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // a token past the end gets 0, or NaN where its head has no other score
        // than -infinity or NaN and is NaN whatever this token adds
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][i], p.scale, base));
        pb[u][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{e, e}), mx_bf16x2));
        sum += __uint_as_float(pb[u][i] & 0xffff0000u);
      }
    l = l * alpha + sum;
    m = mn;
    if (__ballot(alpha != 1.f) != 0) {
#pragma unroll
      for (int y = 0; y < PARTS; ++y)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[y][n][i] *= alpha;
    }
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      uint32_t c[4][W];
      token_pairs<D, 0>(r.v[u], r.vs[u], c[0]);
      token_pairs<D, 1>(r.v[u], r.vs[u], c[1]);
      token_pairs<D, 2>(r.v[u], r.vs[u], c[2]);
      token_pairs<D, 3>(r.v[u], r.vs[u], c[3]);
      const u32x4 even{pb[u][0] & 0xffffu, pb[u][1] & 0xffffu, pb[u][2] & 0xffffu, pb[u][3] & 0xffffu};
      const u32x4 kept{pb[u][0] & parity, pb[u][1] & parity, pb[u][2] & parity, pb[u][3] & parity};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bf16x8 a = __builtin_bit_cast(bf16x8, u32x4{c[0][n], c[1][n], c[2][n], c[3][n]});
        acc[0][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, kept), acc[0][n], 0, 0, 0);
        if constexpr (kWide) acc[PARTS - 1][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, even), acc[PARTS - 1][n], 0, 0, 0);
      }
    }
    if constexpr (!kPart) load_values();
  };

  // Only the piece's last tile can be a partial one. A wave asks for a tile
  // past its last one too: its blocks are empty buffers.
  const bool cut = tiles > 0 && min(seq, c1 * kBlockTokens) < (first + (tiles - 1) * STEP + kTile) * kBlockTokens;
  const int whole = cut ? tiles - 1 : tiles;
  for (int tile = 0; tile < whole; ++tile) compute(tile, std::false_type{});
  if (cut) compute(tiles - 1, std::true_type{});

  // The waves' results into one. Lane (g, j) holds dims (4g + r)*D/16 + 2n + (its parity).
  l = group_sum4(l);
  if (g == 0 && (kWide || j >= 8)) {
    lds_m[w][head] = m * p.scale;
    lds_l[w][head] = bad ? __builtin_nanf("") : l;
  }
#pragma unroll
  for (int x = 0; x < PARTS; ++x) {
    const int odd = kWide ? 1 - x : j / 8;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) lds_o[w][head][(4 * g + i) * (D / 16) + 2 * n + odd] = acc[x][n][i];
  }
  __syncthreads();
  for (int unit = threadIdx.x; unit < p.group * (D / 4); unit += kThreads) {
    const int hj = unit / (D / 4), col = unit % (D / 4);
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, lds_m[i][hj]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float li = lds_l[i][hj], wt = li > 0.f ? __builtin_amdgcn_exp2f(lds_m[i][hj] - top) : 0.f;
      sum += li != li ? li : li * wt;
      if (wt > 0.f) o += *reinterpret_cast<const f32x4*>(&lds_o[i][hj][4 * col]) * wt;
    }
    const int64_t row = (int64_t)b * p.q_heads + (int64_t)h * p.group + hj;
    if (pieces > 1) {
      const int64_t at = row * p.splits + s;
      *reinterpret_cast<f32x4*>(p.part_acc + at * D + 4 * col) = o;
      if (col == 0) *reinterpret_cast<f32x2*>(p.part_ml + at * 2) = f32x2{top, sum};
    } else {
      uint16_t e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = to_bf16(sum != sum ? sum : sum > 0.f ? o[i] / sum : 0.f);
      *reinterpret_cast<u32x2*>(p.out + row * D + 4 * col) = u32x2{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16};
    }
  }
}

// The pieces of a sequence into its output: a workgroup per query head, its
// lanes four dims each, D/4 of them a piece.
template <int D>
__global__ __launch_bounds__(kThreads) void paged_decode_mxfp4_join_kernel(const Mxfp4DecodeParams p) {
  constexpr int COLS = D / 4, TEAMS = kThreads / COLS;
  __shared__ f32x4 lds_o[TEAMS][COLS];
  __shared__ f32x2 lds_ml[TEAMS];
  const int row_head = blockIdx.x, b = blockIdx.y;
  const int seq = p.seq_lens[b];
  const int nblk = seq > 0 ? (int)(((uint32_t)seq + kBlockTokens - 1) / kBlockTokens) : 0;
  if (nblk > p.max_blocks) return;
  const int pieces = (nblk + p.chunk - 1) / p.chunk;
  if (pieces <= 1) return;
  const int team = threadIdx.x / COLS, col = threadIdx.x % COLS;
  const int64_t row = (int64_t)b * p.q_heads + row_head;
  const float* acc = p.part_acc + row * p.splits * D + 4 * col;
  const float* ml = p.part_ml + row * p.splits * 2;
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto join = [&](float mi, float li, const f32x4& x) {
    const float mn = fmaxf(m, mi);
    const float keep = l > 0.f ? __builtin_amdgcn_exp2f(m - mn) : 0.f, wt = li > 0.f ? __builtin_amdgcn_exp2f(mi - mn) : 0.f;
    l = (l != l ? l : l * keep) + (li != li ? li : li * wt);
    o = (keep > 0.f ? o * keep : f32x4{0.f, 0.f, 0.f, 0.f}) + (wt > 0.f ? x * wt : f32x4{0.f, 0.f, 0.f, 0.f});
    m = mn;
  };
  for (int s = team; s < pieces; s += TEAMS) {
    const f32x2 q = *reinterpret_cast<const f32x2*>(ml + 2 * s);
    join(q[0], q[1], *reinterpret_cast<const f32x4*>(acc + (int64_t)s * D));
  }
  lds_o[team][col] = o;
  if (col == 0) lds_ml[team] = f32x2{m, l};
  __syncthreads();
  if (team != 0) return;
#pragma unroll
  for (int i = 1; i < TEAMS; ++i) join(lds_ml[i][0], lds_ml[i][1], lds_o[i][col]);
  uint16_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = to_bf16(l != l ? l : l > 0.f ? o[i] / l : 0.f);
  *reinterpret_cast<u32x2*>(p.out + row * D + 4 * col) = u32x2{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16};
}

// A launch takes fewer than 2^32 threads: a batch of more workgroups is read in
// parts, one after another on the stream.
template <int D>
hipError_t launch(const Mxfp4DecodeParams& p, hipStream_t stream) {
  const int64_t most = std::min<int64_t>(0xffffffffll / kThreads / std::max<int64_t>((int64_t)p.kv_heads * p.splits, p.q_heads), 65535);
  if (most < 1) return hipErrorInvalidConfiguration;
  for (int64_t first = 0; first < p.batch; first += most) {
    Mxfp4DecodeParams q = p;
    q.batch = (int32_t)std::min<int64_t>(most, p.batch - first);
    q.seq_lens += first;
    q.tables += first * p.max_blocks;
    q.q += first * p.q_heads * D;
    q.out += first * p.q_heads * D;
    if (p.splits > 1) {  // the workspace may be none otherwise
      q.part_acc += first * p.q_heads * p.splits * D;
      q.part_ml += first * p.q_heads * p.splits * 2;
    }
    const dim3 grid(p.kv_heads, p.splits, q.batch);
    if (p.group > 8) hipLaunchKernelGGL((paged_decode_mxfp4_kernel<D, true>), grid, dim3(kThreads), 0, stream, q);
    else hipLaunchKernelGGL((paged_decode_mxfp4_kernel<D, false>), grid, dim3(kThreads), 0, stream, q);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.splits == 1) continue;
    hipLaunchKernelGGL((paged_decode_mxfp4_join_kernel<D>), dim3(p.q_heads, q.batch), dim3(kThreads), 0, stream, q);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

int32_t mxfp4_decode_splits(int32_t batch, int32_t kv_heads, int32_t max_blocks, int64_t compute_units) {
  const int64_t rows = (int64_t)batch * kv_heads;
  const int64_t most = (max_blocks + kTile * kWaves - 1) / (kTile * kWaves);  // a tile for every wave
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>({4 * compute_units / rows, most, kMxDecodeMaxSplits}));
}

uint64_t mxfp4_decode_workspace_bytes(int32_t batch, int32_t q_heads, int32_t dim, int32_t splits) {
  if (splits <= 1) return 0;
  return (uint64_t)batch * q_heads * splits * (dim + 2) * 4;
}

void plan_mxfp4_decode(Mxfp4DecodeParams* p, int dim, void* workspace) {
  p->chunk = (p->max_blocks + p->splits - 1) / p->splits;
  if (p->splits == 1) return;
  p->part_acc = static_cast<float*>(workspace);
  p->part_ml = p->part_acc + (uint64_t)p->batch * p->q_heads * p->splits * dim;
}

hipError_t launch_paged_decode_mxfp4(const Mxfp4DecodeParams& p, int dim, hipStream_t stream) {
  if (dim == 128) return launch<128>(p, stream);
  if (dim == 64) return launch<64>(p, stream);
  return hipErrorInvalidValue;
}

}  // namespace pbe
