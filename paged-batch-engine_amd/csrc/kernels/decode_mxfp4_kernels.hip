// Decode reader of MXFP4 pages: paged attention for one query token per
// sequence. score = (q . k) * log2(e)/sqrt(D), online softmax in base 2,
// output = sum(p v) / sum(p) in BF16.
//
// A workgroup of four waves reads one piece of a sequence for one KV head, its
// waves tiles of four blocks (64 tokens) in turn.
//  - loads: a block's codes of one head lie in the order of the lanes that
//    take them, so one load instruction reads all of K, and one all of V.
//  - scores, transposed: A = the block's 16 keys, B = the query heads of the KV
//    head (columns, padded to 16), one v_mfma_f32_16x16x32_bf16 per 32 dims.
//    Lane (g, j) holds quarter g of key j's dims, an eighth of them an MFMA, and
//    ends with tokens 4g..4g+3 of query head j. The scaled converters make two
//    BF16 values of a byte and its scale, exactly.
//  - values: lane (g, i) holds tokens 4g..4g+3 of column i, the D/16 dims
//    [i*D/16, (i+1)*D/16): two blocks give the eight tokens of the A operand
//    of O^T += V^T P^T (row i of MFMA n is dim i*D/16 + n), which are the eight
//    tokens whose probabilities the lane holds as the B operand. Only pairs of
//    tokens have to be put side by side, so values pass no LDS.
//  - probabilities are rounded to BF16 for that product, and the sum they are
//    divided by is of the rounded ones: each weight is off by at most 2^-8 of
//    itself, and they still add up to one.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "decode_device.h"
#include "decode_mxfp4_kernels.h"
#include "mxfp4_device.h"

namespace pbe {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTile = 4;  // blocks of a wave's tile

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

// Tokens kT of column i as BF16 pairs of dims: c[m] holds dims 2m and 2m + 1.
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

template <int D>
__global__ __launch_bounds__(kThreads, 2) void paged_decode_mxfp4_kernel(const Mxfp4DecodeParams p) {
  constexpr int W = D / 32;   // words of K (and of V) codes per lane and block
  constexpr int NK = D / 32;  // score MFMAs per block
  constexpr int NT = D / 16;  // value MFMAs per two blocks
  constexpr int PITCH = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[kWaves][kMxDecodeMaxGroup][PITCH];
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
  const int c0 = s * per;
  int c1 = bad ? c0 : min(c0 + per, nblk);

  const int32_t* table = p.tables + (int64_t)b * p.max_blocks;
  // The wave's tiles: kTile blocks of every kTile * kWaves. Lane l holds the id
  // of block l % kTile of the tile l / kTile further on.
  const int first = c0 + w * kTile;
  auto ids_from = [&](int tile) {
    return table[min(first + (tile + lane / kTile) * (kTile * kWaves) + lane % kTile, p.max_blocks - 1)];
  };
  int32_t window = ids_from(0);
  const uint32_t head_codes = h * mx_head_bytes(D), head_scales = h * mx_head_scales(D);
  const uint32_t code_at = lane * (D / 8);
  const uint32_t ks_at = (D == 128 ? g : g / 2) * kMxTokens + j;
  const uint32_t vs_at = (D == 128 ? j / 4 : j / 8) * kMxTokens + 4 * g;
  // Every call issues the same loads. A block past the piece's end, or whose id
  // is none of the pools', is an empty buffer: zeros, and no memory read.
  auto load = [&](int tile, Tile<D>& r) {
    if (tile && tile % (64 / kTile) == 0) window = ids_from(tile);
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      const int blk = first + tile * (kTile * kWaves) + u;
      int32_t id = __builtin_amdgcn_readlane(window, (tile % (64 / kTile)) * kTile + u);
      const bool want = blk < c1, ok = id >= 0 && id < p.blocks;
      if (want && !ok) bad = true, c1 = min(c1, blk);
      if (!ok) id = 0;
      const uint64_t codes = (uint64_t)id * p.half + head_codes, scales = (uint64_t)id * (p.half / 16) + head_scales;
      const uint32_t code_span = want && ok ? mx_head_bytes(D) : 0, scale_span = want && ok ? mx_head_scales(D) : 0;
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(p.key_pool + codes), (short)0, code_span, 0x00020000);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(p.value_pool + codes), (short)0, code_span, 0x00020000);
      const __amdgpu_buffer_rsrc_t rks = __builtin_amdgcn_make_buffer_rsrc((void*)(p.key_scales + scales), (short)0, scale_span, 0x00020000);
      const __amdgpu_buffer_rsrc_t rvs = __builtin_amdgcn_make_buffer_rsrc((void*)(p.value_scales + scales), (short)0, scale_span, 0x00020000);
      if constexpr (D == 128) {
        const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rk, code_at, 0, 0), y = __builtin_amdgcn_raw_buffer_load_b128(rv, code_at, 0, 0);
#pragma unroll
        for (int e = 0; e < W; ++e) r.k[u][e] = x[e], r.v[u][e] = y[e];
      } else {
        const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rk, code_at, 0, 0), y = __builtin_amdgcn_raw_buffer_load_b64(rv, code_at, 0, 0);
#pragma unroll
        for (int e = 0; e < W; ++e) r.k[u][e] = x[e], r.v[u][e] = y[e];
      }
      r.ks[u] = __builtin_amdgcn_raw_buffer_load_b8(rks, ks_at, 0, 0);
      r.vs[u] = __builtin_amdgcn_raw_buffer_load_b32(rvs, vs_at, 0, 0);
    }
  };

  // Query rows as the B operand: lane (g, j) holds head j's dims [g*D/4 + 8kk, +8).
  bf16x8 q[NK];
  {
    const bool has = j < p.group;
    const uint16_t* row = p.q + ((int64_t)b * p.q_heads + (int64_t)h * p.group + (has ? j : 0)) * D + g * (D / 4);
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(row + 8 * kk);
      q[kk] = __builtin_bit_cast(bf16x8, has ? x : u32x4{0u, 0u, 0u, 0u});
    }
  }
  float m = -INFINITY, l = 0.f;  // of head j; l of this lane's tokens
  f32x4 acc[NT];                 // lane (g, j): head j, dims (4g + r)*D/16 + n
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](int tile, Tile<D>& r) {
    // Tokens of this tile; fewer than 64 only at the piece's end.
    const int blk0 = first + tile * (kTile * kWaves);
    const int valid = min(seq, c1 * kBlockTokens) - blk0 * kBlockTokens;
    const bool part = valid < kTile * kBlockTokens;
    float sv[kTile][4];
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      const float scale = mx_scale(r.ks[u]);
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        const u32x4 kb = mx_values(r.k[u][kk], scale);
        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kb), q[kk], x, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[u][i] = x[i] * p.scale;
    }
    if (part) {
      // Tokens past the end: no score, and zeros for values that may be NaN.
#pragma unroll
      for (int u = 0; u < kTile; ++u) {
        const int mine = min(max(valid - kBlockTokens * u - 4 * g, 0), 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i >= mine) sv[u][i] = -INFINITY;
        const uint32_t keep = mine == 4 ? 0xffffffffu : (1u << 8 * mine) - 1u;
        r.vs[u] &= keep;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if constexpr (D == 128) r.v[u][e] = e < mine ? r.v[u][e] : 0u;
          else r.v[u][e] = 2 * e + 2 <= mine ? r.v[u][e] : 2 * e < mine ? r.v[u][e] & 0xffffu : 0u;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kTile; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, sv[u][i]);
    const float mn = fmaxf(m, group_max4(top));
    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    uint32_t pb[kTile][2];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        // a token past the end gets 0, or NaN where its head has no other score
        // than -infinity or NaN and is NaN whatever this token adds
        const float a = __builtin_amdgcn_exp2f(sv[u][i] - mn), c = __builtin_amdgcn_exp2f(sv[u][i + 1] - mn);
        const uint32_t pair = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, c}), mx_bf16x2));
        pb[u][i / 2] = pair;
        sum += bf16_lo(pair) + bf16_hi(pair);
      }
    }
    l = l * alpha + sum;
    m = mn;
    if (__ballot(alpha != 1.f) != 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] *= alpha;
    }
#pragma unroll
    for (int u = 0; u < kTile; u += 2) {
      const bf16x8 pv = __builtin_bit_cast(bf16x8, u32x4{pb[u][0], pb[u][1], pb[u + 1][0], pb[u + 1][1]});
      uint32_t c[2][4][W];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        token_pairs<D, 0>(r.v[u + x], r.vs[u + x], c[x][0]);
        token_pairs<D, 1>(r.v[u + x], r.vs[u + x], c[x][1]);
        token_pairs<D, 2>(r.v[u + x], r.vs[u + x], c[x][2]);
        token_pairs<D, 3>(r.v[u + x], r.vs[u + x], c[x][3]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t pick = n % 2 ? 0x07060302u : 0x05040100u;  // the upper or the lower halves of two words
        u32x4 a;
#pragma unroll
        for (int x = 0; x < 4; ++x) a[x] = __builtin_amdgcn_perm(c[x / 2][2 * (x % 2) + 1][n / 2], c[x / 2][2 * (x % 2)][n / 2], pick);
        acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), pv, acc[n], 0, 0, 0);
      }
    }
  };

  Tile<D> r;
  for (int tile = 0; first + tile * (kTile * kWaves) < c1; ++tile) {
    load(tile, r);
    compute(tile, r);
  }

  // The waves' results into one: lane (g, j) holds head j.
  l = group_sum4(l);
  if (g == 0) {
    lds_m[w][j] = m;
    lds_l[w][j] = bad ? __builtin_nanf("") : l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < NT; n += 4)
      *reinterpret_cast<f32x4*>(&lds_o[w][j][(4 * g + i) * (D / 16) + n]) = f32x4{acc[n][i], acc[n + 1][i], acc[n + 2][i], acc[n + 3][i]};
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
    hipLaunchKernelGGL((paged_decode_mxfp4_kernel<D>), dim3(p.kv_heads, p.splits, q.batch), dim3(kThreads), 0, stream, q);
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
