// Decode reader of MXFP4 pages: paged attention for one query token per
// sequence. score = (q . k) * log2(e)/sqrt(D), online softmax in base 2,
// output = sum(p v) / sum(p) in BF16.
//
// A workgroup of four waves reads one piece of a sequence for one KV head, its
// waves tiles of two blocks (32 tokens) in turn.
//  - loads: a block's codes of one head lie in the order of the lanes that
//    take them, so one load instruction reads all of K, and one all of V. The
//    next tile's K is asked for when the scores have used this one's, its V
//    after the values' products.
//  - scores, transposed: lane (g, i) holds key i's dims of quarter g, which the
//    scaled converters make BF16 of, exactly; each MFMA takes eight of every quarter
//    (A) and the same of the query heads of the KV head (B, columns), as they are.
//    So terms are exact and sums those of the BF16 MFMA, FP32 (measured: within
//    2^-22 of the terms' magnitudes). The scaled MFMA, which would take the codes as
//    they are, wants the queries in eight bits or less and sums terms of unlike
//    size within 2^-12 alone (measured). Lane (g, j) ends with tokens 4g..4g+3 of
//    head j.
//  - softmax: every weight is 2^((score - largest) * scale), of the difference, so the
//    largest score's is 1 however large it is. (The score times the scale less the
//    largest's, in one multiply-add, is off by the rounding of that product.)
//  - values: lane (g, i) holds tokens 4g..4g+3 of column i, the D/16 dims
//    [i*D/16, (i+1)*D/16). The scaled converters make a BF16 pair of a byte, an
//    even and an odd dim of one token, exactly. Both count as terms of one
//    contraction: A row i, of MFMA n, holds dims 2n and 2n + 1 of column i for
//    four tokens a lane, B the probability against the even dims in the
//    columns of heads 0..7 and against the odd ones in columns 8..15 (which
//    carry the same heads again), zero elsewhere. So no two tokens have to be
//    put side by side and no column of B is idle. More than 8 query heads take
//    two such products, of the even and of the odd dims.
//  - pieces: a batch's blocks are cut into pieces of at most c blocks, even within
//    a sequence, about as many as fill the chip, whatever the sequences' lengths:
//    those are device memory, so every workgroup finds c and its piece
//    from them (find_piece). The workgroup of a sequence's and KV head's that
//    finishes last joins their results, in their order; they are written and
//    read at agent scope (written through, read past the XCD's own L2), so no
//    L2 is written back: a workgroup waits for its stores, then takes a ticket.
//  - a probability goes into that product as two BF16 numbers, its top eight bits
//    and the next eight, within 2^-15 of the FP32 one; the sum they are divided by is
//    of the FP32 ones. With one BF16 number each, the outputs of 64 x 5,040 tokens lay
//    0.0014 of their norm from those of FP32 weights, now 0.0001 (rounding them to
//    BF16 takes 0.0016).
//
// Bound by the pages' bytes and the conversions and products of each block, side by
// side, and for few blocks by the chain of dependent reads (arguments, lengths, ids,
// pages, ticket, results). Calls back to back in a graph, on pages that stay and so
// lie partly in the memory-side cache / on 2 GB of pages in turn: 64 x 5,040 tokens
// of 2 x 128 19.4 / 22.6 us (4.5 / 3.9 TB/s of the bytes needed); 64 mixed up to
// 32,768 of 4 x 128 34.1 / 41.0 us (4.7 / 3.9); 1 x 5,040 of 2 x 64 7.9 us either
// way. Of the first, on pages that stay, calls that end after each part take: launch
// 2.6, its piece found 2.6, all but the tiles and the join 4.4, all but the join 18.0.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "arrival.h"
#include "decode_mxfp4_kernels.h"
#include "mxfp4_device.h"
#include "xcd_order.h"  // kXcds

namespace pbe {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
// Below, in us, on pages that stay: A 64 x 5,040 tokens of 2 x 128, B 64 mixed up to
// 32,768 of 4 x 128, C 150 mixed up to 3,000 of 2 x 64, D 256 mixed up to 600 of 4 x
// 128. As it is: 19.8 / 34.3 / 13.7 / 15.7.
// Blocks of a wave's tile. A / B / C / D with tiles of 1: 21.3 / 37.5 / 14.4 / 16.9,
// of 4 (registers spill): 20.7 / 36.3 / 13.6 / 17.9. Half the workgroups of eight
// waves: 19.8 / 39.5 / 15.7 / 19.9.
constexpr int kTile = 2;
// Blocks of a piece that joining is worth: two tiles for every wave. With one, 64
// mixed up to 250 of 2 x 128 took 6.5 us for 4.9, 8 mixed up to 2,000 of 8 x 128
// 8.9 for 8.1, 1 x 600 of 2 x 128 6.7 for 7.4, A to D the same. Pieces are made even
// after that, so that those of a sequence little longer hold little more than half.
constexpr int kMinChunk = 2 * kTile * kWaves;
// Wanted workgroups per compute unit. A / B / C / D with 1: 21.1 / 39.7 / 15.7 /
// 15.8, 3: 22.3 / 38.1 / 15.2 / 20.2.
constexpr int kPiecesPerUnit = 2;
constexpr int kAgent = 0x10;  // buffer access policy: agent scope
static_assert(kMxDecodeMaxSplits < (1 << kTicketBits), "arrivals fit the ticket");

// ---- which blocks a workgroup reads ----
struct Piece {
  int b = -1;       // sequence; -1: none for this workgroup
  int seq = 0;      // its length
  int s = 0, k = 1; // which of the sequence's pieces, and how many it has
  int c = 0;        // blocks of each but the last
};

// Piece z of the batch. c is the total over the pieces that are wanted, or what
// fits the workspace: with `most` pieces to hold, sum of ceil(n / c) <= total /
// c + batch <= most for c >= total / (most - batch).
__device__ __forceinline__ Piece find_piece(const Mxfp4DecodeParams& p, int z, int lane) {
  Piece r;
  if (p.most == p.batch) {  // every sequence whole
    if (z >= p.batch) return r;
    r.b = z;
    r.seq = p.seq_lens[z];
    r.c = p.max_blocks;
    return r;
  }
  constexpr int kKept = 4;  // sequences of a lane that stay in registers
  int seqs[kKept], sum = 0, longest = 0;
  for (int i0 = 0; i0 < p.batch; i0 += 64 * kKept) {
    int now[kKept];
#pragma unroll
    for (int i = 0; i < kKept; ++i) now[i] = i0 + 64 * i + lane < p.batch ? p.seq_lens[i0 + 64 * i + lane] : 0;
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int n = blocks_of(now[i], p.max_blocks);
      sum += n;
      longest = max(longest, n);
      if (i0 == 0) seqs[i] = now[i];
    }
  }
  const uint32_t total = (uint32_t)__builtin_amdgcn_readlane(wave_scan(sum), 63);
  const uint32_t wanted = max((uint32_t)p.min_chunk, (total + p.wanted - 1) / p.wanted);
  const uint32_t held = (uint32_t)(p.most - p.batch), fits = (total + held - 1) / held;
  // Joining takes a workgroup about 1.3 times as long for a piece as reading
  // takes it for a block: for n blocks in pieces of c, c + 1.3 n / c is least at
  // c = sqrt(1.3 n).
  const uint32_t n = (uint32_t)wave_max_int(longest);
  const uint32_t joined = max((uint32_t)__builtin_amdgcn_sqrtf(1.3f * (float)n), (n + kMxDecodeMaxSplits - 1) / kMxDecodeMaxSplits);
  const uint32_t c = max(max(wanted, fits), joined);
  int before = 0;
  for (int i = 0; i < p.batch; i += 64) {
    int seq = seqs[0];
#pragma unroll
    for (int e = 1; e < kKept; ++e) seq = i == 64 * e ? seqs[e] : seq;
    if (i >= 64 * kKept) seq = i + lane < p.batch ? p.seq_lens[i + lane] : 0;
    const int k = i + lane < p.batch ? max(1, (int)(((uint32_t)blocks_of(seq, p.max_blocks) + c - 1) / c)) : 0;
    const int upto = wave_scan(k) + before;
    const uint64_t past = __ballot(upto > z);
    if (past) {
      const int at = __builtin_ctzll(past);
      r.b = i + at;
      r.seq = __builtin_amdgcn_readlane(seq, at);
      r.k = __builtin_amdgcn_readlane(k, at);
      r.s = z - (__builtin_amdgcn_readlane(upto, at) - r.k);
      // even pieces, of which the sequence may need fewer
      const uint32_t n = (uint32_t)max(1, __builtin_amdgcn_readlane(blocks_of(seq, p.max_blocks), at));
      r.c = (int)((n + (uint32_t)r.k - 1) / (uint32_t)r.k);
      r.k = (int)((n + (uint32_t)r.c - 1) / (uint32_t)r.c);
      if (r.s >= r.k) r.b = -1;
      return r;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return r;
}

// A lane's part of one tile.
template <int D>
struct Tile {
  static constexpr int W = D / 32;  // words of codes
  uint32_t k[kTile][W], v[kTile][W];
  uint32_t ks[kTile];  // scale bytes of its quarter, of four keys
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

// kWide: more than 8 query heads per KV head. The wide form holds for any number
// of them, in 156 registers and three waves a SIMD for 122 and four; for up to
// eight it takes, A / B / C / D above, 22.8 / 40.6 / 15.1 / 20.5 us.
template <int D, bool kWide>
__global__ __launch_bounds__(kThreads, kWide ? 3 : 4) void paged_decode_mxfp4_kernel(const Mxfp4DecodeParams p) {
  constexpr int W = D / 32;                  // words of K (and of V) codes per lane and block
  constexpr int NT = D / 32;                 // value MFMAs per block (of each parity, kWide)
  constexpr int PARTS = kWide ? 2 : 1;       // accumulators: both parities in one, or even and odd
  constexpr int STEP = kTile * kWaves;       // blocks from a wave's tile to its next
  constexpr int AHEAD = 64 / kTile;          // tiles whose ids a window holds
  constexpr int HEADS = kWide ? 16 : 8;
  constexpr int PITCH = D + 4;
  __shared__ __attribute__((aligned(16))) float lds_o[kWaves][HEADS][PITCH];
  __shared__ float lds_m[kWaves][16], lds_l[kWaves][16];
  __shared__ int lds_last;

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  // A piece's KV heads go to one XCD, eight pieces side by side: two to four heads'
  // scales share a cache line, which several XCDs would read each for itself (64
  // x 5,040 tokens of 2 x 128 fetch 90.6 MB of the 88.2 that they need, in the order
  // of the heads 96.0; 19.4 us and 20.9).
  const int eight = (int)fast_div(blockIdx.x, p.by_eight), in_eight = (int)blockIdx.x - eight * (int)p.by_eight.d;
  const int z = eight * (int)kXcds + in_eight % (int)kXcds, h = in_eight / (int)kXcds;
  const Piece piece = find_piece(p, z, lane);
  if (piece.b < 0) return;
  const int b = piece.b, seq = piece.seq, s = piece.s, pieces = piece.k;
  const int nblk = seq > 0 ? (int)(((uint32_t)seq + kBlockTokens - 1) / kBlockTokens) : 0;
  bool bad = seq < 0 || nblk > p.max_blocks;  // then it has one piece
  const int c0 = s * piece.c, first = c0 + w * kTile;
  const int c1 = bad ? c0 : min(c0 + piece.c, nblk);
  const int tiles = c1 > first ? (c1 - first + STEP - 1) / STEP : 0;  // of this wave
  const int32_t* table = p.tables + (int64_t)b * p.max_blocks;
  auto ids_of = [&](int tile) { return table[min(first + (tile + lane / kTile) * STEP + lane % kTile, p.max_blocks - 1)]; };
  int32_t window = ids_of(0);
  // B of the scores: lane (g, j) holds head j's dims of quarter g, as the keys lie.
  // Asked for before the first tile, as loads come back in their order; every wave
  // reads its own, which took no longer than one reading for all of them.
  const int64_t row0 = (int64_t)b * p.q_heads + (int64_t)h * p.group;  // the KV head's first query head
  const int head = kWide ? j : j % 8;
  u32x4 q[W];
#pragma unroll
  for (int n = 0; n < W; ++n)
    q[n] = *reinterpret_cast<const u32x4*>(p.q + (row0 + min(head, p.group - 1)) * D + g * (D / 4) + 8 * n);

  // Lane l holds the id of block l % kTile of the wave's tile l / kTile of
  // AHEAD; -1 for one past the piece's end, or outside the pools.
  auto check_ids = [&](int tile) {
    const bool mine = first + (tile + lane / kTile) * STEP + lane % kTile < c1, ok = window >= 0 && window < p.blocks;
    if (__ballot(mine && !ok) != 0) bad = true;
    window = mine && ok ? window : -1;
  };
  check_ids(0);
  const uint32_t code_at = lane * (D / 8);
  // A turn by ks_turn takes key j's scale byte to the exponent's bits.
  const uint32_t key_scales_at = (D == 128 ? g : g / 2) * kMxTokens + (j & ~3), ks_turn = 8 * (j & 3) + 9;
  const uint32_t value_scales_at = (D == 128 ? j / 4 : j / 8) * kMxTokens + 4 * g;
  // Where a tile's blocks lie: bytes of codes from a pool's start, a 16th of
  // that of scales. A block that is none is read from the pools' first: what a
  // tile holds past the piece's end is not used, and a bad id makes NaN.
  gptr<const uint8_t> k_codes = (gptr<const uint8_t>)p.key_pool + (uint32_t)h * mx_head_bytes(D);
  gptr<const uint8_t> v_codes = (gptr<const uint8_t>)p.value_pool + (uint32_t)h * mx_head_bytes(D);
  gptr<const uint8_t> k_scales = (gptr<const uint8_t>)p.key_scales + (uint32_t)h * mx_head_scales(D);
  gptr<const uint8_t> v_scales = (gptr<const uint8_t>)p.value_scales + (uint32_t)h * mx_head_scales(D);
  uint64_t from[kTile];
  auto find = [&](int tile) {
#pragma unroll
    for (int u = 0; u < kTile; ++u)
      from[u] = (uint64_t)(uint32_t)max(__builtin_amdgcn_readlane(window, (tile % AHEAD) * kTile + u), 0) * p.half;
  };
  auto codes = [&](gptr<const uint8_t> at, uint32_t (&words)[W]) {
    if constexpr (D == 128) {
      const u32x4 x = *(gptr<const u32x4>)at;
#pragma unroll
      for (int e = 0; e < W; ++e) words[e] = x[e];
    } else {
      const u32x2 x = *(gptr<const u32x2>)at;
#pragma unroll
      for (int e = 0; e < W; ++e) words[e] = x[e];
    }
  };
  // A block's address stays scalar, hidden from the compiler, which would add the
  // lane's offset to the pool's address once and the block's to that with 64-bit
  // vector additions.
  auto block_at = [&](gptr<const uint8_t> pool, uint64_t offset) {
    gptr<const uint8_t> at = pool + offset;
    asm volatile("" : "+s"(at));
    return at;
  };
  auto load_keys = [&](Tile<D>& r) {
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      codes(block_at(k_codes, from[u]) + code_at, r.k[u]);
      r.ks[u] = *(gptr<const uint32_t>)(block_at(k_scales, from[u] / 16) + key_scales_at);
    }
  };
  auto load_values = [&](Tile<D>& r) {
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      codes(block_at(v_codes, from[u]) + code_at, r.v[u]);
      r.vs[u] = *(gptr<const uint32_t>)(block_at(v_scales, from[u] / 16) + value_scales_at);
    }
  };

  Tile<D> r;
  find(0);
  if (tiles > 0) {
    load_keys(r);
    load_values(r);
  }
  const int z0 = z - s;  // the sequence's first piece
  const gptr<uint64_t> ticket = (gptr<uint64_t>)p.tickets + (int64_t)z0 * p.kv_heads + h;
  if (pieces > 1 && threadIdx.x == 0) open_ticket(ticket, p.tag);
  if (head >= p.group) {
#pragma unroll
    for (int n = 0; n < W; ++n) q[n] = u32x4{0u, 0u, 0u, 0u};
  }
  // The upper bytes of a probability's part, in the half of a BF16 pair that meets
  // this lane's column, and zeros in the other.
  const uint32_t to_mine = kWide || j >= 8 ? 0x03020c0cu : 0x0c0c0302u;

  float m = -INFINITY, l = 0.f;  // of head j: its largest score, and the sum of this lane's probabilities
  f32x4 acc[PARTS][NT];
#pragma unroll
  for (int x = 0; x < PARTS; ++x)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[x][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  // One tile. kNext: another one follows; kPart: fewer than all of its tokens count.
  auto compute = [&](int tile, auto next, auto part) {
    constexpr bool kNext = decltype(next)::value, kPart = decltype(part)::value;
    if (kNext && (tile + 1) % AHEAD == 0) {
      window = ids_of(tile + 1);
      check_ids(tile + 1);
    }
    // of tokens up to 2^31, counted without a sign
    const int valid = kPart ? (int)(min((uint32_t)seq, (uint32_t)c1 * kBlockTokens) - (uint32_t)(first + tile * STEP) * kBlockTokens) : 0;
    f32x4 x[kTile];
#pragma unroll
    for (int u = 0; u < kTile; ++u) {
      const float ks = __uint_as_float(__builtin_amdgcn_alignbit(r.ks[u], r.ks[u], ks_turn));  // the converters read the exponent bits alone
      x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < W; ++n)
        x[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, mx_values(r.k[u][n], ks)), __builtin_bit_cast(bf16x8, q[n]), x[u], 0, 0, 0);
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
    }
    if constexpr (kNext) {
      __builtin_amdgcn_sched_barrier(0);  // into the registers that the scores have read
      find(tile + 1);
      load_keys(r);
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kTile; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, x[u][i]);
    const float mn = fmaxf(m, group_max4(top));
    // While all scores are -infinity (they may pass FP32's range) the weights are
    // zeros, not 2^(infinity - infinity): a later tile, wave or piece can have others.
    const float base = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f((m - base) * p.scale);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kTile; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[u][i] = __builtin_amdgcn_exp2f((x[u][i] - base) * p.scale);
        sum += x[u][i];
      }
    m = mn;
    l = l * alpha + sum;
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
      // hi keeps a probability's top eight significant bits, lo the next eight.
      u32x4 hi, lo, hi_even, lo_even;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t e = __float_as_uint(x[u][i]);
        const uint32_t rest = __float_as_uint(x[u][i] - __uint_as_float(e & 0xffff0000u));
        hi[i] = __builtin_amdgcn_perm(e, e, to_mine);
        lo[i] = __builtin_amdgcn_perm(rest, rest, to_mine);
        if constexpr (kWide) hi_even[i] = e >> 16, lo_even[i] = rest >> 16;
      }
      // All products of hi before those of lo, so that none waits for the one before
      // it (64 x 5,040 tokens of 2 x 128: 19.0 us, next to each other 20.6).
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bf16x8 a = __builtin_bit_cast(bf16x8, u32x4{c[0][n], c[1][n], c[2][n], c[3][n]});
          acc[0][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, part ? lo : hi), acc[0][n], 0, 0, 0);
          if constexpr (kWide)
            acc[PARTS - 1][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, part ? lo_even : hi_even), acc[PARTS - 1][n], 0, 0, 0);
        }
    }
    if constexpr (kNext) load_values(r);
  };

  // Only the piece's last tile can be a partial one.
  const bool cut = tiles > 0 && min((uint32_t)seq, (uint32_t)c1 * kBlockTokens) < (uint32_t)(first + (tiles - 1) * STEP + kTile) * kBlockTokens;
  const std::true_type yes;
  const std::false_type no;
  for (int tile = 0; tile < tiles - 1; ++tile) compute(tile, yes, no);
  if (cut) compute(tiles - 1, no, yes);
  else if (tiles > 0) compute(tiles - 1, no, no);

  // The waves' results into one. Lane (g, j) holds dims (4g + r)*D/16 + 2n + (its parity).
  l = group_sum4(l);
  if (g == 0) {  // lanes j and j + 8 hold the same
    lds_m[w][head] = m;
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
  // From here on a thread holds four dims of a head, more than one after another
  // where the heads have more dims than the workgroup threads. Of tokens that all
  // score -infinity there is no softmax.
  auto finish = [&](int hj, int col, const f32x4& o, float sum) {
    uint16_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = to_bf16(sum != sum ? sum : sum > 0.f ? o[i] / sum : seq > 0 ? __builtin_nanf("") : 0.f);
    *reinterpret_cast<u32x2*>(p.out + (row0 + hj) * D + 4 * col) = u32x2{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16};
  };
  // The sequence's partial results [piece][query head]; a piece's bytes times
  // 1,024 fit 31 bits.
  const uint32_t acc_pitch = (uint32_t)p.q_heads * (D * 4), ml_pitch = (uint32_t)p.q_heads * 8;
  const __amdgpu_buffer_rsrc_t r_acc = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p.part_acc + (int64_t)z0 * p.q_heads * D), (short)0, pieces > 1 ? (uint32_t)pieces * acc_pitch : 0, 0x00020000);
  const __amdgpu_buffer_rsrc_t r_ml = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p.part_ml + (int64_t)z0 * p.q_heads * 2), (short)0, pieces > 1 ? (uint32_t)pieces * ml_pitch : 0, 0x00020000);
  const uint32_t head0 = (uint32_t)(h * p.group);
  for (int unit = threadIdx.x; unit < p.group * (D / 4); unit += kThreads) {
    const int hj = unit / (D / 4), col = unit % (D / 4);
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, lds_m[i][hj]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float li = lds_l[i][hj], wt = li > 0.f ? __builtin_amdgcn_exp2f((lds_m[i][hj] - top) * p.scale) : 0.f;
      sum += li != li ? li : li * wt;
      if (wt > 0.f) o += *reinterpret_cast<const f32x4*>(&lds_o[i][hj][4 * col]) * wt;
    }
    if (pieces == 1) {
      finish(hj, col, o, sum);
    } else {
      const uint32_t head = head0 + hj;
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), r_acc, s * acc_pitch + head * (D * 4) + 16 * col, 0, kAgent);
      if (col == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{top, sum}), r_ml, s * ml_pitch + head * 8, 0, kAgent);
    }
  }
  if (pieces == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's results have been written
  __syncthreads();
  if (threadIdx.x == 0) lds_last = last_arrival(ticket, p.tag, (uint32_t)pieces);
  __syncthreads();
  if (!__builtin_amdgcn_readfirstlane(lds_last)) return;
  auto join = [&](auto in_flight) {
    constexpr int kJoin = decltype(in_flight)::value;
    for (int unit = threadIdx.x; unit < p.group * (D / 4); unit += kThreads) {
      const int hj = unit / (D / 4), col = unit % (D / 4);
      float top = -INFINITY, sum = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      for (int s0 = 0; s0 < pieces; s0 += kJoin) {
        f32x2 ml[kJoin];
        f32x4 x[kJoin];
#pragma unroll
        for (int i = 0; i < kJoin; ++i) {  // past the end: nothing read
          const uint32_t at = (uint32_t)min(s0 + i, pieces), head = head0 + hj;
          ml[i] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(r_ml, at * ml_pitch + head * 8, 0, kAgent));
          x[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r_acc, at * acc_pitch + head * (D * 4) + 16 * col, 0, kAgent));
        }
        float mn = top;
#pragma unroll
        for (int i = 0; i < kJoin; ++i) mn = fmaxf(mn, s0 + i < pieces ? ml[i][0] : -INFINITY);
        const float keep = sum > 0.f ? __builtin_amdgcn_exp2f((top - mn) * p.scale) : 0.f;
        sum = sum != sum ? sum : sum * keep;
        o = keep > 0.f ? o * keep : f32x4{0.f, 0.f, 0.f, 0.f};
        top = mn;
#pragma unroll
        for (int i = 0; i < kJoin; ++i) {  // a NaN sum stays; a result of weight 0 is left out whatever it holds
          const float li = ml[i][1], wt = li > 0.f ? __builtin_amdgcn_exp2f((ml[i][0] - mn) * p.scale) : 0.f;
          sum += li != li ? li : li * wt;
          if (wt > 0.f) o += x[i] * wt;
        }
      }
      finish(hj, col, o, sum);
    }
  };
  // Few results want few loads, many want them together. Always 16: 64 x 5,040 of
  // 2 x 128 20.9 us for 19.8, 1 x 600 8.1 for 7.4. Always 4: 1 x 32,768 of 4 x 128
  // 16.9 us for 15.4, 1 x 5,040 of 2 x 64 8.6 for 7.9.
  if (pieces <= 4) join(std::integral_constant<int, 4>{});
  else join(std::integral_constant<int, 16>{});
}

template <int D>
hipError_t launch(const Mxfp4DecodeParams& p, int64_t pieces, hipStream_t stream) {
  const dim3 grid((unsigned)((pieces + kXcds - 1) / kXcds * kXcds * p.kv_heads));
  if (p.group > 8) hipLaunchKernelGGL((paged_decode_mxfp4_kernel<D, true>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((paged_decode_mxfp4_kernel<D, false>), grid, dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

// Pieces that fill the chip, of the whole batch.
int64_t wanted_pieces(int32_t kv_heads, int64_t compute_units) { return std::max<int64_t>(1, kPiecesPerUnit * compute_units / kv_heads); }
// Pieces that a sequence of max_blocks blocks can be cut into: tables may be as wide as 2^31 - 1.
int64_t most_pieces(int32_t max_blocks) { return ((int64_t)max_blocks + kMinChunk - 1) / kMinChunk; }

}  // namespace

int32_t mxfp4_decode_splits(int32_t batch, int32_t kv_heads, int32_t max_blocks, int64_t compute_units) {
  // Room for the wanted pieces and one more of each sequence, which a cut of
  // unequal lengths can take; no sequence has more than its shortest pieces.
  // Many whole sequences fill the chip by themselves, with no piece to find and
  // none to join: 1,024 mixed sequences of 4 KV heads, the fewest that 256 compute
  // units take whole, up to 600 tokens 38.5 us, in pieces 54.7; up to 4,000 203
  // and 214.
  if ((int64_t)batch * kv_heads >= 16 * compute_units) return 1;
  const int64_t pieces = wanted_pieces(kv_heads, compute_units) + batch, most = most_pieces(max_blocks);
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>({(pieces + batch - 1) / batch, most, kMxDecodeMaxSplits}));
}

uint64_t mxfp4_decode_workspace_bytes(int32_t batch, int32_t q_heads, int32_t dim, int32_t splits) {
  if (splits <= 1) return 0;
  // a ticket a piece and KV head, of which there are no more than query heads
  return (uint64_t)batch * q_heads * splits * ((uint64_t)(dim + 2) * 4 + 8);
}

hipError_t launch_paged_decode_mxfp4(Mxfp4DecodeParams p, int dim, int32_t splits, void* workspace, int64_t compute_units, hipStream_t stream) {
  // A launch takes fewer than 2^32 threads: a batch of more workgroups is read in
  // parts, one after another on the stream, in the same workspace.
  const int64_t limit = 0xffffffffll / kThreads / p.kv_heads / kXcds * kXcds;
  if (limit < 2) return hipErrorInvalidConfiguration;
  const int32_t batch = p.batch;
  // Totals of blocks are 32-bit sums, a sequence's results are addressed with 31 bits.
  if ((int64_t)batch * p.max_blocks > INT32_MAX || (int64_t)p.q_heads * dim * 4 * kMxDecodeMaxSplits > INT32_MAX) splits = 1;
  const int64_t wanted = wanted_pieces(p.kv_heads, compute_units);
  const int64_t part = splits > 1 ? std::max<int64_t>(1, limit - wanted) : limit;
  for (int64_t first = 0; first < batch; first += part) {
    Mxfp4DecodeParams q = p;
    q.batch = (int32_t)std::min<int64_t>(part, batch - first);
    q.seq_lens += first;
    q.tables += first * p.max_blocks;
    q.q += first * p.q_heads * dim;
    q.out += first * p.q_heads * dim;
    const int64_t each = std::min<int64_t>(splits, most_pieces(p.max_blocks));
    const int64_t pieces = std::min<int64_t>({(int64_t)q.batch * each, wanted + q.batch, limit});
    q.most = (int32_t)pieces;
    q.wanted = (uint32_t)wanted;
    q.min_chunk = kMinChunk;
    q.by_eight = make_fast_div(kXcds * (uint32_t)p.kv_heads);
    if (pieces > q.batch) {
      q.part_acc = static_cast<float*>(workspace);
      q.part_ml = q.part_acc + (uint64_t)pieces * p.q_heads * dim;
      q.tickets = reinterpret_cast<uint64_t*>(q.part_ml + (uint64_t)pieces * p.q_heads * 2);
      q.tag = decode_tag();
    }
    const hipError_t e = dim == 128 ? launch<128>(q, pieces, stream) : dim == 64 ? launch<64>(q, pieces, stream) : hipErrorInvalidValue;
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace pbe
