// Prompt reader: causal attention of many query tokens a sequence over its keys.
//
// o = sum_j w_j v_j / sum_j w_j, w_j = 2^((q . k_j - m) * scale), scale = log2(e) /
// sqrt(D), over the keys that a query sees; one pass over the keys, m and the sums
// held in FP32. The query heads that share a KV head are stacked: row r of a sequence
// is token r / group, head r % group, so K and V are read once for all of them, and a
// single query of a large group still fills a wave's 32 columns.
//
// A wave has 32 rows and computes S^T = K Q^T and O^T += V^T W^T with the 32x32x16
// BF16 MFMA. Transposed, because a lane then holds one row's scores (32 of a tile's 64,
// its other half in lane + 32): maximum and sum need no exchange but one swap of
// halves, and the scores' registers are the weights' operand as they are, without LDS.
// V comes as the A operand by LDS reads that transpose; Q stays in registers.
//
// Bound: MFMA, 4 * D FLOP a row and seen key. 4 * 128 dims take 32 products of 8
// passes each a wave and tile, beside about 400 instructions for 64 weights a lane pair.
// Over 8,192 tokens of 28 heads of 128 dims, back to back in a graph: 455 to 497 us by GPU
// (one GPU repeats itself within 1%), 969 to 1,058 TFLOP/s, of the 1,387 that a large
// matrix product reaches; MFMA busy 49% at 2.05 GHz (the clock falls as the kernel gets
// faster). A SIMD's two waves share a barrier a
// tile and mostly multiply, and mostly weigh, at the same time. Leaving out the
// exponentials, or the maxima, or the sums, takes 6 to 9% off (on the way there, of 526
// us): no single part is the bound.
// What that took, in us, each measured against the one before: 128 rows a workgroup 526;
// special values (see there) looked for in masked tiles only, in place 507; reads some
// products ahead and one multiply-add before each exponential 485; 256 rows 469; no bank
// conflicts 462.
// Tried and slower: 64 rows a wave, operands from LDS used twice, one half's softmax
// beside the other's products (554 for 469: with 478 registers the compiler moves operands
// between the files before most products), the next tile's scores among this one's
// weights in one wave (510 for 469), the workgroup's halves taking turns (507 for 462),
// three tiles in LDS (503 for 469), V's loads after all of K's (500 for 467). Waves'
// priorities changed nothing.
//
// A weight goes into its product as one BF16 number, off by at most 2^-8 of itself (two
// numbers each would double the second product's MFMA). Over rows, BF16 and MXFP4 pages
// the sum is that of the rounded weights, so a row's outputs are a mean of its values
// all the same, and constant values come back exactly. Over FP8 pages the value's scale
// goes into the weight before the rounding, and the sum is of those before.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "decode_device.h"
#include "mxfp4_device.h"
#include "prompt_kernels.h"
#include "prompt_order.h"

namespace pbe {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

#define PBE_LDS __attribute__((address_space(3)))

constexpr int kKeys = 64;         // keys of a tile
// Key tiles that a part has at least, on the average: a part's start, end and share of
// the join cost about as much as four of its tiles. 64 x 4 drafted tokens over FP8
// pages: 44.0 us with 4, 46.3 with 8.
constexpr int kPiece = 4;
constexpr int kEdge = 4;          // key tiles of a tile that is cut before and behind the cuts
constexpr int kMaxCuts = 4096;    // parts at most, so also cuts of a tile
// How far (in base 2) scores may pass the maximum that weights refer to. Weights of up
// to 2^8 lose nothing in BF16 or FP32, and after a row's first tiles sums are scaled
// hardly ever.
constexpr float kLazy = 8.f;
// Maxima (in base 2) beyond which weights come from the scores' differences: below, the
// rounding of maximum * scale is at most 2^-14 and the same for all of a row's weights.
constexpr float kFar = 1024.f;
constexpr int kXcds = 8;
static_assert(kBlockTokens == 16, "a key tile is four blocks");

// ---- which rows and keys a workgroup has ----
struct Seq {
  int begin = 0, rows = 0;  // first row of q, tokens (those within n_q)
  int first = 0, len = 0;   // first row of k (rows), keys
  int tiles = 0;
  bool bad = false;         // starts or length make no sense
  // What tile t costs, in sixteenths of a key: base + step * (t + 1). A model: it
  // only has to be the same for all workgroups.
  int64_t base = 0, step = 0;
  __device__ __forceinline__ int64_t cost(int t) const { return base + step * (t + 1); }
  __device__ __forceinline__ int64_t before(int64_t t) const { return base * t + step * (t * (t + 1) / 2); }
};

constexpr int64_t kTileCost = 16 * 2 * kKeys;  // of a tile's start and end

template <KeyKind kKind, int kRows>
__device__ __forceinline__ Seq seq_of(const PromptParams& p, int b) {
  Seq u;
  const int lo = p.q_starts[b], hi = p.q_starts[b + 1];
  u.begin = min(max(lo, 0), p.n_q);
  u.bad = lo < 0 || hi < lo || hi > p.n_q;
  u.rows = max(0, min(hi, p.n_q) - u.begin);
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
  u.tiles = (int)(((uint32_t)u.rows * (uint32_t)p.group + kRows - 1) / kRows);
  u.base = kTileCost + 16 * (int64_t)max(0, u.len - u.rows);
  u.step = u.len ? p.step : 0;
  return u;
}

__device__ __forceinline__ int key_tiles(int len) { return (int)(((uint32_t)len + kKeys - 1) / kKeys); }

// Row r of a sequence's, tokens times query heads of a KV head: its token (rows
// behind the last: the last one's), and the keys that a token sees.
__device__ __forceinline__ int token_of(const PromptParams& p, const Seq& u, int r) {
  return (int)fast_div((uint32_t)min(r, u.rows * p.group - 1), p.by_group);
}
__device__ __forceinline__ int seen_by(const Seq& u, int token) { return max(0, u.len - u.rows + token + 1); }
template <int kRows>
__device__ __forceinline__ int tiles_seen(const PromptParams& p, const Seq& u, int t) {
  return key_tiles(seen_by(u, token_of(p, u, t * kRows + kRows - 1)));
}

__device__ __forceinline__ int64_t of_lane(int64_t x, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, lane) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32);
}
// Inclusive prefix sum over the wave's lanes of numbers below 2^62: 32-bit scans of
// 21 bits each.
__device__ __forceinline__ int64_t wave_scan64(int64_t x) {
  const int64_t a = wave_scan((int)(x & 0x1fffff)), b = wave_scan((int)(x >> 21 & 0x1fffff)), c = wave_scan((int)(x >> 42));
  return a + (b << 21) + (c << 42);
}

// The sequence in which place x of a running sum over the sequences lies, `of` being
// what a sequence adds to it, and the sum before it; b = batch behind the last.
struct Found {
  int b;
  int64_t before;
};
template <typename Of>
__device__ __forceinline__ Found find_seq(int batch, int64_t x, int lane, Of of) {
  int64_t before = 0;
  for (int i = 0; i < batch; i += 64) {
    const int64_t mine = i + lane < batch ? of(i + lane) : 0, upto = before + wave_scan64(mine);
    const uint64_t past = __ballot(upto > x);
    if (past) {
      const int at = __builtin_ctzll(past);
      return {i + at, of_lane(upto - mine, at)};
    }
    before = of_lane(upto, 63);
  }
  return {batch, before};
}

// Parts. Tiles of a causal batch cost from one key tile to hundreds, and there may be
// a few of them for 256 compute units. So the work (the sum of the tiles' costs, a model
// linear in the tile's number, so that a place is found by a prefix sum over the
// sequences and the root of a quadratic) is cut into equal parts, one a workgroup that
// the GPU holds at once; a part is the end of a tile, whole tiles, the start of another.
// A cut tile's partial results go to the workspace and prompt_join_kernel joins them.
// The device does all of it from the starts and lengths, so captured calls follow them.
// 2,041 tokens behind 5,040 others, 12 heads: 105 to 110 us. What it costs: 2.5 to 3.3 us
// to find a part, about 3 to write partials, 9 to 16 the join (15 here: of 256 rows a
// tile, some 40 MB of partials).
// Where there are two tiles a slot or more, a workgroup takes one whole tile and those
// that cost the most go first (16 mixed prompts: 96 us; cut into parts 126).
//
// The batch's work, cut into `parts` of `each`: as many as there are workgroups for,
// but none that is less than a tile or kPiece key tiles on the average.
struct Work {
  int64_t total, each;
  int parts;
  __device__ __forceinline__ int64_t begin(int w) const { return min(total, each * w); }
};
__device__ __forceinline__ Work work_in(const PromptParams& p, int64_t total, int tiles) {
  Work r;
  r.total = total;
  r.parts = (int)min((int64_t)p.parts, max((int64_t)tiles, total / (kPiece * 16 * kKeys)));
  r.parts = max(1, __builtin_amdgcn_readfirstlane(r.parts));
  r.each = (int64_t)((double)total / (double)r.parts) + 1 + (total >> 50);  // at least a parts-th
  return r;
}
template <KeyKind kKind, int kRows>
__device__ __forceinline__ int64_t work_of(const PromptParams& p, int b) {
  const Seq u = seq_of<kKind, kRows>(p, b);
  return u.before(u.tiles);
}

// Key tile k of tile t of sequence b; the work before the tile.
struct Place {
  int b, t, k;
  int64_t start;
};

// The key tile at which a part that begins at y of a tile's `cost` cuts its n key
// tiles: kEdge at least from both of its ends, or not at all.
__device__ __forceinline__ int cut_at(int64_t y, int64_t cost, int n) {
  const int k = min((int)((double)y * (double)n / (double)cost), n - kEdge);
  return k < kEdge ? 0 : k;
}

// Place x of the work, which is sequence f's.
template <KeyKind kKind, int kRows>
__device__ __forceinline__ Place place_at(const PromptParams& p, const Found& f, int64_t x) {
  if (f.b >= p.batch) return {p.batch, 0, 0, f.before};
  const Seq u = seq_of<kKind, kRows>(p, f.b);
  if (u.tiles <= 0) return {p.batch, 0, 0, f.before};  // only where overlapping rows' work passes 63 bits
  const int64_t y = x - f.before;
  // before(t) <= y < before(t + 1), from the root of its quadratic
  const float half = (float)u.base + 0.5f * (float)u.step, root = __builtin_amdgcn_sqrtf(half * half + 2.f * (float)u.step * (float)y);
  int t = min(max((int)(2.f * (float)y / (half + root)), 0), u.tiles - 1);
  while (t > 0 && u.before(t) > y) --t;
  while (t + 1 < u.tiles && u.before(t + 1) <= y) ++t;
  t = __builtin_amdgcn_readfirstlane(t);
  const int64_t before = u.before(t);
  return {f.b, t, __builtin_amdgcn_readfirstlane(cut_at(y - before, u.cost(t), tiles_seen<kRows>(p, u, t))), f.before + before};
}

// Where part w begins and ends.
template <KeyKind kKind, int kRows>
__device__ __forceinline__ Work find_part(const PromptParams& p, int w, int lane, Place* at, Place* end) {
  if (p.batch <= 64) {
    const Seq u = lane < p.batch ? seq_of<kKind, kRows>(p, lane) : Seq{};
    const int64_t mine = u.before(u.tiles), upto = wave_scan64(mine);
    const Work work = work_in(p, of_lane(upto, 63), __builtin_amdgcn_readlane(wave_scan(u.tiles), 63));
    auto place = [&](int64_t x) {
      const uint64_t past = __ballot(upto > x);
      const int b = past ? __builtin_ctzll(past) : p.batch;
      return place_at<kKind, kRows>(p, Found{b, past ? of_lane(upto - mine, b) : work.total}, x);
    };
    *at = place(work.begin(w));
    if (end) *end = place(work.begin(w + 1));
    return work;
  }
  int64_t sum = 0;
  int tiles = 0;
  for (int b = lane; b < p.batch; b += 64) {
    const Seq u = seq_of<kKind, kRows>(p, b);
    sum += u.before(u.tiles);
    tiles += u.tiles;
  }
  const Work work = work_in(p, of_lane(wave_scan64(sum), 63), __builtin_amdgcn_readlane(wave_scan(tiles), 63));
  auto place = [&](int64_t x) { return place_at<kKind, kRows>(p, find_seq(p.batch, x, lane, [&](int b) { return work_of<kKind, kRows>(p, b); }), x); };
  *at = place(work.begin(w));
  if (end) *end = place(work.begin(w + 1));
  return work;
}

// The w-th tile of the batch, those that cost the most first (so that none of them is
// among the last to begin), of `places` workgroups: as many as sequences that lie apart
// have tiles. Starts that go back can make tiles more; then every workgroup takes
// about as many, one after another (a loop around finding one instead costs registers
// that took 8,192 tokens from 462 to 495 us). Returns whether there is one.
template <KeyKind kKind, int kRows>
__device__ __forceinline__ bool find_tile(const PromptParams& p, int w, int places, int lane, Place* at, Place* end) {
  if (p.batch == 1) {
    const Seq u = seq_of<kKind, kRows>(p, 0);
    *at = {0, u.tiles - 1 - w, 0, 0};
    *end = {0, u.tiles - w, 0, 0};
    return w < u.tiles;
  }
  auto first_of = [&](int64_t tiles, int place) { return tiles / places * place + min((int64_t)place, tiles % places); };
  if (p.batch > 64) {  // too many to rank: a sequence's last tile first
    auto of = [&](int b) { return (int64_t)seq_of<kKind, kRows>(p, b).tiles; };
    int64_t sum = 0;
    for (int b = lane; b < p.batch; b += 64) sum += of(b);
    const int64_t tiles = of_lane(wave_scan64(sum), 63);
    if (tiles > places) {
      const int64_t x = first_of(tiles, w), y = first_of(tiles, w + 1);
      const Found f = find_seq(p.batch, x, lane, of), g = find_seq(p.batch, y, lane, of);
      *at = {f.b, (int)(x - f.before), 0, 0};
      *end = {g.b, (int)(y - g.before), 0, 0};
      return true;
    }
    if (w >= tiles) return false;
    const Found f = find_seq(p.batch, w, lane, of);
    *at = {f.b, (int)(of(f.b) - 1 - (w - f.before)), 0, 0};
    *end = {f.b, at->t + 1, 0, 0};
    return true;
  }
  const Seq u = lane < p.batch ? seq_of<kKind, kRows>(p, lane) : Seq{};
  const int before = wave_scan(u.tiles) - u.tiles, tiles = __builtin_amdgcn_readlane(before + u.tiles, 63);  // below 2^31
  if (tiles > places) {
    auto place = [&](int x) {
      const uint64_t past = __ballot(before + u.tiles > x);
      const int b = past ? __builtin_ctzll(past) : 0;
      return past ? Place{b, x - __builtin_amdgcn_readlane(before, b), 0, 0} : Place{p.batch, 0, 0, 0};
    };
    *at = place((int)first_of(tiles, w));
    *end = place((int)first_of(tiles, w + 1));
    return true;
  }
  if (w >= tiles) return false;
  const TileRun run = tile_run(u.tiles, u.base, u.step);
  const uint32_t costs_end = cost_end(wave_max_int(u.tiles ? (int)(u.cost(u.tiles - 1) / 32) : 0));
  const CostRange costs = costs_of(costs_end, w, [&](uint32_t c) { return __builtin_amdgcn_readlane(wave_scan(tiles_above(run, c)), 63); });
  // what is left between them is taken in the sequences' order
  const int over = tiles_above(run, costs.high), between = tiles_above(run, costs.low) - over;
  const int rank = w - __builtin_amdgcn_readlane(wave_scan(over), 63);
  const int upto = wave_scan(between);
  const int b = __builtin_ctzll(__ballot(upto > rank));
  auto of = [&](int x) { return __builtin_amdgcn_readlane(x, b); };
  *at = {b, of(u.tiles) - 1 - of(over) - (rank - of(upto - between)), 0, 0};
  *end = {b, at->t + 1, 0, 0};
  return true;
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
__device__ __forceinline__ float sum_bf16(uint32_t x, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2, x), s16x2{0x3f80, 0x3f80}, c, false);
}

// Where the 16-byte chunk c of row r of a tile of K or V lies in LDS (in bytes): the
// chunks of a row change places so that the lanes of a read hit different banks.
template <int D>
__device__ __forceinline__ uint32_t k_flip(uint32_t r) { return r / (128 / D) & (D / 8 - 1); }
template <int D>
__device__ __forceinline__ uint32_t v_flip(uint32_t r) { return 4 * (r / (128 / D)) & (D / 8 - 1); }
template <int D>
__device__ __forceinline__ uint32_t code_flip(uint32_t r) { return (r / (256 / D)) & (D / 16 - 1); }
template <int D>
__device__ __forceinline__ uint32_t k_at(uint32_t r, uint32_t c) { return r * (2 * D) + ((c ^ k_flip<D>(r)) * 16); }
template <int D>
__device__ __forceinline__ uint32_t v_at(uint32_t r, uint32_t c) { return r * (2 * D) + ((c ^ v_flip<D>(r)) * 16); }
template <int D>
__device__ __forceinline__ uint32_t code_at(uint32_t r, uint32_t c) { return r * D + ((c ^ code_flip<D>(r)) * 16); }

// ---- keys and values into LDS ----
// A lane's 16 (or 4) bytes to LDS, lane after lane from `to` on, past the registers.
// Written as instructions because the compiler would wait for the builtin's result
// before any read of LDS; here arrived() says when it is there. They write no
// register but m0. That one is reserved, of which the compiler warns; it still takes the
// clobber as a write that uses of m0 of its own (here there are none) may not pass.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const uint8_t* from, PBE_LDS uint8_t* to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"((uint32_t)(uintptr_t)to) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t lane_at, PBE_LDS uint8_t* to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_at), "s"(base), "s"((uint32_t)(uintptr_t)to) : "memory", "m0");
}
__device__ __forceinline__ void load_word_to_lds(const uint8_t* from, PBE_LDS uint8_t* to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"((uint32_t)(uintptr_t)to) : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most kLeft of what this wave has asked global memory for is on its way.
template <int kLeft>
__device__ __forceinline__ void arrived() {
  static_assert(kLeft < 64, "six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kLeft & 15) | (kLeft >> 4) << 14);
  asm volatile("" ::: "memory");
}

// Key tiles in LDS, loaded there directly, in turns: while one is used, the next
// kTurns - 1 are on their way.
//  - rows and BF16 pages: as they are. FP8 pages: as they are too; reads convert.
//  - MXFP4 pages: codes as they are, in two turns; each thread makes BF16 rows of what
//    it asked for before a tile is used (the values' codes cannot be transposed).
template <int D, KeyKind kKind, int kWaves>
struct Stage {
  static constexpr bool kMx = kKind == KeyKind::kMxfp4, kFp8 = kKind == KeyKind::kFp8, kScaled = kMx || kFp8;
  static constexpr int kTile = kKeys * D * (kFp8 ? 1 : 2);                 // bytes of K (or V) as they are read
  static constexpr int kRaw = kMx ? kKeys * D / 2 : kTile;                 // as they are loaded
  static constexpr int kTurns = 2;
  static constexpr int kAhead = kMx ? 2 : 1;                               // tiles asked for before one is used
  static constexpr int kInstr = kRaw / 1024;                               // loads for K (or V)
  static constexpr int kLoads = (2 * kInstr + kWaves - 1) / kWaves;        // of a wave
  static constexpr int kScaleBytes = kScaled ? 512 : 0;                    // K's and V's of a tile
  static constexpr int kAll = kTurns * 2 * kRaw + (kMx ? 2 * kTile : 0) + 3 * kScaleBytes;
  static constexpr int kPerTile = kLoads + kScaled * (kWaves == 1 ? 2 : 1);                        // loads of a wave and tile
  static constexpr int kRowBytes = kFp8 ? D : 2 * D, kChunks = kRowBytes / 16, kRowsALoad = 64 / kChunks;  // rows, FP8, BF16

  const PromptParams& p;
  const Seq& u;
  PBE_LDS uint8_t* const mem;
  int b, head, lane, wave, nblocks;
  int32_t ids = 0, next = 0;  // of 64 blocks from `chunk` on, a lane each; the next 64's entries
  uint64_t bad = 0;           // those of the 64 that are not in the pools (their id is 0 here)
  int chunk = -1;

  __device__ __forceinline__ Stage(const PromptParams& p_, const Seq& u_, PBE_LDS uint8_t* mem_, int b_, int head_, int lane_, int wave_)
      : p(p_), u(u_), mem(mem_), b(b_), head(head_), lane(lane_), wave(wave_), nblocks((int)(((uint32_t)u_.len + kBlockTokens - 1) / kBlockTokens)) {}

  __device__ __forceinline__ PBE_LDS uint8_t* raw(int turn) const { return mem + turn % kTurns * (2 * kRaw); }
  __device__ __forceinline__ PBE_LDS uint8_t* keys(int turn) const { return kMx ? mem + kTurns * 2 * kRaw : raw(turn); }
  __device__ __forceinline__ PBE_LDS uint8_t* values(int turn) const { return keys(turn) + kTile; }
  __device__ __forceinline__ PBE_LDS uint8_t* scales(int turn) const { return mem + kAll - 3 * kScaleBytes + turn % 3 * kScaleBytes; }

  __device__ __forceinline__ int32_t entry(int first) const { return p.tables[(int64_t)b * p.max_blocks + min(first + lane, nblocks - 1)]; }
  // Makes the ids of key tile kt's blocks (kt counts up by one) ready. Returns which
  // of its four are not in the pools.
  __device__ __forceinline__ uint32_t ids_for(int kt) {
    if constexpr (kKind != KeyKind::kRows) {
      const int c = kt / 16 * 64;
      if (c != chunk) {
        const int32_t id = chunk < 0 ? entry(c) : next;
        const bool off = id < 0 || id >= p.blocks;
        bad = __ballot(off);
        ids = off ? 0 : id;
        chunk = c;
        next = entry(c + 64);
      }
      return (uint32_t)(bad >> (kt % 16 * 4)) & 15u;
    }
    return 0;
  }
  // A block's id, of the same block for all lanes, or each lane's own.
  __device__ __forceinline__ uint64_t id_of(int block) const { return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(ids, min(block, nblocks - 1) & 63); }
  __device__ __forceinline__ uint64_t own_id_of(int block) const { return (uint64_t)(uint32_t)__shfl(ids, min(block, nblocks - 1) & 63, 64); }

  // Load i of this wave: K's or V's, and the place of its first byte among them.
  __device__ __forceinline__ int load_of(int i) const {
    // neighbouring ones of both in turn
    return kLoads % 2 ? (wave + i * kWaves) % (2 * kInstr) : i % 2 * kInstr + wave * (kLoads / 2) + i / 2;
  }

  // Asks for key tile kt, the turn-th of this workgroup's. Returns which of its
  // blocks are not in the pools. What lies behind the last key, in its block, is
  // loaded with it; rows behind it are the last one again.
  __device__ __forceinline__ uint32_t load(int kt, int turn) {
    if (kKind == KeyKind::kRows && kt * kKeys + kKeys <= u.len && max(p.k_stride, p.v_stride) < (1u << 28)) return load_tile<true>(kt, turn);
    return load_tile<false>(kt, turn);
  }
  // kFast (rows): the whole tile is there, and the distances within it fit 32 bits.
  template <bool kFast>
  __device__ __forceinline__ uint32_t load_tile(int kt, int turn) {
    const uint32_t wrong = ids_for(kt);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int n = load_of(i);
      const bool value = n >= kInstr;
      const int at = (value ? n - kInstr : n) * 64;  // in 16 bytes, among K's (or V's)
      const uint8_t* const from = value ? p.v : p.k;
      PBE_LDS uint8_t* const to = raw(turn) + n * 1024;
      if constexpr (!kMx) {
        const uint64_t stride = value ? p.v_stride : p.k_stride;
        const uint32_t r0 = (uint32_t)at / kChunks, r = (uint32_t)lane / kChunks, c = (uint32_t)lane % kChunks;
        const uint32_t flip = kFp8 ? code_flip<D>(r0 + r) : value ? v_flip<D>(r0 + r) : k_flip<D>(r0 + r);
        const uint64_t in_row = (uint64_t)head * kRowBytes;
        if constexpr (kKind == KeyKind::kRows && kFast) {
          load_to_lds(from + (uint64_t)(u.first + kt * kKeys + (int)r0) * stride + in_row, r * (uint32_t)stride + (c ^ flip) * 16, to);
        } else if constexpr (kKind == KeyKind::kRows) {
          load_to_lds(from + (uint64_t)(u.first + min(kt * kKeys + (int)(r0 + r), u.len - 1)) * stride + in_row + (c ^ flip) * 16, to);
        } else {
          load_to_lds(from + id_of(kt * 4 + (int)(r0 / kBlockTokens)) * p.half + r0 % kBlockTokens * stride + in_row,
                      r * (uint32_t)stride + (c ^ flip) * 16, to);
        }
      } else {
        // K: [4 quarters][16 tokens][D/8 bytes] a block, V: [4 quads][16 columns][D/8]
        constexpr int kBlock = D / 2;  // of 16 bytes, in a block
        const uint64_t in_block = (uint64_t)head * mx_head_bytes(D);
        if constexpr (D == 128) load_to_lds(from + id_of(kt * 4 + at / kBlock) * p.half + in_block, (uint32_t)lane * 16, to);
        else load_to_lds(from + own_id_of(kt * 4 + (at + lane) / kBlock) * p.half + in_block + (uint32_t)(lane % kBlock) * 16, to);
      }
    }
    if constexpr (kScaled) {
      // K's by even waves, V's by odd ones; a wave alone asks for both
#pragma unroll
      for (int i = 0; i < (kWaves == 1 ? 2 : 1); ++i) {
        const bool value = kWaves == 1 ? i : wave & 1;
        const uint8_t* from = value ? p.v_scales : p.k_scales;
        if constexpr (kMx) {  // [D/32 groups][16 tokens] a block
          constexpr int kWords = D / 8;
          from += own_id_of(kt * 4 + (lane / kWords) % 4) * (p.half / 16) + (uint64_t)head * mx_head_scales(D) + lane % kWords * 4;
        } else {
          from += ((own_id_of(kt * 4 + lane / kBlockTokens) * kBlockTokens + (uint64_t)(lane % kBlockTokens)) * (uint64_t)p.kv_heads + (uint64_t)head) * 4;
        }
        load_word_to_lds(from, scales(turn) + value * 256);
      }
    }
    return wrong;
  }

  // What this wave asked for of a tile is there; `more`: a later one was asked for, too.
  __device__ __forceinline__ void wait(bool more) const {
    if (more) arrived<(kAhead - 1) * kPerTile>();
    else arrived<0>();
  }

  // MXFP4: BF16 rows of the turn-th tile from its codes.
  __device__ __forceinline__ void convert(int turn) const {
    PBE_LDS uint8_t* const ks = keys(0);
    PBE_LDS uint8_t* const vs = values(0);
    PBE_LDS const uint8_t* const sc = scales(turn);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (kLoads % 2 && wave + i * kWaves >= 2 * kInstr) break;
      const int n = load_of(i);
      const bool value = n >= kInstr;
      const uint32_t at = (uint32_t)((value ? n - kInstr : n) * 64 + lane);
      const u32x4 x = *(PBE_LDS const u32x4*)(raw(turn) + n * 1024 + lane * 16);
      const uint32_t block = at / (D / 2), o = at % (D / 2), groups = block * mx_head_scales(D);
      if (!value) {
        // 16 bytes: a token's quarter of the dims (D 128), or that of two tokens
        constexpr uint32_t kTok = 128 / D, kEach = 4 / kTok;  // tokens; chunks of each
        const uint32_t quarter = o / (kBlockTokens / kTok), tok = o % (kBlockTokens / kTok) * kTok, group = D == 128 ? quarter : quarter / 2;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          const uint32_t t = tok + e / kEach;
          const float f = mx_scale(sc[groups + group * kBlockTokens + t]);
          *(PBE_LDS u32x4*)(ks + k_at<D>(block * kBlockTokens + t, quarter * (D / 32) + e % kEach)) = mx_values(x[e], f);
        }
      } else {
        // four tokens' dims of a column (D 128: eight), or of two columns (four each)
        constexpr uint32_t kCols = 128 / D;
        const uint32_t quad = o / (16 / kCols), column = o % (16 / kCols) * kCols, group = D == 128 ? column / 4 : column / 8;
        const uint32_t four = *(PBE_LDS const uint32_t*)(sc + 256 + groups + group * kBlockTokens + quad * 4);
#pragma unroll
        for (uint32_t t = 0; t < 4; ++t) {
          const float f = mx_scale((four >> (8 * t)) & 255u);
          const uint32_t row = block * kBlockTokens + quad * 4 + t;
          if constexpr (D == 128) {
            *(PBE_LDS u32x4*)(vs + v_at<D>(row, column)) = mx_values(x[t], f);
          } else {
            const uint32_t a = x[t / 2] >> (16 * (t % 2)), c = x[2 + t / 2] >> (16 * (t % 2));
            *(PBE_LDS u32x4*)(vs + v_at<D>(row, column / 2)) = u32x4{mx_pair<0>(a, f), mx_pair<1>(a, f), mx_pair<0>(c, f), mx_pair<1>(c, f)};
          }
        }
      }
    }
  }
};

__device__ __forceinline__ u32x4 e4m3x8_to_bf16x8(u32x2 x) {
  const u32x2 lo = e4m3x4_to_bf16x4_cvt(x.x), hi = e4m3x4_to_bf16x4_cvt(x.y);
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}

// Non-zero where one of a word's BF16 values is an infinity or a NaN, or one of its
// E4M3 codes a NaN; and the word with zeros in their place.
template <bool kFp8>
__device__ __forceinline__ uint32_t special(uint32_t x) {
  return kFp8 ? ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((x & 0x7fff7fffu) + 0x00800080u) & 0x80008000u;
}
template <bool kFp8>
__device__ __forceinline__ uint32_t without_special(uint32_t x) {
  const uint32_t s = special<kFp8>(x);
  return kFp8 ? x & ~(s | (s - (s >> 7))) : x & ~(s | (s - (s >> 15)));
}

// Which part (or tile) and head a workgroup has. Workgroups go to the eight XCDs in
// turn, each with an L2 of its own. FP8 and MXFP4 pages' lines hold several heads' bytes
// (scales all of them): all heads of a part on one XCD. Of BF16 every head has lines of
// its own: neighbouring workgroups take neighbouring heads, so that with 4 or 8 KV heads
// an XCD's L2 holds one or two heads' K and V instead of all.
template <KeyKind kKind>
__device__ __forceinline__ void workgroup_of(const PromptParams& p, int* w, int* head) {
  const int x = blockIdx.x;
  if constexpr (kKind == KeyKind::kFp8 || kKind == KeyKind::kMxfp4) {
    const int q = x / kXcds;
    *w = q / p.kv_heads * kXcds + x % kXcds;
    *head = q % p.kv_heads;
  } else {
    *w = x / p.kv_heads;
    *head = x - *w * p.kv_heads;
  }
}

// One part (or tile) a workgroup: kWaves waves of 32 rows that share the key tiles in
// LDS. A tile's 64 keys are asked for a tile (MXFP4: two) ahead, straight into LDS; one
// barrier a tile (MXFP4: two), behind which the tile read before is overwritten.
// Registers: O 4 x 16, scores 32, Q 32, weights 16; two waves a SIMD.
// FP8 codes become BF16 operands at the LDS reads: once a tile instead, into BF16 tiles,
// took the same time (130.8 and 130.4 us, 128 tokens at the end of 32,768) and more LDS.
// A lane reads eight of a chunk's 16 codes of a key, so each half of a wave uses half of
// the banks (37% of the kernel's LDS cycles are conflicts; over rows none). The matrix
// product of 8-bit operands is no faster at this shape and would round the queries.
template <int D, KeyKind kKind, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves > 2 ? 2 : 1) void prompt_attention_kernel(const PromptParams p) {
  using S = Stage<D, kKind, kWaves>;
  constexpr int kRows = 32 * kWaves, kDims = D / 32;
  constexpr bool kFp8 = S::kFp8;
  __shared__ __align__(1024) uint8_t tile_mem[S::kAll];
  __shared__ uint32_t special_mem[kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int w, head;
  workgroup_of<kKind>(p, &w, &head);
  const int h = lane >> 5, col = lane & 31;
  Place at, end;
  if (p.parts) {
    if (w >= p.parts) return;
    if (w >= find_part<kKind, kRows>(p, w, lane, &at, &end).parts) return;
  } else {
    if (!find_tile<kKind, kRows>(p, w, (int)(gridDim.x / (uint32_t)p.kv_heads), lane, &at, &end)) return;
  }
  bool opened = false;  // a tile was worked on before
  for (int b = at.b; b < p.batch && b <= end.b; ++b) {
    const Seq u = seq_of<kKind, kRows>(p, b);
    const int t1 = b == end.b ? min(u.tiles, end.t + (end.k > 0)) : u.tiles;
    for (int t = b == at.b ? at.t : 0; t < t1; ++t) {
      const int row0 = t * kRows + wave * 32;                     // of the wave
      const int stacked = u.rows * p.group;                       // rows of the sequence and this head
      const int token = token_of(p, u, row0 + col), g = min(row0 + col, stacked - 1) - token * p.group;
      const int q_heads = p.kv_heads * p.group, q_head = head * p.group + g;
      const int64_t q_row = (int64_t)u.begin + token;
      const int seen = seen_by(u, token);
      const int wave_least = seen_by(u, token_of(p, u, row0)), wave_most = row0 < stacked ? seen_by(u, token_of(p, u, row0 + 31)) : 0;
      const int tile_least = seen_by(u, token_of(p, u, t * kRows));
      const int all = tiles_seen<kRows>(p, u, t);
      const bool opens = b == at.b && t == at.t, ends = b == end.b && t == end.t;
      const int kt0 = opens ? at.k : 0, kt1 = ends ? end.k : all;
      if (kt0 == kt1 && all > 0) continue;

      f32x16 o[kDims];
#pragma unroll
      for (int i = 0; i < kDims; ++i) o[i] = f32x16{};
      float m = -INFINITY, l = 0.f;
      bool far = false;

      S stage(p, u, (PBE_LDS uint8_t*)tile_mem, b, head, lane, wave);
      if (opened) __syncthreads();  // the tile before has been read
      opened = true;
      // Blocks not in the pools: of this key tile and those asked for.
      constexpr int kAhead = S::kAhead;
      uint32_t wrong = 0, wrongs[kAhead] = {};
      if (kt0 < kt1) wrongs[0] = stage.load(kt0, 0);
      bf16x8 q[D / 16];
      {
        const uint8_t* from = p.q + (uint64_t)q_row * p.q_stride + (uint64_t)q_head * (2 * D) + h * 16;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) q[i] = *(PBE_GLOBAL const bf16x8*)(uintptr_t)(from + i * 32);
      }
      arrived<0>();  // here, so that no wait for q stands in the loop
#pragma unroll
      for (int i = 1; i < kAhead; ++i)
        if (kt0 + i < kt1) wrongs[i] = stage.load(kt0 + i, i);
      for (int kt = kt0; kt < kt1; ++kt) {
        const int turn = kt - kt0, first = kt * kKeys;
        stage.wait(kt + 1 < kt1);
        __syncthreads();
        if constexpr (S::kMx) {
          stage.convert(turn);
          __syncthreads();
        }
        wrong = wrongs[0];
#pragma unroll
        for (int i = 0; i + 1 < kAhead; ++i) wrongs[i] = wrongs[i + 1];
        if (kt + kAhead < kt1) wrongs[kAhead - 1] = stage.load(kt + kAhead, turn + kAhead);
        PBE_LDS const uint8_t* const kb = stage.keys(turn);
        PBE_LDS uint8_t* const vb = stage.values(turn);
        PBE_LDS const float* const scales = (PBE_LDS const float*)stage.scales(turn);
        auto key_of = [&](int sub, int i) { return first + sub * 32 + 8 * (i / 4) + 4 * h + i % 4; };
        // A operand of keys 32 sub.. and dims 16 i..: a key's eight dims a lane.
        auto keys = [&](int sub, int i) {
          if constexpr (kFp8) return e4m3x8_to_bf16x8(*(PBE_LDS const u32x2*)(kb + code_at<D>(sub * 32 + col, i) + 8 * h));
          else return *(PBE_LDS const u32x4*)(kb + k_at<D>(sub * 32 + col, 2 * i + h));
        };
        // A operand of dims 32 d.. and keys 16 n..: a dim's eight keys a lane, those that
        // the scores' registers have: 4h.. and 8 + 4h... Transposing reads: of 16 lanes each
        // asks for a part of a key's 16 dims and gets one dim of four (or eight) keys.
        auto values = [&](int d, int n) {
          const uint32_t i = lane & 15, half = (lane >> 4) & 1;
          if constexpr (kFp8) {
            const uint32_t r = 16 * n + 4 * h + i / 2 + (i >= 8 ? 4 : 0);
            const auto x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((PBE_LDS i32x2*)(vb + code_at<D>(r, 2 * d + half) + 8 * (i % 2)));
            return e4m3x8_to_bf16x8(__builtin_bit_cast(u32x2, x));
          } else {
            const uint32_t chunk = 4 * d + 2 * half + (i % 4) / 2, r = 16 * n + 4 * h + i / 4;
            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((PBE_LDS s16x4*)(vb + v_at<D>(r, chunk) + 8 * (i % 2))));
            const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((PBE_LDS s16x4*)(vb + v_at<D>(r + 8, chunk) + 8 * (i % 2))));
            return u32x4{x.x, x.y, y.x, y.y};
          }
        };
        // Values that some of the tile's rows do not see may be anything: an infinity or a
        // NaN times a weight of zero would reach those rows. Where there are any, rows that
        // see them get them here, and the product below finds zeros in their place.
        if (first + kKeys > tile_least) {
          // 16 bytes a thread at a time
          constexpr int kStep = 64 * kWaves * 16, kEach = (S::kTile + kStep - 1) / kStep;
          const bool has = kStep <= S::kTile || (int)threadIdx.x * 16 < S::kTile;
          uint32_t some = 0;
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            if (!has) break;
            const u32x4 x = *(PBE_LDS const u32x4*)(vb + i * kStep + threadIdx.x * 16);
            some |= special<kFp8>(x.x) | special<kFp8>(x.y) | special<kFp8>(x.z) | special<kFp8>(x.w);
          }
          const bool any = __ballot(some != 0) != 0;
          if (lane == 0) special_mem[wave] = any;
          __syncthreads();
          bool odd = false;
#pragma unroll
          for (int i = 0; i < kWaves; ++i) odd |= special_mem[i] != 0;
          if (odd) {
            if (first < wave_most) {
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
                f32x16 up = {}, down = {};  // how many a row sees; a NaN counts as both
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                  const u32x4 x = values(d, n);
                  u32x4 plus, minus;
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = x[e] & 0xffffu, hi = x[e] >> 16;
                    const bool lo_off = (lo & 0x7f80u) == 0x7f80u, hi_off = (hi & 0x7f80u) == 0x7f80u;
                    plus[e] = (lo_off && lo != 0xff80u ? 0x3f80u : 0u) | (hi_off && hi != 0xff80u ? 0x3f800000u : 0u);
                    minus[e] = (lo_off && lo != 0x7f80u ? 0x3f80u : 0u) | (hi_off && hi != 0x7f80u ? 0x3f800000u : 0u);
                  }
                  up = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, plus), sees[n], up, 0, 0, 0);
                  down = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, minus), sees[n], down, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] += (up[i] > 0.f ? INFINITY : 0.f) - (down[i] > 0.f ? INFINITY : 0.f);
              }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
              if (!has) break;
              PBE_LDS u32x4* const to = (PBE_LDS u32x4*)(vb + i * kStep + threadIdx.x * 16);
              u32x4 x = *to;
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = without_special<kFp8>(x[e]);
              *to = x;
            }
            __syncthreads();
          }
        }
        if (first < wave_most) {
          f32x16 s[2];
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) s[sub] = f32x16{};
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
              const bf16x8 a = __builtin_bit_cast(bf16x8, keys(sub, i));
              s[sub] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, q[i], s[sub], 0, 0, 0);
            }
          // six reads ahead of the products
          constexpr int kProducts = D / 8, kFirst = 6;
          __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);
#pragma unroll
          for (int i = 0; i < kProducts - kFirst; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          __builtin_amdgcn_sched_group_barrier(0x8, kFirst, 0);
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
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[sub][i]);
          top = halves_max(top);
          // The maximum that weights refer to follows the largest score only when that
          // has passed it by 2^kLazy: sums then need no scaling for most tiles.
          if (__any((top - m) * p.scale > kLazy)) {
            const float now = fmaxf(m, top);
            const float fade = m == now || m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - now) * p.scale);
            m = now;
            far = __any(m != -INFINITY && fabsf(m * p.scale) > kFar);
            l *= fade;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[d][i] *= fade;
          }
          // 2^((score - maximum) * scale), by one multiply-add: its rounding of maximum *
          // scale is in all weights of a row alike, and below kFar far below their own.
          const float base = m == -INFINITY ? 0.f : m;
          float scaled = base * p.scale;
          if (far) {
            scaled = 0.f;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub)
#pragma unroll
              for (int i = 0; i < 16; ++i) s[sub][i] -= base;
          }
          float sum = 0.f;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              s[sub][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][i], p.scale, -scaled));
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
            if (masked) {  // a scale that the row does not see may be an infinity or a NaN
#pragma unroll
              for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[sub][i] = key_of(sub, i) < seen ? s[sub][i] : 0.f;
            }
          }
          bf16x8 weights[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            u32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = pack_bf16(s[n / 2][8 * (n % 2) + 2 * e], s[n / 2][8 * (n % 2) + 2 * e + 1]);
            weights[n] = __builtin_bit_cast(bf16x8, x);
            if constexpr (kKind != KeyKind::kFp8) {
#pragma unroll
              for (int e = 0; e < 4; ++e) sum = sum_bf16(x[e], sum);
            }
          }
          l += sum;
#pragma unroll
          for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int n = 0; n < 4; ++n)
              o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, values(d, n)), weights[n], o[d], 0, 0, 0);
          // four products' reads ahead
          constexpr int kMore = kDims * 4 - 4, kReads = kFp8 ? 1 : 2;
          __builtin_amdgcn_sched_group_barrier(0x100, 4 * kReads, 1);
#pragma unroll
          for (int i = 0; i < kMore; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, kReads, 1);
          }
          __builtin_amdgcn_sched_group_barrier(0x8, 4, 1);
        }
      }

      l = halves_sum(l);
      if (row0 + col >= stacked) continue;
      if (kt0 == 0 && kt1 == all) {
        const float over = u.bad ? NAN : seen > 0 ? 1.f / l : 0.f;
        uint8_t* to = p.out + ((uint64_t)q_row * (uint64_t)q_heads + (uint64_t)q_head) * (2 * D) + h * 8;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *(PBE_GLOBAL u32x2*)(uintptr_t)(to + d * 64 + i * 16) =
                u32x2{pack_bf16(o[d][4 * i] * over, o[d][4 * i + 1] * over), pack_bf16(o[d][4 * i + 2] * over, o[d][4 * i + 3] * over)};
      } else {
        const uint64_t slot = ((uint64_t)w * 2 + !opens) * (uint64_t)p.kv_heads + (uint64_t)head;
        const uint64_t row = slot * kRows + (uint64_t)(row0 - t * kRows + col);
        float* acc = p.part_acc + row * D + 4 * h;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *(PBE_GLOBAL f32x4*)(uintptr_t)(acc + d * 32 + i * 8) = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (h == 0) *(PBE_GLOBAL f32x2*)(uintptr_t)(p.part_ml + row * 2) = f32x2{m, l};
      }
    }
  }
}

// Joins the tiles that were cut: o = sum 2^((m_i - m) scale) o_i / sum 2^((m_i - m)
// scale) l_i, in the parts' order. Of a tile's n + 1 parts, each of the n that do not
// begin it has a workgroup here, which takes its share of the tile's rows: a launch of its
// own, so that as many workgroups join as there are parts. The last part to arrive at a
// tile could join it instead, by tickets (arrival.h) and in the same order; one workgroup
// would then read all of a tile's partials. That was not tried.
constexpr int kTogether = 4;  // loads of a thread that are on their way together
template <int D, int kRows>
constexpr int join_threads() {
  return D / 4 * kRows / kTogether < 1024 ? D / 4 * kRows / kTogether : 1024;
}
template <int D, KeyKind kKind, int kRows>
__global__ __launch_bounds__((join_threads<D, kRows>())) void prompt_join_kernel(const PromptParams p) {
  constexpr int kLanes = D / 4;
  __shared__ int cuts[kMaxCuts + 2];  // the key tiles at which the tile's parts begin
  const int lane = threadIdx.x & 63;
  int w, head;
  workgroup_of<kKind>(p, &w, &head);
  if (w >= p.parts) return;
  Place at;
  const Work work = find_part<kKind, kRows>(p, w, lane, &at, nullptr);
  if (w >= work.parts || at.b >= p.batch || at.k == 0) return;
  const Seq u = seq_of<kKind, kRows>(p, at.b);
  const int64_t cost = u.cost(at.t);
  const int all = tiles_seen<kRows>(p, u, at.t);
  // Part i's start: its cut of this tile, -1 before the tile, `all` behind it.
  auto cut_of = [&](int i) {
    const int64_t y = work.begin(i) - at.start;
    return y < 0 ? -1 : y >= cost ? all : cut_at(y, cost, all);
  };
  // the last part that begins at or before the tile's start
  int w0 = w;
  for (;;) {
    const uint64_t inside = __ballot(w0 - 1 - lane >= 0 && cut_of(w0 - 1 - lane) > 0);
    const int n = ~inside ? __builtin_ctzll(~inside) : 64;
    w0 -= n;
    if (n < 64) break;
  }
  w0 = max(w0 - 1, 0);  // w0 + 1 is the first that begins inside; part 0 begins at no tile's inside
  int n = 0;  // parts that begin inside
  for (int i = w0;; i += 64) {
    const int c = i + lane <= work.parts ? cut_of(i + lane) : all;
    const uint64_t past = __ballot(c >= all);
    const int many = past ? __builtin_ctzll(past) : 64;
    if (threadIdx.x < 64 && lane <= many && i - w0 + lane < kMaxCuts + 2) cuts[i - w0 + lane] = c;
    n = i - w0 + many - 1;
    if (past) break;
  }
  __syncthreads();
  if (w <= w0 || w > w0 + n) return;  // never, but where overlapping rows' work passes 63 bits
  const int share = w - w0 - 1, rows = min(kRows, u.rows * p.group - at.t * kRows);
  const int from = (int)((int64_t)rows * share / n), to = (int)((int64_t)rows * (share + 1) / n);
  const int q_heads = p.kv_heads * p.group;
  const bool begins = cuts[0] == 0;  // else its first tile was another one
  constexpr int kStep = join_threads<D, kRows>() / kLanes;
  const int d = 4 * ((int)threadIdx.x % kLanes);
  // A thread has kTogether rows and a part at a time, or, where the share has no more
  // rows than are under way at once, a row and kTogether parts (128 tokens at the end of
  // 32,768: 129 to 119 us; 4 x 4 tokens over 5,040: 35 to 30). Eight parts take registers
  // that cost more workgroups at once than they save: 64 x 4 tokens of 28 heads of 128 dims
  // over MXFP4 pages 81 to 90.
  const bool few = to - from <= kStep;
  const int next_row = few ? 0 : kStep, next_part = few ? 1 : 0;
  auto add_to = [&](float& m, float& l, f32x4& acc, float pm, float pl, f32x4 x) {
    const float now = fmaxf(m, pm), base = now == -INFINITY ? 0.f : now;
    const float old = m == now ? 1.f : __builtin_amdgcn_exp2f((m - base) * p.scale);
    const float add = pm == now ? 1.f : __builtin_amdgcn_exp2f((pm - base) * p.scale);
    m = now;
    l = l * old + pl * add;
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = acc[c] * old + x[c] * add;
  };
  for (int r0 = from + (int)threadIdx.x / kLanes; r0 < to; r0 += kTogether * kStep) {
    float m[kTogether], l[kTogether];
    f32x4 acc[kTogether];
#pragma unroll
    for (int e = 0; e < kTogether; ++e) m[e] = -INFINITY, l[e] = 0.f, acc[e] = f32x4{};
    for (int i0 = 0; i0 <= n; i0 += few ? kTogether : 1) {
      f32x2 ml[kTogether];
      f32x4 x[kTogether];
#pragma unroll
      for (int e = 0; e < kTogether; ++e) {
        const int i = i0 + e * next_part;
        ml[e] = f32x2{-INFINITY, 0.f}, x[e] = f32x4{};
        if (i > n || max(cuts[i], 0) == cuts[i + 1]) continue;  // nothing between two cuts
        const uint64_t place = (((uint64_t)(w0 + i) * 2 + (i == 0 && !begins)) * (uint64_t)p.kv_heads + (uint64_t)head) * kRows;
        const uint64_t at_row = place + (uint64_t)min(r0 + e * next_row, to - 1);
        ml[e] = *(PBE_GLOBAL const f32x2*)(uintptr_t)(p.part_ml + at_row * 2);
        x[e] = *(PBE_GLOBAL const f32x4*)(uintptr_t)(p.part_acc + at_row * D + d);
      }
#pragma unroll
      for (int e = 0; e < kTogether; ++e) add_to(m[e], l[e], acc[e], ml[e].x, ml[e].y, x[e]);
    }
    if (few) {
#pragma unroll
      for (int e = 1; e < kTogether; ++e) add_to(m[0], l[0], acc[0], m[e], l[e], acc[e]);
    }
#pragma unroll
    for (int e = 0; e < kTogether; ++e) {
      if (e > 0 && (few || r0 + e * kStep >= to)) break;
      const int row = at.t * kRows + r0 + e * kStep;
      const int token = (int)fast_div((uint32_t)row, p.by_group), g = row - token * p.group;
      const float over = seen_by(u, token) > 0 ? 1.f / l[e] : 0.f;
      *(PBE_GLOBAL u32x2*)(uintptr_t)(p.out + (((uint64_t)u.begin + token) * (uint64_t)q_heads + (uint64_t)(head * p.group + g)) * (2 * D) + 2 * d) =
          u32x2{pack_bf16(acc[e][0] * over, acc[e][1] * over), pack_bf16(acc[e][2] * over, acc[e][3] * over)};
    }
  }
}

template <int D, KeyKind kKind, int kWaves>
hipError_t launch(const PromptParams& p, int64_t workgroups, hipStream_t stream) {
  const int64_t rounded = (workgroups + kXcds - 1) / kXcds * kXcds;
  const dim3 grid((uint32_t)(rounded * p.kv_heads));
  hipLaunchKernelGGL((prompt_attention_kernel<D, kKind, kWaves>), grid, dim3(64 * kWaves), 0, stream, p);
  if (p.parts) hipLaunchKernelGGL((prompt_join_kernel<D, kKind, 32 * kWaves>), grid, dim3(join_threads<D, 32 * kWaves>()), 0, stream, p);
  return hipGetLastError();
}

template <int D, KeyKind kKind>
hipError_t launch_rows(const PromptParams& p, int rows, int64_t workgroups, hipStream_t stream) {
  switch (rows) {
    case 32:
      if constexpr (kKind == KeyKind::kFp8 && D == 128) return launch<D, kKind, 1>(p, workgroups, stream);
      return hipErrorInvalidValue;
    case 64: return launch<D, kKind, 2>(p, workgroups, stream);
    case 128: return launch<D, kKind, 4>(p, workgroups, stream);
    default: return launch<D, kKind, 8>(p, workgroups, stream);
  }
}

template <int D>
hipError_t launch_kind(const PromptParams& p, KeyKind kind, int rows, int64_t workgroups, hipStream_t stream) {
  switch (kind) {
    case KeyKind::kRows: return launch_rows<D, KeyKind::kRows>(p, rows, workgroups, stream);
    case KeyKind::kBf16: return launch_rows<D, KeyKind::kBf16>(p, rows, workgroups, stream);
    case KeyKind::kFp8: return launch_rows<D, KeyKind::kFp8>(p, rows, workgroups, stream);
    default: return launch_rows<D, KeyKind::kMxfp4>(p, rows, workgroups, stream);
  }
}

}  // namespace

// Bytes of LDS of a workgroup.
static int64_t lds_bytes(KeyKind kind, int dim) {
  auto of = [&](auto stage64, auto stage128) { return dim == 64 ? decltype(stage64)::value : decltype(stage128)::value; };
  switch (kind) {
    case KeyKind::kFp8: return of(std::integral_constant<int, Stage<64, KeyKind::kFp8, 1>::kAll>(), std::integral_constant<int, Stage<128, KeyKind::kFp8, 1>::kAll>());
    case KeyKind::kMxfp4:
      return of(std::integral_constant<int, Stage<64, KeyKind::kMxfp4, 1>::kAll>(), std::integral_constant<int, Stage<128, KeyKind::kMxfp4, 1>::kAll>());
    default: return of(std::integral_constant<int, Stage<64, KeyKind::kRows, 1>::kAll>(), std::integral_constant<int, Stage<128, KeyKind::kRows, 1>::kAll>());
  }
}

PromptPlan plan_prompt(int64_t n_q, int64_t batch, int32_t group, int32_t kv_heads, KeyKind kind, int64_t most_keys, int64_t units, uint64_t workspace,
                       int32_t head_dim) {
  PromptPlan r;
  const int64_t rows = n_q * group;
  // The fewest rows that hold an average sequence's: more rows read K and V from LDS and
  // cache less often (256 and 128 rows a tile over 8,192 tokens: 469 and 495 us; over
  // 2,041 behind 5,040: 109 and 122), rows that no token fills cost as much as others.
  r.rows = rows <= 64 * batch ? 64 : rows <= 128 * batch ? 128 : 256;
  // A wave alone loads and waits by itself, and is slower (64 x 4 tokens of 12 heads of 128
  // dims over 5,040 of MXFP4 pages: 66 us, two waves with one at work 54; of BF16 pages 80
  // and 81; 4 x 4 over FP8 pages 40 and 34), but for FP8 pages of 128 dims and heads enough
  // for a quarter of the GPU: 64 x 4 tokens 57 and 70, 16 x 4 of four KV heads 45 and 48,
  // 16 x 4 of two 46 and 42 (all before the join took four parts at once; 64 x 4 is 53 with
  // it). Three batches are few for such a border.
  if (rows <= 32 * batch && kind == KeyKind::kFp8 && head_dim == 128 && 4 * batch * kv_heads >= units) r.rows = 32;
  // Few short prompts, whose tiles are not cut: smaller tiles, so that more compute units
  // have one (41 tokens of 14 heads of 64 dims: 256 rows a tile 7.2 us, 128 5.9, 64 5.6;
  // eight of 128 tokens 14.5, 12.7, 13.2).
  const int64_t keys = kind == KeyKind::kRows ? most_keys / batch : most_keys;  // of a sequence, on the average or at most
  while (r.rows > 64 && keys < 2 * kEdge * kKeys && 2 * (rows / r.rows + std::min(batch, n_q)) * kv_heads < units) r.rows /= 2;
  r.tiles = rows / r.rows + std::min(batch, n_q);
  // workgroups that a compute unit holds: eight waves' registers, 160 KiB of LDS
  const int64_t held = std::min<int64_t>(256 / r.rows, 160 * 1024 / (lds_bytes(kind, head_dim) + 64));
  const int64_t slots = std::max<int64_t>(1, held * units / kv_heads);
  r.each = 2ull * (uint64_t)kv_heads * (uint64_t)r.rows * (uint64_t)(head_dim + 2) * 4;
  const int64_t parts = std::min<int64_t>(slots, (int64_t)std::min<uint64_t>(workspace / r.each, kMaxCuts));
  // Parts where there are fewer than two tiles a slot, tiles long enough to be cut, and a
  // workspace for nearly all slots (or more parts than tiles).
  const bool cut = parts > 1 && most_keys >= 2 * kEdge * kKeys && r.tiles < 2 * slots && (8 * parts >= 7 * slots || parts >= r.tiles);
  r.parts = cut ? (int32_t)parts : 0;
  return r;
}

hipError_t launch_prompt_attention(PromptParams p, const PromptPlan& plan, int dim, KeyKind kind, hipStream_t stream) {
  p.parts = plan.parts;
  p.step = 16 * plan.rows / p.group;
  const int64_t workgroups = plan.parts ? plan.parts : plan.tiles;
  if (dim == 128) return launch_kind<128>(p, kind, plan.rows, workgroups, stream);
  if (dim == 64) return launch_kind<64>(p, kind, plan.rows, workgroups, stream);
  return hipErrorInvalidValue;
}

}  // namespace pbe
