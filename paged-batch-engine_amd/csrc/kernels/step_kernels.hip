// gfx950 step tables: what the host's build_block_tables, build_seq_lens and
// build_slot_mapping make, from page lists and lengths in device memory, for
// requests that add any number of tokens.
//   start_b = sum over i < b of max(new_i, 0), len_b = cached_b + new_b;
//   token t of request b: position p = cached_b + t - start_b,
//   slot = page[p / block_size] * block_size + p % block_size.
//
// One launch. A workgroup writes the slots and positions of 1,024 tokens, or
// 2,048 entries of the tables, which need no sums; the first one writes
// lengths and starts as well. The tokens' requests follow from a prefix sum
// over new_lens, which every token workgroup makes for itself, 1,024 requests
// at a time, up to the last request of its tokens: the lengths are a few KB
// out of L2, and a second launch would cost more than the sum.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_device.h"
#include "step_kernels.h"

namespace pbe {
namespace {

constexpr int kThreads = 256, kPer = 4, kChunk = kThreads * kPer;  // requests summed at a time
static_assert(kStepTokens == kChunk, "a thread sums four requests and writes four tokens");

template <int kCtrl, int kRows>
__device__ __forceinline__ int scan_step(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, kCtrl, kRows, 0xf, false);
}
// Inclusive prefix sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x = scan_step<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: within rows of 16
  x = scan_step<0x112, 0xf>(x);
  x = scan_step<0x114, 0xf>(x);
  x = scan_step<0x118, 0xf>(x);
  x = scan_step<0x142, 0xa>(x);     // row_bcast 15 into rows 1 and 3
  return scan_step<0x143, 0xc>(x);  // row_bcast 31 into rows 2 and 3
}

// A request's pages, and whether its lengths and pages make sense.
struct Request {
  int64_t len;     // cached + new
  uint32_t first;  // of page_ids
  uint32_t pages;
  bool ok;
};
__device__ __forceinline__ Request request(const StepTablesParams& p, uint32_t b, int32_t added) {
  Request r;
  const int32_t cached = p.cached_lens[b], lo = p.page_starts[b], hi = p.page_starts[b + 1];
  r.len = (int64_t)cached + added;
  const bool listed = lo >= 0 && hi >= lo && (uint32_t)hi <= p.n_page_ids;
  r.first = listed ? (uint32_t)lo : 0u;
  r.pages = listed ? (uint32_t)(hi - lo) : 0u;
  const uint32_t last = (uint32_t)min(max(r.len - 1, (int64_t)0), (int64_t)0x7ffffffe);
  const uint32_t blocks = r.len > 0 ? fast_div(last, p.by_block_size) + 1 : 0;
  r.ok = listed && cached >= 0 && added >= 0 && r.len <= 0x7fffffff && blocks <= r.pages && blocks <= p.max_blocks;
  return r;
}

// Exclusive prefix sum of `mine` over the workgroup and the workgroup's sum.
// 64 bits in two 32-bit scans: of the low 16 bits and of what lies above.
__device__ __forceinline__ uint64_t group_scan(uint64_t mine, uint64_t* sums, uint32_t t, uint64_t* total) {
  const int lo = (int)(mine & 0xffffu), hi = (int)(mine >> 16);
  const uint64_t upto = (uint64_t)(uint32_t)wave_scan(lo) + ((uint64_t)(uint32_t)wave_scan(hi) << 16);
  if ((t & 63) == 63) sums[t >> 6] = upto;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (uint32_t i = 0; i < kThreads / 64; ++i) {
    before += i < t >> 6 ? sums[i] : 0;
    all += sums[i];
  }
  *total = all;
  return before + upto - mine;
}

__device__ __forceinline__ uint32_t capped(uint64_t start) { return (uint32_t)min(start, (uint64_t)0x7fffffff); }

__device__ __forceinline__ void write_tables(const StepTablesParams& p, uint32_t group) {
  const uint32_t entries = p.batch * p.max_blocks, first = group * kStepEntries + threadIdx.x;
#pragma unroll
  for (uint32_t i = 0; i < kStepEntries; i += kThreads) {
    const uint32_t e = first + i;
    if (e >= entries) return;
    const uint32_t b = fast_div(e, p.by_max_blocks), j = e - b * p.max_blocks;
    const int32_t lo = p.page_starts[b], hi = p.page_starts[b + 1];
    const bool there = lo >= 0 && hi >= lo && (uint32_t)hi <= p.n_page_ids && j < (uint32_t)(hi - lo);
    p.block_tables[e] = there ? p.page_ids[(uint32_t)lo + j] : -1;
  }
}

__global__ __launch_bounds__(kThreads) void step_tables_kernel(const StepTablesParams p) {
  if (blockIdx.x >= p.token_groups) {
    write_tables(p, blockIdx.x - p.token_groups);
    return;
  }
  __shared__ uint32_t starts[kChunk + 1];
  __shared__ uint64_t sums[2][kThreads / 64];  // chunks take them in turn
  const uint32_t t = threadIdx.x;
  const bool lengths = blockIdx.x == 0;  // this workgroup writes these as well
  const uint32_t first = blockIdx.x * kStepTokens, end = min(first + kStepTokens, p.max_tokens);
  int32_t slot[kPer], position[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) slot[i] = position[i] = -1;
  uint64_t before = 0;  // tokens of the requests before this chunk's
  for (uint32_t b0 = 0, turn = 0; b0 < p.batch && (lengths || before < end); b0 += kChunk, turn ^= 1) {
    int32_t added[kPer];
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t b = b0 + kPer * t + i;
      added[i] = b < p.batch ? (p.new_lens ? p.new_lens[b] : 1) : 0;
      mine += (uint32_t)max(added[i], 0);
    }
    uint64_t total, at = before + group_scan(mine, sums[turn], t, &total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t b = b0 + kPer * t + i;
      starts[kPer * t + i] = capped(at);  // beyond any token: a thread's tokens are below max_tokens
      if (lengths && b < p.batch) {
        const uint64_t past = at + (uint32_t)max(added[i], 0);
        const Request r = request(p, b, added[i]);
        p.token_starts[b] = (int32_t)capped(at);
        p.seq_lens[b] = r.ok && past <= p.max_tokens ? (int32_t)r.len : -1;
        if (b + 1 == p.batch) p.token_starts[p.batch] = (int32_t)capped(past);
      }
      at += (uint32_t)max(added[i], 0);
    }
    if (t == kThreads - 1) starts[kChunk] = capped(at);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t token = first + i * kThreads + t;
      if (token >= end || token < before || token >= before + total) continue;
      // the last request that starts at or before the token: an empty one
      // starts where the next does
      uint32_t lo = 0, hi = kChunk;  // starts[lo] <= token < starts[hi]
#pragma unroll
      for (int step = 0; step < 10; ++step) {
        const uint32_t mid = (lo + hi) / 2;
        if (starts[mid] <= token) lo = mid;
        else hi = mid;
      }
      const uint32_t b = b0 + lo, row = token - starts[lo];
      const int32_t n = p.new_lens ? p.new_lens[b] : 1;
      const Request r = request(p, b, n);
      if (!r.ok || starts[lo] + (uint32_t)n > p.max_tokens) continue;
      const uint32_t pos = (uint32_t)(r.len - n) + row;
      const uint32_t block = fast_div(pos, p.by_block_size);
      const int32_t page = p.page_ids[r.first + block];
      const int64_t s = (int64_t)page * p.block_size + (pos - block * p.block_size);
      position[i] = (int32_t)pos;
      slot[i] = page >= 0 && s <= 0x7fffffff ? (int32_t)s : -1;
    }
    before += total;
    __syncthreads();  // the next chunk rewrites the starts
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t token = first + i * kThreads + t;
    if (token >= end) continue;
    p.slots[token] = slot[i];
    p.positions[token] = position[i];
  }
}

}  // namespace

hipError_t launch_step_tables(StepTablesParams p, hipStream_t stream) {
  p.token_groups = (p.max_tokens + kStepTokens - 1) / kStepTokens;
  const uint32_t table_groups = (p.batch * p.max_blocks + kStepEntries - 1) / kStepEntries;
  hipLaunchKernelGGL(step_tables_kernel, dim3(p.token_groups + table_groups), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace pbe
