// gfx950 step tables: what the host's build_block_tables, build_seq_lens and
// build_slot_mapping make, from page lists and lengths in device memory, for
// requests that add any number of tokens.
//   start_b = sum over i < b of max(new_i, 0), len_b = cached_b + new_b;
//   token t of request b: position p = cached_b + t - start_b,
//   slot = page[p / block_size] * block_size + p % block_size.
//
// One launch. A workgroup writes the slots and positions of 256 tokens, or
// 1,024 entries of the tables, which need no sums; the first one writes
// lengths and starts as well. The tokens' requests follow from a prefix sum
// over new_lens, which every token workgroup makes for itself, 1,024 requests
// at a time, up to the last request of its tokens: the lengths are a few KB
// out of L2, and a second launch would cost more than the sum.
//
// What bounds it: the launch and three round trips (lengths and lists, page,
// store). us in a graph: one request 3.0, 256 decoding ones with tables of 440
// blocks 3.7, 48 requests up to 32,768 tokens that add 12,288 3.9. With four
// tokens a thread, one after another, the last took 6.0, side by side 5.1 and the
// second 4.6.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_device.h"
#include "step_kernels.h"

namespace pbe {
namespace {

constexpr int kThreads = 256, kPer = 4, kChunk = kThreads * kPer;  // requests summed at a time
static_assert(kStepTokens == kThreads, "a token a thread");

// Whether a request's lengths and pages make sense, and its length then.
__device__ __forceinline__ bool fits(const StepTablesParams& p, int32_t cached, int32_t added, int32_t lo, int32_t hi) {
  if (lo < 0 || hi < lo || (uint32_t)hi > p.n_page_ids || cached < 0 || added < 0 || (int64_t)cached + added > 0x7fffffff) return false;
  const uint32_t len = (uint32_t)cached + (uint32_t)added;
  const uint32_t blocks = len ? fast_div(len - 1, p.by_block_size) + 1 : 0;
  return blocks <= (uint32_t)(hi - lo) && blocks <= p.max_blocks;
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
  constexpr int kEach = kStepEntries / kThreads;  // a thread's entries, in flight together
  const uint32_t entries = p.batch * p.max_blocks, first = group * kStepEntries + threadIdx.x;
  uint32_t j[kEach];
  int32_t lo[kEach], hi[kEach], id[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const uint32_t e = min(first + i * kThreads, entries - 1), b = fast_div(e, p.by_max_blocks);
    j[i] = e - b * p.max_blocks;
    lo[i] = p.page_starts[b];
    hi[i] = p.page_starts[b + 1];
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool there = lo[i] >= 0 && hi[i] >= lo[i] && (uint32_t)hi[i] <= p.n_page_ids && j[i] < (uint32_t)(hi[i] - lo[i]);
    id[i] = there ? p.page_ids[(uint32_t)lo[i] + j[i]] : -1;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (first + i * kThreads < entries) p.block_tables[first + i * kThreads] = id[i];
}

__global__ __launch_bounds__(kThreads) void step_tables_kernel(const StepTablesParams p) {
  if (blockIdx.x >= p.token_groups) {
    write_tables(p, blockIdx.x - p.token_groups);
    return;
  }
  // Of the chunk's requests: first row, cached tokens and first page (-1: a wrong one).
  __shared__ uint32_t starts[kChunk + 1];
  __shared__ int32_t cached_of[kChunk], page_of[kChunk];
  __shared__ uint64_t sums[2][kThreads / 64];  // chunks take them in turn
  const uint32_t t = threadIdx.x;
  const bool lengths = blockIdx.x == 0;  // this workgroup writes these as well
  const uint32_t token = blockIdx.x * kStepTokens + t, end = min((blockIdx.x + 1) * kStepTokens, p.max_tokens);
  int32_t slot = -1, position = -1;
  uint64_t before = 0;  // tokens of the requests before this chunk's
  for (uint32_t b0 = 0, turn = 0; b0 < p.batch && (lengths || before < end); b0 += kChunk, turn ^= 1) {
    // All that is known of a request is asked for at once: one round trip.
    int32_t added[kPer], cached[kPer], lo[kPer], hi[kPer];
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t b = b0 + kPer * t + i;
      const bool there = b < p.batch;
      added[i] = !there ? 0 : p.new_lens ? p.new_lens[b] : 1;
      cached[i] = there ? p.cached_lens[b] : 0;
      lo[i] = there ? p.page_starts[b] : 0;
      hi[i] = there ? p.page_starts[b + 1] : 0;
      mine += (uint32_t)max(added[i], 0);
    }
    uint64_t total, at = before + group_scan(mine, sums[turn], t, &total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t r = kPer * t + i, b = b0 + r;
      const uint64_t past = at + (uint32_t)max(added[i], 0);
      const bool ok = fits(p, cached[i], added[i], lo[i], hi[i]) && past <= p.max_tokens;
      starts[r] = capped(at);  // beyond any token: a thread's tokens are below max_tokens
      cached_of[r] = cached[i];
      page_of[r] = ok ? lo[i] : -1;
      if (lengths && b < p.batch) {
        p.token_starts[b] = (int32_t)capped(at);
        p.seq_lens[b] = ok ? cached[i] + added[i] : -1;
        if (b + 1 == p.batch) p.token_starts[p.batch] = (int32_t)capped(past);
      }
      at = past;
    }
    if (t == kThreads - 1) starts[kChunk] = capped(at);
    __syncthreads();
    if (token < end && token >= before && token < before + total) {
      // the last request that starts at or before the token (an empty one
      // starts where the next does): starts[low] <= token < starts[high]
      uint32_t low = 0, high = min(p.batch - b0, (uint32_t)kChunk);
      for (uint32_t span = high; span > 1; span = (span + 1) / 2) {  // high - low is at most that
        const uint32_t mid = (low + high) / 2;                       // low, where the two are next to each other
        const bool down = starts[mid] > token;
        high = down ? mid : high;
        low = down ? low : mid;
      }
      if (page_of[low] >= 0) {
        const uint32_t pos = (uint32_t)cached_of[low] + token - starts[low], block = fast_div(pos, p.by_block_size);
        const int32_t page = p.page_ids[(uint32_t)page_of[low] + block];
        const int64_t s = (int64_t)page * p.block_size + (pos - block * p.block_size);
        position = (int32_t)pos;
        slot = page >= 0 && s <= 0x7fffffff ? (int32_t)s : -1;
      }
    }
    before += total;
    __syncthreads();  // the next chunk rewrites the starts
  }
  if (token < end) {
    p.slots[token] = slot;
    p.positions[token] = position;
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
