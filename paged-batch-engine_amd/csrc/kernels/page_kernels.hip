// Page movers. Two launches each: one workgroup makes the plan from the tables (which
// pages are held, which ones are free, what has to be copied), then workgroups write
// the tables and copy pages side by side.
//
// Held pages are bits in LDS (2^20 pages: 128 KiB), marked from the tables themselves, so
// a call needs no counts kept from one step to the next, and gives the same answer
// whatever order the marks come in. Fresh pages are the zero bits, counted by a prefix
// sum: the lowest ones, in order.
//
// Bound: the plan, for small pools: a chain of table reads, marks and scans in one
// workgroup, 6 to 9 us for a fork and 4 to 5 for a compaction (kernel trace), which several
// workgroups with a pass over the grid between them would not shorten; then the copies, two
// passes over the pages' bytes at HBM's rate. One page of 458,752 bytes forked four ways
// 10.4 us, 64 x 4 drafts forked 18.9 us, 96 pages compacted 9.2 us, 200 of 1,024 pages of
// 917,504 bytes moved 72 us (5.1 TB/s read and written; a large library copy 6.6 TB/s).
// One workgroup's plan grows with the tables: 256 rows of 2,048 entries over 2^17 pages
// take a fork 128 us and a compaction that moves nothing 196.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "decode_device.h"
#include "page_kernels.h"
#include "xcd_order.h"

namespace pbe {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
static_assert(kMostRows <= 0x7fffffff - (kPlanThreads - 1), "a row's number and the next turn's fit 31 bits");
constexpr int kWords = kMostPages / 32;
constexpr int kForkRows = 3584;  // whose first children fit LDS beside the map; more take the workspace
constexpr uint32_t kCopyGroup = 192 * 1024 / kPageSlice;  // slices that an XCD takes one after another
constexpr int kCopyThreads = 256, kCopyEach = kPageSlice / (16 * kCopyThreads);

// Page of an entry, or -1 where it names none of the pool's.
__device__ __forceinline__ int page_of(int id, int n_pages, int stride, const FastDiv& by_stride) {
  if (id < 0) return -1;
  const uint32_t page = fast_div((uint32_t)id, by_stride);
  return page < (uint32_t)n_pages && page * (uint32_t)stride == (uint32_t)id ? (int)page : -1;
}

// Exclusive prefix sum over the workgroup, and the sum of all.
__device__ __forceinline__ uint32_t plan_scan(uint32_t mine, uint32_t* sums, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t upto = (uint32_t)wave_scan((int)mine);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (uint32_t i = 0; i < kPlanWaves; ++i) {
    before += i < wave ? sums[i] : 0;
    all += sums[i];
  }
  __syncthreads();
  *total = all;
  return before + upto - mine;
}

// What child i wants of its parent. parent -1: it has none; bad: lengths or table
// make no sense.
struct Child {
  int parent = -1, len = 0, kept = 0, want = 0;
  bool bad = false;
};
__device__ __forceinline__ Child child_of(const ForkParams& p, int i) {
  Child c;
  const int parent = p.parents[i], more = p.new_lens ? p.new_lens[i] : 1;
  if (parent < 0) return c;
  if (parent >= p.rows_in) {
    c.bad = true;
    return c;
  }
  const int len = p.lens_in[parent];
  if (len < 0 || more < 0 || (int64_t)len + more > 0x7fffffff) {
    c.bad = true;
    return c;
  }
  auto blocks = [&](uint32_t n) { return n ? (int)fast_div(n - 1, p.by_block_size) + 1 : 0; };
  c.kept = blocks((uint32_t)len);
  c.want = blocks((uint32_t)len + (uint32_t)more);
  if (c.want > p.max_blocks) {
    c.bad = true;
    return c;
  }
  c.parent = parent;
  c.len = len;
  return c;
}

// Bits of pages that others hold, and of those that there are not.
__device__ __forceinline__ uint64_t held_elsewhere(const int32_t* reserved, int n_pages, int first, int lane) {
  const int i = first + lane;
  return __ballot(i >= n_pages || (reserved && reserved[i] != 0));
}

__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(const ForkParams p) {
  __shared__ uint32_t held[kWords];
  __shared__ int32_t firsts[kForkRows];                     // a row's first child
  __shared__ int32_t row_of[kPlanThreads], kept_of[kPlanThreads];  // of the children whose parents are marked
  __shared__ uint32_t sums[kPlanWaves];
  __shared__ int marked;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int words = (p.n_pages + 63) / 64 * 2;
  const bool few = p.rows_in <= kForkRows;
  Child mine = t < p.rows_out ? child_of(p, t) : Child();   // the first kPlanThreads children's
  for (int w = wave; w < words / 2; w += kPlanWaves) {
    const uint64_t bits = held_elsewhere(p.reserved, p.n_pages, w * 64, lane);
    if (lane == 0) held[2 * w] = (uint32_t)bits;
    if (lane == 1) held[2 * w + 1] = (uint32_t)(bits >> 32);
  }
  for (int i = t; i < p.rows_in; i += kPlanThreads) {
    if (few) firsts[i] = 0x7fffffff;
    else p.firsts[i] = 0x7fffffff;
  }
  if (!few) __threadfence();
  __syncthreads();
  auto child = [&](int i) { return i < kPlanThreads ? mine : i < p.rows_out ? child_of(p, i) : Child(); };
  for (int i = t; i < p.rows_out; i += kPlanThreads) {
    const Child c = child(i);
    if (c.parent < 0) continue;
    if (few) atomicMin(&firsts[c.parent], i);
    else atomicMin(p.firsts + c.parent, i);
  }
  if (!few) __threadfence();
  __syncthreads();
  auto first_of = [&](int parent) {
    return few ? firsts[parent] : __hip_atomic_load(p.firsts + parent, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  // What the children's parents hold, each parent once: kPlanThreads children at a
  // time are listed, then waves mark the rows listed, kMarks of them together.
  for (int i0 = 0; i0 < p.rows_out; i0 += kPlanThreads) {
    if (t == 0) marked = 0;
    __syncthreads();
    const Child c = child(i0 + t);
    if (c.parent >= 0 && first_of(c.parent) == i0 + t) {
      const int at = atomicAdd(&marked, 1);  // in any order: bits are set
      row_of[at] = c.parent;
      kept_of[at] = c.kept;
    }
    __syncthreads();
    constexpr int kMarks = 4;
    for (int r = wave * kMarks; r < marked; r += kPlanWaves * kMarks) {
      int most = 0;
#pragma unroll
      for (int e = 0; e < kMarks; ++e) most = max(most, r + e < marked ? kept_of[r + e] : 0);
      for (int k = lane; k < most; k += 64) {
        int id[kMarks];
#pragma unroll
        for (int e = 0; e < kMarks; ++e) id[e] = r + e < marked && k < kept_of[r + e] ? p.tables_in[(int64_t)row_of[r + e] * p.max_blocks + k] : -1;
#pragma unroll
        for (int e = 0; e < kMarks; ++e) {
          const int page = page_of(id[e], p.n_pages, p.stride, p.by_stride);
          if (page >= 0) atomicOr(&held[page / 32], 1u << (page % 32));
        }
      }
    }
    __syncthreads();
  }
  const int each = (words + kPlanThreads - 1) / kPlanThreads, from = min(words, t * each), to = min(words, from + each);
  uint32_t open = 0;
  for (int w = from; w < to; ++w) open += 32 - __popc(held[w]);
  uint32_t available;
  uint32_t rank = plan_scan(open, sums, &available);
  // needs in the children's order
  uint32_t needed = 0, copied = 0;
  for (int i0 = 0; i0 < p.rows_out; i0 += kPlanThreads) {
    const int i = i0 + t;
    Child c = child(i);
    bool copy = c.parent >= 0 && c.kept * (int64_t)p.block_size != c.len && first_of(c.parent) != i;
    // a copy needs a page to copy from
    if (copy && page_of(p.tables_in[(int64_t)c.parent * p.max_blocks + c.kept - 1], p.n_pages, p.stride, p.by_stride) < 0)
      c = Child(), c.bad = true, copy = false;
    const uint32_t need = c.parent >= 0 ? (uint32_t)(c.want - c.kept + copy) : 0;
    uint32_t total, copies;
    const uint32_t at = needed + plan_scan(need, sums, &total);
    const bool ok = c.parent >= 0 && (need == 0 || at + need <= available);
    const uint32_t place = copied + plan_scan(ok && copy, sums, &copies);
    if (i < p.rows_out) {
      p.base[i] = ok ? at : ~0u;
      p.shared[i] = c.kept - copy;
      p.wanted[i] = c.want;
      p.lens_out[i] = ok ? c.len : c.parent >= 0 || c.bad ? -1 : 0;
      if (ok && copy) p.copies[place] = i;
    }
    needed += total;
    copied += copies;
  }
  const uint32_t listed = min(needed, available);
  for (int w = from; w < to && rank < listed; ++w)
    for (uint32_t free = ~held[w]; free && rank < listed; free &= free - 1) p.fresh[rank++] = w * 32 + __builtin_ctz(free);
  if (t == 0) {
    p.header[0] = copied;
    p.counts[0] = (int32_t)needed;
    p.counts[1] = (int32_t)available;
  }
}

// Copies slice `slice` of page `from` to page `to`.
__device__ __forceinline__ void copy_slice(const PagePlanes& planes, uint32_t slice, uint32_t from, uint32_t to) {
  uint32_t low = 0, high = planes.n;
  while (high - low > 1) {
    const uint32_t mid = (low + high) / 2;
    const bool down = planes.start[mid] > slice;
    high = down ? mid : high;
    low = down ? low : mid;
  }
  const uint32_t bytes = planes.page_bytes[low], begin = (slice - planes.start[low]) * kPageSlice, seg = planes.seg_pages[low];
  auto at = [&](uint32_t page) { return planes.base[planes.first[low] + page / seg] + (uint64_t)(page % seg) * bytes + begin; };
  const uint64_t src = at(from), dst = at(to);
  const uint32_t n = min(bytes - begin, kPageSlice);
  u32x4 x[kCopyEach];
#pragma unroll
  for (int i = 0; i < kCopyEach; ++i) {
    const uint32_t o = (i * kCopyThreads + threadIdx.x) * 16;
    if (o < n) x[i] = __builtin_nontemporal_load((PBE_GLOBAL const u32x4*)(src + o));
  }
#pragma unroll
  for (int i = 0; i < kCopyEach; ++i) {
    const uint32_t o = (i * kCopyThreads + threadIdx.x) * 16;
    if (o < n) __builtin_nontemporal_store(x[i], (PBE_GLOBAL u32x4*)(dst + o));
  }
}

__global__ __launch_bounds__(kCopyThreads) void fork_move_kernel(const ForkParams p, const PagePlanes planes) {
  if (blockIdx.x >= p.copiers) {
    const uint32_t entries = (uint32_t)p.rows_out * (uint32_t)p.max_blocks;
#pragma unroll
    for (uint32_t k = 0; k < kPageEntries / kCopyThreads; ++k) {
      const uint32_t e = (blockIdx.x - p.copiers) * kPageEntries + k * kCopyThreads + threadIdx.x;
      if (e >= entries) return;
      const uint32_t i = fast_div(e, p.by_max_blocks), j = e - i * (uint32_t)p.max_blocks;
      const uint32_t base = p.base[i];
      int id = -1;
      if (base != ~0u) {
        const int shared = p.shared[i];
        if ((int)j < shared) id = p.tables_in[(int64_t)p.parents[i] * p.max_blocks + j];
        else if ((int)j < p.wanted[i]) id = p.fresh[base + j - (uint32_t)shared] * p.stride;
      }
      p.tables_out[e] = id;
    }
    return;
  }
  const uint64_t units = (uint64_t)p.header[0] * planes.slices;
  for (uint64_t u = xcd_grouped(blockIdx.x, p.copiers, kCopyGroup); u < units; u += p.copiers) {
    const uint32_t m = (uint32_t)(u / planes.slices), child = (uint32_t)p.copies[m];
    const int shared = p.shared[child];
    const int from = page_of(p.tables_in[(int64_t)p.parents[child] * p.max_blocks + shared], p.n_pages, p.stride, p.by_stride);
    copy_slice(planes, (uint32_t)(u - (uint64_t)m * planes.slices), (uint32_t)from, (uint32_t)p.fresh[p.base[child]]);
  }
}

// Pages in use that nobody else holds, M of them, take the first M places that
// nobody else holds: those among them stay, the others go to the places that are
// left, both in their order.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(const CompactParams p) {
  __shared__ uint32_t used[kWords];
  __shared__ uint32_t sums[kPlanWaves];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int groups = (p.n_pages + 63) / 64, each = (groups + kPlanWaves - 1) / kPlanWaves;  // of 64 pages; a wave's
  const int from = min(groups, wave * each), to = min(groups, from + each);
  for (int w = t; w < 2 * groups; w += kPlanThreads) used[w] = 0;
  __syncthreads();
  for (uint32_t e = t; e < p.entries; e += kPlanThreads) {
    const int page = page_of(p.tables_in[e], p.n_pages, p.stride, p.by_stride);
    if (page >= 0) atomicOr(&used[page / 32], 1u << (page % 32));
  }
  __syncthreads();
  auto bits = [&](int g) { return (uint64_t)used[2 * g] | (uint64_t)used[2 * g + 1] << 32; };
  // lane 0 of a wave carries its sums into the scans
  uint32_t open = 0, moving = 0, total_open, total;
  for (int g = from; g < to; ++g) {
    const uint64_t held = held_elsewhere(p.reserved, p.n_pages, g * 64, lane);
    open += __popcll(~held);
    moving += __popcll(bits(g) & ~held);
  }
  const uint32_t open_before = plan_scan(lane == 0 ? open : 0, sums, &total_open);
  (void)plan_scan(lane == 0 ? moving : 0, sums, &total);
  uint32_t place = (uint32_t)__builtin_amdgcn_readfirstlane((int)open_before);
  const uint64_t below = (1ull << lane) - 1;
  // Of 64 pages: whether this lane's is among the first `total` open ones.
  auto front_of = [&](uint64_t held, uint32_t at) { return __ballot(!(held >> lane & 1) && at + __popcll(~held & below) < total); };
  uint32_t out = 0, in = 0;
  for (int g = from, at = place; g < to; ++g) {
    const uint64_t held = held_elsewhere(p.reserved, p.n_pages, g * 64, lane), front = front_of(held, at);
    out += __popcll(bits(g) & ~held & ~front);
    in += __popcll(~bits(g) & front);
    at += __popcll(~held);
  }
  uint32_t movers, holes;
  uint32_t out_at = (uint32_t)__builtin_amdgcn_readfirstlane((int)plan_scan(lane == 0 ? out : 0, sums, &movers));
  uint32_t in_at = (uint32_t)__builtin_amdgcn_readfirstlane((int)plan_scan(lane == 0 ? in : 0, sums, &holes));
  for (int g = from; g < to; ++g) {
    const uint64_t held = held_elsewhere(p.reserved, p.n_pages, g * 64, lane), front = front_of(held, place);
    const uint64_t leaves = bits(g) & ~held & ~front, takes = ~bits(g) & front;
    const int page = g * 64 + lane;
    if (leaves >> lane & 1) p.sources[out_at + __popcll(leaves & below)] = page;
    else if (page < p.n_pages) p.moved_to[page] = bits(g) >> lane & 1 ? page : -1;
    if (takes >> lane & 1) p.places[in_at + __popcll(takes & below)] = page;
    out_at += __popcll(leaves);
    in_at += __popcll(takes);
    place += __popcll(~held);
  }
  __threadfence_block();
  __syncthreads();
  for (uint32_t k = t; k < movers; k += kPlanThreads) p.moved_to[p.sources[k]] = p.places[k];
  if (t == 0) {
    p.header[0] = movers;
    p.counts[0] = (int32_t)total;
    p.counts[1] = (int32_t)movers;
  }
}

__global__ __launch_bounds__(kCopyThreads) void compact_move_kernel(const CompactParams p, const PagePlanes planes) {
  if (blockIdx.x >= p.copiers) {
#pragma unroll
    for (uint32_t k = 0; k < kPageEntries / kCopyThreads; ++k) {
      const uint32_t e = (blockIdx.x - p.copiers) * kPageEntries + k * kCopyThreads + threadIdx.x;
      if (e >= p.entries) return;
      const int id = p.tables_in[e], page = page_of(id, p.n_pages, p.stride, p.by_stride);
      p.tables_out[e] = page >= 0 ? p.moved_to[page] * p.stride : id;
    }
    return;
  }
  const uint64_t units = (uint64_t)p.header[0] * planes.slices;
  for (uint64_t u = xcd_grouped(blockIdx.x, p.copiers, kCopyGroup); u < units; u += p.copiers) {
    const uint32_t m = (uint32_t)(u / planes.slices);
    copy_slice(planes, (uint32_t)(u - (uint64_t)m * planes.slices), (uint32_t)p.sources[m], (uint32_t)p.places[m]);
  }
}

// Workgroups that copy: 64 a compute unit, and no more than there can be work for (those
// without any end at once). Of a thousand pages: 8 a unit 84.5 us, 32 72.7, 64 72.1, 256
// 73.4; 128 threads 117.6, 512 71.3 to 74, 1,024 84 to 107; plain instead of non-temporal
// accesses 94; an XCD's group of slices of 192 KiB to 1 MiB 71.2 to 72.1.
uint32_t copiers(int64_t pages, const PagePlanes& planes, int64_t units) {
  return (uint32_t)std::max<int64_t>(1, std::min<int64_t>(64 * units, pages * (int64_t)planes.slices));
}

}  // namespace

hipError_t launch_fork_pages(ForkParams p, const PagePlanes& planes, int64_t units, hipStream_t stream) {
  p.copiers = copiers(p.rows_out, planes, units);
  p.fills = ((uint32_t)p.rows_out * (uint32_t)p.max_blocks + kPageEntries - 1) / kPageEntries;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  hipLaunchKernelGGL(fork_move_kernel, dim3(p.copiers + p.fills), dim3(kCopyThreads), 0, stream, p, planes);
  return hipGetLastError();
}

hipError_t launch_compact_pages(CompactParams p, const PagePlanes& planes, int64_t units, hipStream_t stream) {
  p.copiers = copiers(p.n_pages / 2, planes, units);
  p.fills = (p.entries + kPageEntries - 1) / kPageEntries;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  hipLaunchKernelGGL(compact_move_kernel, dim3(p.copiers + p.fills), dim3(kCopyThreads), 0, stream, p, planes);
  return hipGetLastError();
}

}  // namespace pbe
