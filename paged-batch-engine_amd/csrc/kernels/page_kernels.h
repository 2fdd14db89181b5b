// Internal interface of the page movers: the next step's tables from the last
// one's (forks, ends, growth), and pages moved to the front of their pool.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernels.h"  // FastDiv

namespace pbe {

constexpr int kPagePlanes = 112;         // pools of a call
constexpr int kPageBases = 224;          // their allocations
constexpr int32_t kMostPages = 1 << 20;  // bits of the plan's map, in LDS
constexpr int32_t kMostRows = 0x7fffffff - 1023;  // the plan counts 1,024 rows at a time
constexpr uint32_t kPageSlice = 16384;   // bytes that a workgroup copies at a time
constexpr uint32_t kPageEntries = 1024;  // table entries of a workgroup
constexpr int kPageHeader = 16;          // first words of a workspace

// Where page i of the pool lies in each plane.
struct PagePlanes {
  uint64_t base[kPageBases];         // of a plane's segments, from first[plane] on
  uint32_t page_bytes[kPagePlanes];
  uint32_t seg_pages[kPagePlanes];
  uint32_t start[kPagePlanes];       // slices of a page before this plane's
  uint16_t first[kPagePlanes];
  uint32_t n, slices;                // planes; slices of a page
};

struct ForkParams {
  const int32_t* tables_in;
  const int32_t* lens_in;
  const int32_t* parents;
  const int32_t* new_lens;   // or null: one each
  const int32_t* reserved;   // or null
  int32_t* tables_out;
  int32_t* lens_out;
  int32_t* counts;
  // workspace
  uint32_t* header;          // [0]: pages to copy
  int32_t* firsts;           // [rows_in] first child of a row
  uint32_t* base;            // [rows_out] a child's first fresh page; ~0: none for it
  int32_t* shared;           // [rows_out] entries that are its parent's
  int32_t* wanted;           // [rows_out] entries in all
  int32_t* copies;           // [rows_out] children whose first fresh page is a copy
  int32_t* fresh;            // [n_pages]
  int32_t n_pages, stride, rows_in, rows_out, max_blocks, block_size;
  uint32_t fills, copiers;   // workgroups of the second launch
  FastDiv by_stride, by_block_size, by_max_blocks;
};

struct CompactParams {
  const int32_t* tables_in;
  const int32_t* reserved;   // or null
  int32_t* tables_out;
  int32_t* moved_to;         // [n_pages]
  int32_t* counts;
  // workspace
  uint32_t* header;          // [0]: pages to copy
  int32_t* sources;          // [n_pages]
  int32_t* places;           // [n_pages]
  int32_t n_pages, stride;
  uint32_t entries;
  uint32_t fills, copiers;
  FastDiv by_stride;
};

hipError_t launch_fork_pages(ForkParams p, const PagePlanes& planes, int64_t units, hipStream_t stream);
hipError_t launch_compact_pages(CompactParams p, const PagePlanes& planes, int64_t units, hipStream_t stream);

}  // namespace pbe
