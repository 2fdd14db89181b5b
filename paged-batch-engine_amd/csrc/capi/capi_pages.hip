// C ABI: the page movers (requests that fork, end and grow; pages moved to the
// front of their pool).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <vector>

#include "capi_internal.h"
#include "../kernels/page_kernels.h"

using namespace pbe_capi;

namespace {

struct Array {
  const void* at;
  uint64_t bytes;
  bool out;
};

// Checks the pool's planes and lays them out for the kernels.
int planes_of(const pbe_page_plane* planes, int32_t n_planes, int32_t n_pages, pbe::PagePlanes* out) {
  if (!planes || n_planes <= 0) return fail(PBE_ERR_INVALID, "a pool needs at least one plane");
  if (n_planes > pbe::kPagePlanes) return fail(PBE_ERR_UNSUPPORTED, "at most %d planes a call", pbe::kPagePlanes);
  uint32_t bases = 0, slices = 0;
  for (int32_t i = 0; i < n_planes; ++i) {
    const pbe_arena_view& v = planes[i].memory;
    const uint64_t page = planes[i].page_bytes;
    if (!view_ok(&v)) return fail(PBE_ERR_INVALID, "invalid view of plane %d", (int)i);
    if (page == 0 || page % 16 || page > 0x40000000ull) return fail(PBE_ERR_INVALID, "a plane's pages must be multiples of 16 bytes of at most 1 GiB");
    if (v.nseg > 1 && v.segment_bytes % page) return fail(PBE_ERR_INVALID, "segments must hold whole pages");
    if (v.bytes / page < (uint64_t)n_pages) return fail(PBE_ERR_INVALID, "plane %d holds %llu of %d pages", (int)i, (unsigned long long)(v.bytes / page), (int)n_pages);
    if (bases + v.nseg > (uint32_t)pbe::kPageBases) return fail(PBE_ERR_UNSUPPORTED, "at most %d segments a call", pbe::kPageBases);
    out->page_bytes[i] = (uint32_t)page;
    out->seg_pages[i] = (uint32_t)std::min<uint64_t>(v.nseg > 1 ? v.segment_bytes / page : 0x7fffffffu, 0x7fffffffu);
    out->start[i] = slices;
    out->first[i] = (uint16_t)bases;
    for (uint32_t s = 0; s < v.nseg; ++s) {
      if (reinterpret_cast<uintptr_t>(v.base[s]) % 16) return fail(PBE_ERR_INVALID, "planes must be 16-byte aligned");
      out->base[bases++] = reinterpret_cast<uint64_t>(v.base[s]);
    }
    slices += (uint32_t)((page + pbe::kPageSlice - 1) / pbe::kPageSlice);
  }
  out->n = (uint32_t)n_planes;
  out->slices = slices;
  return PBE_OK;
}

// Alignment, overlaps and places of the arrays and planes of a call.
int check_memory(const pbe_page_plane* planes, int32_t n_planes, std::initializer_list<Array> arrays, int device) {
  std::vector<Span> pools;
  for (int32_t i = 0; i < n_planes; ++i) {
    const pbe_arena_view& v = planes[i].memory;
    for (uint32_t s = 0; s < v.nseg; ++s) pools.push_back({v.base[s], std::min(v.segment_bytes, v.bytes - (uint64_t)s * v.segment_bytes)});
  }
  for (size_t i = 0; i < pools.size(); ++i)
    for (size_t k = 0; k < i; ++k)
      if (meet(pools[i], pools[k])) return fail(PBE_ERR_INVALID, "planes must lie apart from each other");
  for (const Array& a : arrays) {
    if (reinterpret_cast<uintptr_t>(a.at) % 4) return fail(PBE_ERR_INVALID, "tables and lists must be 4-byte aligned");
    for (const Array& o : arrays)
      if (&a != &o && o.out && meet({a.at, a.bytes}, {o.at, o.bytes})) return fail(PBE_ERR_INVALID, "an output overlaps another array");
    for (const Span& pool : pools)
      if (meet(pool, {a.at, a.bytes})) return fail(PBE_ERR_INVALID, "tables and lists must lie apart from the planes");
  }
  PBE_DEVICE_SCOPE(device);
  std::vector<Range> known;
  for (const Array& a : arrays)
    if (a.at && a.bytes && !accessible(a.at, a.bytes, device, &known)) return fail(PBE_ERR_INVALID, "operands must be memory of device %d", device);
  for (int32_t i = 0; i < n_planes; ++i)
    if (!view_accessible(planes[i].memory, device, &known)) return fail(PBE_ERR_INVALID, "planes must be memory of device %d", device);
  return PBE_OK;
}

int check_pool(int32_t n_pages, int32_t id_stride) {
  if (n_pages <= 0 || id_stride <= 0) return fail(PBE_ERR_INVALID, "n_pages and id_stride > 0");
  if (n_pages > pbe::kMostPages) return fail(PBE_ERR_UNSUPPORTED, "at most %d pages", (int)pbe::kMostPages);
  if ((int64_t)n_pages * id_stride > INT32_MAX) return fail(PBE_ERR_INVALID, "n_pages * id_stride must be at most INT32_MAX");
  return PBE_OK;
}

}  // namespace

extern "C" {

uint64_t pbe_fork_pages_workspace_bytes(int32_t n_pages, int32_t rows_in, int32_t rows_out) {
  if (n_pages <= 0 || rows_in <= 0 || rows_out <= 0) return 0;
  return 4ull * (pbe::kPageHeader + (uint64_t)n_pages + (uint64_t)rows_in + 4ull * (uint64_t)rows_out);
}

int pbe_fork_pages(const pbe_page_plane* planes, int32_t n_planes, int32_t n_pages,
                   int32_t id_stride, int32_t block_size, const int32_t* tables_in,
                   const int32_t* lens_in, int32_t rows_in, const int32_t* parents,
                   const int32_t* new_lens, int32_t rows_out, int32_t max_blocks_per_seq,
                   const int32_t* reserved, int32_t* tables_out, int32_t* lens_out,
                   int32_t* counts, void* workspace, uint64_t workspace_bytes, int device,
                   void* stream) {
  if (block_size <= 0 || rows_in <= 0 || rows_out <= 0 || max_blocks_per_seq <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "block_size, rows and max_blocks_per_seq > 0 and a device");
  int rc = check_pool(n_pages, id_stride);
  if (rc != PBE_OK) return rc;
  if (std::max(rows_in, rows_out) > pbe::kMostRows) return fail(PBE_ERR_INVALID, "at most %d rows", (int)pbe::kMostRows);
  if ((int64_t)std::max(rows_in, rows_out) * max_blocks_per_seq > INT32_MAX)
    return fail(PBE_ERR_INVALID, "rows * max_blocks_per_seq must be at most INT32_MAX");
  if (!tables_in || !lens_in || !parents || !tables_out || !lens_out || !counts || !workspace) return fail(PBE_ERR_INVALID, "null page mover operand");
  const uint64_t need = pbe_fork_pages_workspace_bytes(n_pages, rows_in, rows_out);
  if (workspace_bytes < need)
    return fail(PBE_ERR_INVALID, "workspace holds %llu of %llu bytes", (unsigned long long)workspace_bytes, (unsigned long long)need);
  pbe::PagePlanes laid{};
  rc = planes_of(planes, n_planes, n_pages, &laid);
  if (rc != PBE_OK) return rc;
  const uint64_t in = 4ull * (uint64_t)rows_in, out = 4ull * (uint64_t)rows_out, width = (uint64_t)max_blocks_per_seq;
  rc = check_memory(planes, n_planes,
                    {{tables_in, in * width, false}, {lens_in, in, false}, {parents, out, false}, {new_lens, new_lens ? out : 0, false},
                     {reserved, reserved ? 4ull * (uint64_t)n_pages : 0, false}, {tables_out, out * width, true}, {lens_out, out, true},
                     {counts, 8, true}, {workspace, need, true}},
                    device);
  if (rc != PBE_OK) return rc;
  pbe::ForkParams p{};
  p.tables_in = tables_in;
  p.lens_in = lens_in;
  p.parents = parents;
  p.new_lens = new_lens;
  p.reserved = reserved;
  p.tables_out = tables_out;
  p.lens_out = lens_out;
  p.counts = counts;
  p.header = static_cast<uint32_t*>(workspace);
  p.firsts = static_cast<int32_t*>(workspace) + pbe::kPageHeader;
  p.base = reinterpret_cast<uint32_t*>(p.firsts + rows_in);
  p.shared = p.firsts + rows_in + rows_out;
  p.wanted = p.shared + rows_out;
  p.copies = p.wanted + rows_out;
  p.fresh = p.copies + rows_out;
  p.n_pages = n_pages;
  p.stride = id_stride;
  p.rows_in = rows_in;
  p.rows_out = rows_out;
  p.max_blocks = max_blocks_per_seq;
  p.block_size = block_size;
  p.by_stride = pbe::make_fast_div((uint32_t)id_stride);
  p.by_block_size = pbe::make_fast_div((uint32_t)block_size);
  p.by_max_blocks = pbe::make_fast_div((uint32_t)max_blocks_per_seq);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_fork_pages(p, laid, compute_units(device), static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

uint64_t pbe_compact_pages_workspace_bytes(int32_t n_pages) {
  return n_pages <= 0 ? 0 : 4ull * (pbe::kPageHeader + 3ull * (uint64_t)n_pages);
}

int pbe_compact_pages(const pbe_page_plane* planes, int32_t n_planes, int32_t n_pages,
                      int32_t id_stride, const int32_t* tables_in, int32_t rows,
                      int32_t max_blocks_per_seq, const int32_t* reserved, int32_t* tables_out,
                      int32_t* moved_to, int32_t* counts, void* workspace,
                      uint64_t workspace_bytes, int device, void* stream) {
  if (rows <= 0 || max_blocks_per_seq <= 0 || device < 0) return fail(PBE_ERR_INVALID, "rows and max_blocks_per_seq > 0 and a device");
  int rc = check_pool(n_pages, id_stride);
  if (rc != PBE_OK) return rc;
  if ((int64_t)rows * max_blocks_per_seq > INT32_MAX) return fail(PBE_ERR_INVALID, "rows * max_blocks_per_seq must be at most INT32_MAX");
  if (!tables_in || !tables_out || !counts || !workspace) return fail(PBE_ERR_INVALID, "null page mover operand");
  const uint64_t need = pbe_compact_pages_workspace_bytes(n_pages);
  if (workspace_bytes < need)
    return fail(PBE_ERR_INVALID, "workspace holds %llu of %llu bytes", (unsigned long long)workspace_bytes, (unsigned long long)need);
  pbe::PagePlanes laid{};
  rc = planes_of(planes, n_planes, n_pages, &laid);
  if (rc != PBE_OK) return rc;
  const uint64_t entries = (uint64_t)rows * (uint64_t)max_blocks_per_seq, pages = 4ull * (uint64_t)n_pages;
  rc = check_memory(planes, n_planes,
                    {{tables_in, 4 * entries, false}, {reserved, reserved ? pages : 0, false}, {tables_out, 4 * entries, true},
                     {moved_to, moved_to ? pages : 0, true}, {counts, 8, true}, {workspace, need, true}},
                    device);
  if (rc != PBE_OK) return rc;
  pbe::CompactParams p{};
  p.tables_in = tables_in;
  p.reserved = reserved;
  p.tables_out = tables_out;
  p.counts = counts;
  p.header = static_cast<uint32_t*>(workspace);
  p.sources = static_cast<int32_t*>(workspace) + pbe::kPageHeader;
  p.places = p.sources + n_pages;
  p.moved_to = moved_to ? moved_to : p.places + n_pages;
  p.n_pages = n_pages;
  p.stride = id_stride;
  p.entries = (uint32_t)entries;
  p.by_stride = pbe::make_fast_div((uint32_t)id_stride);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_compact_pages(p, laid, compute_units(device), static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

}  // extern "C"
