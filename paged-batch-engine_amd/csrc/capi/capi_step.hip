// C ABI: what a decode worker makes ready for a step (its tables).
#include <hip/hip_runtime.h>

#include <vector>

#include "capi_internal.h"
#include "../kernels/step_kernels.h"

using namespace pbe_capi;

extern "C" {

int pbe_build_step_tables(const int32_t* page_ids, int64_t n_page_ids, const int32_t* page_starts,
                          const int32_t* cached_lens, const int32_t* new_lens, int32_t batch,
                          int32_t block_size, int32_t* block_tables, int32_t max_blocks_per_seq,
                          int32_t* seq_lens, int32_t* token_starts, int32_t* slot_mapping,
                          int32_t* positions, int32_t max_tokens, int device, void* stream) {
  if (batch <= 0 || block_size <= 0 || max_blocks_per_seq <= 0 || max_tokens <= 0 || device < 0)
    return fail(PBE_ERR_INVALID, "batch, block_size, max_blocks_per_seq, max_tokens > 0 and a device");
  if (n_page_ids < 0 || n_page_ids > INT32_MAX) return fail(PBE_ERR_INVALID, "n_page_ids must be 0..INT32_MAX");
  if ((int64_t)batch * max_blocks_per_seq > INT32_MAX)
    return fail(PBE_ERR_INVALID, "batch * max_blocks_per_seq must be at most INT32_MAX");
  if ((n_page_ids && !page_ids) || !page_starts || !cached_lens || !block_tables || !seq_lens || !token_starts || !slot_mapping || !positions)
    return fail(PBE_ERR_INVALID, "null step table operand");
  const struct {
    const int32_t* at;
    uint64_t count;
    bool out;
  } arrays[] = {{page_ids, (uint64_t)n_page_ids, false},
                {page_starts, (uint64_t)batch + 1, false},
                {cached_lens, (uint64_t)batch, false},
                {new_lens, new_lens ? (uint64_t)batch : 0, false},
                {block_tables, (uint64_t)batch * (uint64_t)max_blocks_per_seq, true},
                {seq_lens, (uint64_t)batch, true},
                {token_starts, (uint64_t)batch + 1, true},
                {slot_mapping, (uint64_t)max_tokens, true},
                {positions, (uint64_t)max_tokens, true}};
  for (const auto& a : arrays) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(a.at);
    if (begin % 4) return fail(PBE_ERR_INVALID, "step table arrays must be 4-byte aligned");
    // Workgroups read lengths and lists while others write: an output in the
    // place of an input (seq_lens over cached_lens) would race with them.
    for (const auto& o : arrays) {
      const uintptr_t o_begin = reinterpret_cast<uintptr_t>(o.at);
      if (&a != &o && o.out && begin < o_begin + 4 * o.count && o_begin < begin + 4 * a.count)
        return fail(PBE_ERR_INVALID, "a step table output overlaps another array");
    }
  }
  {
    PBE_DEVICE_SCOPE(device);
    std::vector<Range> known;
    for (const auto& a : arrays)
      if (a.count && !accessible(a.at, 4 * a.count, device, &known))
        return fail(PBE_ERR_INVALID, "step table operands must be memory of device %d", device);
  }
  pbe::StepTablesParams p{};
  p.page_ids = page_ids;
  p.page_starts = page_starts;
  p.cached_lens = cached_lens;
  p.new_lens = new_lens;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.token_starts = token_starts;
  p.slots = slot_mapping;
  p.positions = positions;
  p.n_page_ids = (uint32_t)n_page_ids;
  p.batch = (uint32_t)batch;
  p.max_blocks = (uint32_t)max_blocks_per_seq;
  p.max_tokens = (uint32_t)max_tokens;
  p.block_size = (uint32_t)block_size;
  p.by_block_size = pbe::make_fast_div((uint32_t)block_size);
  p.by_max_blocks = pbe::make_fast_div((uint32_t)max_blocks_per_seq);
  PBE_DEVICE_SCOPE(device);
  PBE_HIP(pbe::launch_step_tables(p, static_cast<hipStream_t>(stream)));
  return PBE_OK;
}

}  // extern "C"
