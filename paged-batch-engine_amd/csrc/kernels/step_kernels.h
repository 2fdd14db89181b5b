// Internal interface of the step tables: a decode worker's block tables,
// lengths, slots and positions from its requests' page lists.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernels.h"  // FastDiv

namespace pbe {

struct StepTablesParams {
  const int32_t* page_ids;     // [n_page_ids], request after request
  const int32_t* page_starts;  // [batch + 1]
  const int32_t* cached_lens;  // [batch]
  const int32_t* new_lens;     // [batch], or null: one each
  int32_t* block_tables;       // [batch][max_blocks]
  int32_t* seq_lens;           // [batch]
  int32_t* token_starts;       // [batch + 1]
  int32_t* slots;              // [max_tokens]
  int32_t* positions;          // [max_tokens]
  uint32_t n_page_ids;         // <= INT32_MAX, as the others and batch * max_blocks
  uint32_t batch, max_blocks, max_tokens, block_size;
  uint32_t token_groups;       // workgroups that write tokens; the rest write tables
  FastDiv by_block_size, by_max_blocks;
};

// Tokens and table entries that one workgroup writes.
constexpr uint32_t kStepTokens = 256, kStepEntries = 1024;

hipError_t launch_step_tables(StepTablesParams p, hipStream_t stream);

}  // namespace pbe
