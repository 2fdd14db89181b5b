// Internal interface of the prompt reader: causal attention of many queries a
// sequence over rows or pages of keys and values.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernels.h"  // FastDiv

namespace pbe {

enum class KeyKind : int32_t { kRows, kBf16, kFp8, kMxfp4 };

struct PromptParams {
  const uint8_t* q;         // bf16 rows [n_q] of q_heads heads, q_stride bytes apart
  const uint8_t* k;         // rows, or the layer's K pool
  const uint8_t* v;
  const uint8_t* k_scales;  // FP8: fp32 [block][token][head]; MXFP4: bytes
  const uint8_t* v_scales;
  uint8_t* out;             // bf16 [n_q][q_heads][head_dim]
  const int32_t* q_starts;  // [batch + 1]
  const int32_t* lens;      // pages: [batch] lengths; rows: [batch + 1] first rows
  const int32_t* tables;    // pages: [batch][max_blocks]
  float* part_acc;          // [part][2][kv_heads][rows of a tile][head_dim]
  float* part_ml;           // [part][2][kv_heads][rows of a tile][2]: maximum, sum
  uint64_t q_stride, k_stride, v_stride;  // bytes between rows (k, v: of rows, or of a page's tokens)
  uint64_t half;            // pages: bytes of one block of one pool
  int32_t n_q, n_k;         // rows there are (n_k: of rows)
  int32_t batch, kv_heads, group;
  int32_t max_blocks, blocks;  // pages: of a table, of the pools
  int32_t parts;            // per KV head that the work is cut into; 0: a workgroup a tile
  int32_t step;             // what a tile costs more than the one before (sixteenths of a key)
  float scale;              // log2(e) / sqrt(head_dim): scores in base 2
  FastDiv by_group;
};

// How a call is cut up: tiles of `rows` rows (tokens times query heads of a KV
// head), at most `tiles` of them; `parts` equal parts of all their work per KV head,
// with `each` bytes of partial results, or 0.
struct PromptPlan {
  int rows = 0;
  int64_t tiles = 0;
  int32_t parts = 0;
  uint64_t each = 0;
};
// most_keys: that a sequence may have (rows: that there are); units: compute units.
PromptPlan plan_prompt(int64_t n_q, int64_t batch, int32_t group, int32_t kv_heads, KeyKind kind, int64_t most_keys, int64_t units, uint64_t workspace,
                       int32_t head_dim);

hipError_t launch_prompt_attention(PromptParams p, const PromptPlan& plan, int dim, KeyKind kind, hipStream_t stream);

}  // namespace pbe
