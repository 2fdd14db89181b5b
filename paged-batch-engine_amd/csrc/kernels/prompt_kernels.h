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
  float* part_acc;          // [unit][kv_heads][rows of a tile][head_dim]
  float* part_ml;           // [unit][kv_heads][rows of a tile][2]: maximum, sum
  uint64_t q_stride, k_stride, v_stride;  // bytes between rows (k, v: of rows, or of a page's tokens)
  uint64_t half;            // pages: bytes of one block of one pool
  int32_t n_q, n_k;         // rows there are (n_k: of rows)
  int32_t batch, kv_heads, group;
  int32_t max_blocks, blocks;  // pages: of a table, of the pools
  int32_t units;            // pieces of tiles that the launch has workgroups for, per KV head
  int32_t wanted;           // pieces that fill the GPU, per KV head; 0: no tile is cut
  float scale;              // log2(e) / sqrt(head_dim): scores in base 2
  FastDiv by_group;
};

// Rows (tokens times query heads of a KV head) of a workgroup's tile.
int prompt_tile_rows(int64_t n_q, int64_t batch, int32_t group);
// Most pieces per KV head of tiles of `rows`: as many as are wanted and one a tile.
int64_t prompt_units(int64_t n_q, int64_t batch, int32_t group, int rows, int64_t wanted);
// Bytes of partial results of `units` pieces, 16-byte multiples.
uint64_t prompt_workspace_bytes(int64_t units, int32_t kv_heads, int32_t head_dim, int rows);

hipError_t launch_prompt_attention(const PromptParams& p, int dim, KeyKind kind, int rows, hipStream_t stream);

}  // namespace pbe
