// Internal interface of the decode reader of MXFP4 pages.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernels.h"  // FastDiv

namespace pbe {

constexpr int kMxDecodeMaxGroup = 16;     // query heads per KV head
constexpr int kMxDecodeMaxSplits = 1024;  // pieces of one sequence

struct Mxfp4DecodeParams {
  const uint8_t* key_pool;    // block b at b * half
  const uint8_t* value_pool;
  const uint8_t* key_scales;  // block b at b * half / 16
  const uint8_t* value_scales;
  const uint16_t* q;          // bf16 [batch][q_heads][dim]
  uint16_t* out;
  const int32_t* tables;      // [batch][max_blocks]
  const int32_t* seq_lens;    // [batch]
  uint32_t half;
  int32_t batch, q_heads, kv_heads, group, max_blocks;
  int32_t blocks;             // ids below it lie in all four pools
  float scale;                // log2(e) / sqrt(dim): scores in base 2
  // Set by launch_paged_decode_mxfp4.
  int32_t most;               // pieces there is room for; batch: every sequence whole
  uint32_t wanted;            // pieces that fill the chip
  int32_t min_chunk;          // blocks of a piece, at least, before a sequence's are made even
  FastDiv by_eight;           // workgroups of eight pieces
  float* part_acc;            // [most][q_heads][dim]: results of pieces
  float* part_ml;             // [most][q_heads][2]: maximum, sum
  uint64_t* tickets;          // [most][kv_heads]: arrivals (arrival.h)
  uint64_t tag;               // of this launch
};

// Pieces a sequence to make room for, and the bytes they take (one: none).
int32_t mxfp4_decode_splits(int32_t batch, int32_t kv_heads, int32_t max_blocks, int64_t compute_units);
uint64_t mxfp4_decode_workspace_bytes(int32_t batch, int32_t q_heads, int32_t dim, int32_t splits);

hipError_t launch_paged_decode_mxfp4(Mxfp4DecodeParams p, int dim, int32_t splits, void* workspace, int64_t compute_units, hipStream_t stream);

}  // namespace pbe
