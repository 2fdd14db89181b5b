// Internal interface of the decode reader of MXFP4 pages.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

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
  float* part_acc;            // [batch][q_heads][splits][dim], splits > 1
  float* part_ml;             // [batch][q_heads][splits][2]: maximum, sum
  uint32_t half;
  int32_t batch, q_heads, kv_heads, group, max_blocks;
  int32_t blocks;             // ids below it lie in all four pools
  int32_t splits, chunk;      // a sequence of n blocks takes ceil(n / chunk) <= splits pieces
  float scale;                // log2(e) / sqrt(dim): scores in base 2
};

// Pieces of a sequence that the longest of a batch is cut into.
int32_t mxfp4_decode_splits(int32_t batch, int32_t kv_heads, int32_t max_blocks, int64_t compute_units);
// Bytes of partial results; one split has none.
uint64_t mxfp4_decode_workspace_bytes(int32_t batch, int32_t q_heads, int32_t dim, int32_t splits);

// Parts the workspace into the partial results and sets p.chunk.
void plan_mxfp4_decode(Mxfp4DecodeParams* p, int dim, void* workspace);

hipError_t launch_paged_decode_mxfp4(const Mxfp4DecodeParams& p, int dim, hipStream_t stream);

}  // namespace pbe
