// The shared-prefix pass of a decode step, launched by ps_paged_decode_shared
// (paged_decode.cu) and run by the tcgen05 prefill kernel (paged_prefill.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ps {

// Every row of group g (batch rows [group_starts[g], group_starts[g + 1])) attends
// over keys [0, shared_lens[first row]) of its first row's block table, in
// pieces of piece_keys keys (a multiple of 128). Each piece leaves one partial result per
// row (two when `paired`, for its even and odd key tiles): unnormalised output, running
// maximum (log2 units) and row sum. Batch row b, KV head h and head g of its group is
// row r = (h * num_seqs + b) * G + g of a partial; rows go in blocks of 32, a partial has
// N = ceil(num_seqs * num_q_heads / 32) of them:
//   part_o[partial][r / 32][column / 4][r % 32][column % 4]     part_ml[partial][r]
struct SharedPrefix {
  const char* fn;
  const void* query;
  int64_t query_seq_stride;
  const void* k_pool;
  const void* v_pool;
  int64_t num_blocks;
  const int32_t* block_tables;
  int64_t block_table_stride;
  const int32_t* group_starts;
  const int32_t* shared_lens;
  int num_groups;
  int max_group;
  int num_seqs;
  int num_q_heads;
  int num_kv_heads;
  int head_dim;
  int block_size;
  int max_blocks;
  int pieces;
  int piece_keys;
  bool paired;  // max_group rows fill one query tile at most
  float scale;
  float* part_o;
  float2* part_ml;
  int dtype;
  int32_t* device_error;
};

int launch_shared_prefix(const SharedPrefix& a, cudaStream_t s);

}  // namespace ps
