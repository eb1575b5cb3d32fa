// The shared-prefix pass of a decode step, launched by ps_paged_decode_shared
// (paged_decode.cu) and run by the tcgen05 prefill kernel (paged_prefill.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ps {

// Every row of group g (batch rows [group_starts[g], group_starts[g + 1])) attends
// over keys [0, shared_lens[first row]) of its first row's block table, in
// pieces of piece_keys keys (a multiple of 128). Piece x of batch row b and query
// head h leaves its unnormalised output, running maximum (log2 units) and row sum
// at row (x * num_seqs + b) * num_q_heads + h of part_o / part_ml.
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
  float scale;
  float* part_o;
  float2* part_ml;
  int dtype;
  int32_t* device_error;
};

int launch_shared_prefix(const SharedPrefix& a, cudaStream_t s);

}  // namespace ps
