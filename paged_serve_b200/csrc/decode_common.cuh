// What the paged decode kernels share: launch parameters, the split-K unit list
// (plan kernel), the merge of a split sequence's partitions (combine kernel)
// and the host-side helpers around them. Included by one translation unit per
// cache format, so everything here has internal linkage.
#pragma once

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "capi_internal.h"
#include "common.cuh"

namespace ps {
namespace {

constexpr int kChunk = 16;  // keys per MMA step (one 16-row TMA tile per K and V half)

struct DecodeParams {
  void* out;
  const void* q;
  int64_t out_stride;
  int64_t q_stride;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* ctx_lens;
  float* ws_o;    // [B][max_splits][Hq][D]
  float* ws_lse;  // [B][max_splits][Hq]   (log2 domain)
  int64_t num_blocks;
  int num_seqs;
  int num_launch;  // launch positions: num_seqs, or the length of a listed subset
  int num_q_heads;
  int num_kv_heads;
  int group;  // Hq / Hkv
  int max_blocks;
  int block_size;
  int part_tokens;  // partition length (multiple of 16 and of the block size)
  int max_splits;
  int table_cap;  // ints of block table staged per CTA
  float scale_log2;
  int32_t* err;
  // Split-K only: the (sequence, partition) pairs that have keys, as
  // b * max_splits + split, and their number; written by decode_plan_kernel.
  int32_t* items;
  int32_t* item_count;
  int32_t* item_next;  // claim counter of the persistent CTAs (reset by the plan and the combine)
  bool planned;        // the unit list was written by ps_paged_decode_plan for this step
  // Optional permutation of [0, num_seqs) (longest first, from
  // ps_paged_decode_order): the order CTAs / planned units take sequences in.
  const int32_t* seq_order;
  // Optional fused append of the step's new token (ps_paged_decode_append):
  // new_k/new_v [num_seqs][Hkv][D] rows go to slot new_slots[b] of the pools
  // (raw pointers; -1 = no token) before the unit that reads that slot loads it.
  void* k_pool_w;
  void* v_pool_w;
  const void* new_k;
  const void* new_v;
  int64_t new_k_stride;
  int64_t new_v_stride;
  const int64_t* new_slots;
  int64_t num_slots;
  // Optional shared prefix (ps_paged_decode_shared): the first shared_lens[b] keys of
  // sequence b are attended by the prefix pass, which leaves pre_parts partials per piece
  // of pre_keys keys in pre_o and pre_ml (laid out as in shared_prefix.h). Partitions
  // cut the keys behind them.
  const int32_t* shared_lens;
  const float* pre_o;
  const float2* pre_ml;
  int pre_keys;
  int pre_parts;
  int pre_max;  // largest prefix the pieces hold
};

// Partials of a shared prefix: their number for a prefix of `pre` keys, and where a
// row's start (float4 columns for pre_o, 32 apart; rows for pre_ml).
struct SharedRows {
  int64_t row, blocks;
  __device__ __forceinline__ SharedRows(const DecodeParams& p, int b, int h, int g)
      : row((static_cast<int64_t>(h) * p.num_seqs + b) * p.group + g),
        blocks((static_cast<int64_t>(p.num_seqs) * p.num_q_heads + 31) / 32) {}
  __device__ __forceinline__ float2 ml(const DecodeParams& p, int part) const {
    return p.pre_ml[part * blocks * 32 + row];
  }
  template <int D>
  __device__ __forceinline__ float4 o(const DecodeParams& p, int part, int col4) const {
    return reinterpret_cast<const float4*>(
        p.pre_o)[((part * blocks + row / 32) * (D / 4) + col4) * 32 + row % 32];
  }
};

// Adds a prefix's partials to one column of four of a row: m, l, acc = running maximum,
// sum and unnormalised output. Eight partials' loads are in flight at a time, also where
// fewer are left: one after the other they were 9,300 of a CTA's 35,000 cycles at 256
// sequences over 4 partials (112 us a call against 117).
template <int D>
__device__ __forceinline__ void merge_shared(const DecodeParams& p, const SharedRows& rows,
                                             int parts, int col4, float& m, float& l,
                                             float (&acc)[4]) {
  constexpr int kBatch = 8;
  for (int s0 = 0; s0 < parts; s0 += kBatch) {
    float2 ml[kBatch];
    float4 o[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f);
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s0 + u < parts) {
        ml[u] = rows.ml(p, s0 + u);
        o[u] = rows.o<D>(p, s0 + u, col4);
      }
    }
    float m_new = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) m_new = fmaxf(m_new, ml[u].x);
    const float keep = m == -INFINITY ? 0.f : exp2f(m - m_new);
    l *= keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= keep;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float w = ml[u].x == -INFINITY ? 0.f : exp2f(ml[u].x - m_new);
      l += w * ml[u].y;
      acc[0] += w * o[u].x;
      acc[1] += w * o[u].y;
      acc[2] += w * o[u].z;
      acc[3] += w * o[u].w;
    }
    m = m_new;
  }
}

__device__ __forceinline__ int shared_parts(const DecodeParams& p, int pre) {
  return pre > 0 ? (pre + p.pre_keys - 1) / p.pre_keys * p.pre_parts : 0;
}

// Shared-prefix tokens of sequence b with ctx keys; 0 (and an error bit) when
// the prefix is not whole blocks of the sequence or longer than the pieces hold.
__device__ __forceinline__ int shared_prefix(const DecodeParams& p, int b, int ctx, bool report) {
  const int pre = p.shared_lens[b];
  if (pre < 0 || pre > ctx || pre > p.pre_max || pre % p.block_size != 0) {
    if (report) set_device_error(p.err, PS_DEVERR_LENGTH);
    return 0;
  }
  return pre;
}

// Sequence at position i of the launch order; -1 (and an error bit) for an
// entry that is not a sequence index.
__device__ __forceinline__ int ordered_seq(const DecodeParams& p, int i) {
  if (!p.seq_order) return i;
  const int b = p.seq_order[i];
  if (b < 0 || b >= p.num_seqs) {
    set_device_error(p.err, PS_DEVERR_LENGTH);
    return -1;
  }
  return b;
}

// Lists the (sequence, partition) units of a split-K launch in launch order
// (seq_order when given, else batch order):
// a sequence with ctx keys has ceil(ctx / part) partitions, and one unit even
// without keys (its output is written as zeros). One CTA of 1024 threads; a
// running block-wide prefix sum places each sequence's units.
template <bool kShared>
__global__ void __launch_bounds__(1024) decode_plan_kernel(const DecodeParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int wsum[32];
  __shared__ int carry;
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int base = 0; base < p.num_launch; base += 1024) {
    const int i = base + threadIdx.x;
    const int b = i < p.num_launch ? ordered_seq(p, i) : -1;
    int ns = 0;
    if (b >= 0) {
      int ctx = p.ctx_lens[b];
      if (ctx > p.max_blocks * p.block_size) ctx = 0;  // the decode kernel reports it
      if constexpr (kShared) ctx -= shared_prefix(p, b, ctx, false);
      ns = ctx <= 0 ? 1 : (ctx + p.part_tokens - 1) / p.part_tokens;
    }
    int x = ns;  // inclusive scan within the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    if (warp == 0) {
      const int w = wsum[lane];
      int y = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
      }
      wsum[lane] = y - w;  // exclusive, per warp
    }
    __syncthreads();
    const int off = carry + wsum[warp] + x - ns;
    for (int k = 0; k < ns; ++k) p.items[off + k] = b * p.max_splits + k;
    __syncthreads();  // every thread has read carry
    if (threadIdx.x == blockDim.x - 1) carry = off + ns;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *p.item_count = carry;
    *p.item_next = 0;
  }
}

// Merge the partitions of each split sequence: out = sum_s w_s O_s, with
// w_s = 2^(lse_s - max lse) / sum. One warp per (sequence, query head).
// kShared: the pieces of the sequence's shared prefix are merged too.
template <typename T, int D, bool kShared = false>
__global__ void __launch_bounds__(128) decode_combine_kernel(const DecodeParams p) {
  pdl_trigger();
  pdl_wait();
  // The decode launch has finished claiming units: rearm the claim counter, so
  // the next layer of a planned step can reuse the unit list without a plan.
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.item_next = 0;
  const int warp_global = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (warp_global >= p.num_launch * p.num_q_heads) return;
  const int b = ordered_seq(p, warp_global / p.num_q_heads);  // only launched sequences
  if (b < 0) return;
  const int qh = warp_global % p.num_q_heads;
  int ctx = p.ctx_lens[b];
  if (ctx > p.max_blocks * p.block_size) ctx = 0;
  int pre = 0;
  if constexpr (kShared) pre = shared_prefix(p, b, ctx, false);
  ctx -= pre;
  const int nsplit = (ctx + p.part_tokens - 1) / p.part_tokens;
  if (nsplit <= 1) return;
  const int64_t base = static_cast<int64_t>(b) * p.max_splits * p.num_q_heads + qh;
  float mmax = -INFINITY;
  for (int s = lane; s < nsplit; s += 32)
    mmax = fmaxf(mmax, p.ws_lse[base + static_cast<int64_t>(s) * p.num_q_heads]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mmax = fmaxf(mmax, __shfl_xor_sync(0xffffffffu, mmax, o));
  constexpr int kPer = D / 32;  // dims per lane
  using Vec = typename std::conditional<kPer == 4, float4, float2>::type;
  float acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  float wsum = 0.f;
  auto add = [&](float w, const Vec& v) {
    wsum += w;
    acc[0] += w * v.x;
    acc[1] += w * v.y;
    if constexpr (kPer == 4) {
      acc[2] += w * reinterpret_cast<const float4&>(v).z;
      acc[3] += w * reinterpret_cast<const float4&>(v).w;
    }
  };
  auto load = [&](int s) {
    return *reinterpret_cast<const Vec*>(p.ws_o + (base + static_cast<int64_t>(s) * p.num_q_heads) * D +
                                         lane * kPer);
  };
  // Partitions in order (the sum order is fixed); lane l computes the weight of
  // partition s0 + l. Eight partitions' loads are in flight at a time: when few
  // sequences are split, the longest one's chain of loads (64 partitions for
  // 32k tokens) sets the length of the launch (four in flight: 156.6 against
  // 153.3 us per 64-sequence 70B layer); sixteen gain a little more there but
  // cost occupancy when many sequences are split.
  for (int s0 = 0; s0 < nsplit; s0 += 32) {
    const int n = min(32, nsplit - s0);
    const float lse = lane < n ? p.ws_lse[base + static_cast<int64_t>(s0 + lane) * p.num_q_heads]
                               : -INFINITY;
    const float wl = (lse == -INFINITY) ? 0.f : exp2f(lse - mmax);
    int k = 0;
    for (; k + 8 <= n; k += 8) {
      Vec v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = load(s0 + k + u);
#pragma unroll
      for (int u = 0; u < 8; ++u) add(__shfl_sync(0xffffffffu, wl, k + u), v[u]);
    }
    for (; k + 4 <= n; k += 4) {
      Vec v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = load(s0 + k + u);
#pragma unroll
      for (int u = 0; u < 4; ++u) add(__shfl_sync(0xffffffffu, wl, k + u), v[u]);
    }
    for (; k < n; ++k) add(__shfl_sync(0xffffffffu, wl, k), load(s0 + k));
  }
  if constexpr (kShared) {
    // A lane's kPer columns are all or half of a column of four.
    const int at = lane * kPer % 4;
    float four[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) four[at == 0 ? i : (2 + i) & 3] = acc[i];
    merge_shared<D>(p, SharedRows(p, b, qh / p.group, qh % p.group), shared_parts(p, pre),
                    lane * kPer / 4, mmax, wsum, four);
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = at == 0 ? four[i] : four[(2 + i) & 3];
  }
  const float inv = (wsum > 0.f) ? 1.f / wsum : 0.f;
  T* orow = static_cast<T*>(p.out) + b * p.out_stride + static_cast<int64_t>(qh) * D + lane * kPer;
#pragma unroll
  for (int i = 0; i < kPer; i += 2)
    *reinterpret_cast<uint32_t*>(orow + i) = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
}

// ------------------------------------------------------------ host side
int effective_part_tokens(int split_tokens, int max_blocks, int block_size) {
  return split_tokens > 0 ? split_tokens : max_blocks * block_size;
}

// Guards the per-device launch caches below against concurrent host threads.
std::mutex g_launch_mu;

// The dynamic shared-memory attribute is per function and per device; raise it
// only when a larger block table than any seen so far needs more.
template <typename K>
int reserve_smem(K kern, size_t smem, size_t (&configured)[64]) {
  std::lock_guard<std::mutex> lock(g_launch_mu);
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || configured[dev] < smem) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess)
      return fail(PS_ERR_CUDA, "ps_paged_decode: cannot reserve %zu B shared memory: %s", smem,
                  cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev] = smem;
  }
  return PS_OK;
}

// CTAs of a persistent launch: what one SM holds of `kern` with this many threads
// and this much dynamic shared memory, and the SMs. `cache` (64 devices) belongs
// to the kernel: kernels of one signature are one type here.
struct Resident {
  size_t smem = 0;
  int per_sm = 0;
  int sms = 0;
};

template <typename K>
int resident_ctas(K kern, const char* fn, int threads, size_t smem, Resident (&cache)[64],
                  Resident* out) {
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(g_launch_mu);
  Resident fresh;
  Resident& r = dev >= 0 && dev < 64 ? cache[dev] : fresh;
  if (r.per_sm == 0 || r.smem != smem) {
    int n = 0, count = 0;
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess || n <= 0)
      return fail(PS_ERR_CUDA, "%s: occupancy query failed: %s", fn, cudaGetErrorString(e));
    r.smem = smem;
    r.per_sm = n;
    r.sms = count;
  }
  *out = r;
  return PS_OK;
}

// Argument checks shared by every decode entry point; on success fills the
// partition length (tokens), the partitions per sequence and the block-table
// window a partition spans. Returns PS_OK, or the status of the first failure
// with its message naming `fn`.
int validate_decode(const char* fn, const void* out, int64_t out_seq_stride, const void* query,
                    int64_t query_seq_stride, const void* k_pool, const void* v_pool,
                    int64_t num_blocks, const int32_t* block_tables, int64_t block_table_stride,
                    const int32_t* ctx_lens, int num_seqs, int num_q_heads, int num_kv_heads,
                    int head_dim, int block_size, int max_blocks_per_seq, int split_tokens,
                    int dtype, int* part_out, int* max_splits_out, int* table_cap_out) {
  if (dtype != PS_DTYPE_BF16 && dtype != PS_DTYPE_F16)
    return fail(PS_ERR_UNSUPPORTED, "%s: dtype %d unsupported (bf16/f16 only)", fn, dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(PS_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", fn, head_dim);
  if (block_size != 8 && block_size != 16 && block_size != 32)
    return fail(PS_ERR_UNSUPPORTED, "%s: block_size %d unsupported (8, 16 or 32)", fn,
                block_size);
  if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0)
    return fail(PS_ERR_INVALID, "%s: bad sizes", fn);
  if (num_q_heads % num_kv_heads != 0)
    return fail(PS_ERR_INVALID, "%s: num_q_heads %d not divisible by num_kv_heads %d", fn,
                num_q_heads, num_kv_heads);
  const int group = num_q_heads / num_kv_heads;
  if (group > 16)
    return fail(PS_ERR_UNSUPPORTED, "%s: %d query heads per kv head unsupported (max 16)", fn, group);
  if (num_seqs == 0) return PS_OK;  // nothing to launch; the caller checks num_seqs too
  if (num_seqs > 65535 || num_kv_heads > 65535)
    return fail(PS_ERR_INVALID, "%s: too many sequences/heads for one launch", fn);
  if (!out || !query || !k_pool || !v_pool || !block_tables || !ctx_lens)
    return fail(PS_ERR_INVALID, "%s: null pointer argument", fn);
  if (block_table_stride < max_blocks_per_seq)
    return fail(PS_ERR_INVALID, "%s: block_table_stride < max_blocks_per_seq", fn);
  if (query_seq_stride < static_cast<int64_t>(num_q_heads) * head_dim ||
      out_seq_stride < static_cast<int64_t>(num_q_heads) * head_dim || (query_seq_stride % 8) ||
      (out_seq_stride % 8) || !aligned(query, 16) || !aligned(out, 16))
    return fail(PS_ERR_INVALID, "%s: query/out must be 16-byte aligned, strides >= Hq*D and %% 8", fn);
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16))
    return fail(PS_ERR_INVALID, "%s: pools must be 16-byte aligned", fn);
  const int64_t rows = num_blocks * num_kv_heads * block_size;
  if (rows >= (int64_t(1) << 31))
    return fail(PS_ERR_INVALID, "%s: pool too large for 32-bit TMA row coordinates", fn);
  const int unit = block_size > kChunk ? block_size : kChunk;
  if (split_tokens < 0 || (split_tokens % unit))
    return fail(PS_ERR_INVALID, "%s: split_tokens must be >= 0 and a multiple of %d", fn, unit);
  const int part = effective_part_tokens(split_tokens, max_blocks_per_seq, block_size);
  const int max_splits = (max_blocks_per_seq * block_size + part - 1) / part;
  const int table_cap = (part + block_size - 1) / block_size;
  if (table_cap > 8192)
    return fail(PS_ERR_UNSUPPORTED, "%s: partition of %d blocks too long; set split_tokens", fn,
                table_cap);
  if (max_splits > 65535) return fail(PS_ERR_INVALID, "%s: too many partitions", fn);
  *part_out = part;
  *max_splits_out = max_splits;
  *table_cap_out = table_cap;
  return PS_OK;
}

// Checks the split-K workspace and lays the partials, their LSEs, the unit list
// and its counters out in it.
int set_split_workspace(const char* fn, DecodeParams* p, int num_seqs, int num_q_heads,
                        int head_dim, int block_size, int max_blocks_per_seq, int split_tokens,
                        int max_splits, void* workspace, int64_t workspace_bytes) {
  const int64_t need = ps_paged_decode_workspace_bytes(num_seqs, num_q_heads, head_dim, block_size,
                                                       max_blocks_per_seq, split_tokens);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
    return fail(PS_ERR_INVALID, "%s: split-K needs a 256-byte aligned workspace of %lld bytes", fn,
                (long long)need);
  if (static_cast<int64_t>(num_seqs) * max_splits >= (int64_t(1) << 31))
    return fail(PS_ERR_INVALID, "%s: too many (sequence, partition) units", fn);
  const int64_t rows_ws = static_cast<int64_t>(num_seqs) * max_splits * num_q_heads;
  const int64_t o_bytes = ((rows_ws * head_dim * 4) + 255) / 256 * 256;
  const int64_t lse_bytes = ((rows_ws * 4) + 255) / 256 * 256;
  const int64_t item_bytes = ((static_cast<int64_t>(num_seqs) * max_splits * 4) + 255) / 256 * 256;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p->ws_o = reinterpret_cast<float*>(ws);
  p->ws_lse = reinterpret_cast<float*>(ws + o_bytes);
  p->items = reinterpret_cast<int32_t*>(ws + o_bytes + lse_bytes);
  p->item_count = reinterpret_cast<int32_t*>(ws + o_bytes + lse_bytes + item_bytes);
  p->item_next = p->item_count + 1;
  return PS_OK;
}

}  // namespace
}  // namespace ps
