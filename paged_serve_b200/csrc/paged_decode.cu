// Paged decode attention (one query token per sequence, GQA) for sm_100a.
//
// Work decomposition: one CTA per (kv-head, partition, sequence). A partition
// is `split_tokens` keys of one sequence (the whole context when not split).
// The CTA's warps take the partition's KV blocks round-robin; each warp owns a
// private ring of NS shared-memory stages fed by TMA (two 64-column boxes per
// K or V tile, 128-byte swizzle) and runs its own fp32 online softmax, so the
// steady state needs no CTA-wide barrier. The group of G = Hq/Hkv query heads
// that share the KV head forms the 16-row A operand of a bf16/f16 warp MMA
// (rows >= G are zero; for G <= 8 rows 8-15 are not even carried through the
// softmax), so every K/V byte is read from HBM exactly once per step and
// consumed by all G heads:
//   S[16 x 16 keys]  = Q[16 x D] . K_blk^T      (D/16 MMAs per n-tile, 2 n-tiles)
//   O[16 x D]       += P[16 x 16 keys] . V_blk  (D/8 MMAs)
// The S accumulator fragment is re-used directly as the A fragment of P.V.
// At the end the warps merge (m, l, O) through shared memory; partitions of a
// split sequence are merged by ps_decode_combine_kernel with a log-sum-exp.
//
// Arithmetic intensity is ~4 flop per KV byte, so the tensor pipe is nearly
// idle and the kernel is bound by HBM bandwidth; what matters is keeping
// enough TMA bytes in flight per SM (NW * NS * 2 tiles per CTA).
#include <cudaTypedefs.h>

#include "decode_common.cuh"
#include "shared_prefix.h"

namespace ps {
namespace {

template <int D>
struct TileGeom {
  static constexpr int kHalves = D / 64;              // 64-column TMA boxes per tile
  static constexpr int kHalfBytes = kChunk * 128;     // one chunk half: 16 rows x 128 B
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  // Byte offset of 16-byte chunk c (0..D/8) of token row t inside a swizzled tile.
  __device__ __forceinline__ static uint32_t off(int t, int c) {
    return (c >> 3) * kHalfBytes + t * 128 + ((((c & 7) ^ (t & 7))) << 4);
  }
};

template <int D, int NW, int NS>
struct DecodeSmem {
  static constexpr int kStageBytes = 2 * TileGeom<D>::kTileBytes;  // K + V
  static constexpr int kRingBytes = NW * NS * kStageBytes;
  static constexpr int kMergeBytes = NW * 16 * (D + 2) * 4;  // m, l, O of up to 16 rows per warp
  static_assert(kMergeBytes <= kRingBytes, "merge area must fit in the ring");
  static constexpr int kBarOffset = kRingBytes;
  static constexpr int kTableOffset = kBarOffset + NW * NS * 8;
  static size_t bytes(int table_cap) {
    return 1024 /*alignment slack*/ + kTableOffset + static_cast<size_t>(table_cap) * 4;
  }
};

// BS = tokens per KV block (8, 16 or 32). A 16-key chunk is one 16-row box of
// its block (BS 16), the first or second half of a block (BS 32), or two 8-row
// boxes of consecutive blocks (BS 8); an 8-row box is one 1024-byte swizzle
// atom, so every case lands in the same shared-memory tile layout.
// R = MMA rows carried (8 when G <= 8, else 16).
// kList: persistent CTAs (one per resident slot) claim (kv head, unit) pairs of
// the split-K work list from an atomic counter, one ahead; otherwise one CTA
// per (kv head, 1, sequence).
// kShared: a sequence's first shared_lens[b] keys belong to the prefix pass (the
// kernel launched just before this one); this kernel walks the keys behind them
// without waiting for that pass, and merges its pieces at the end.
template <typename T, int D, int NW, int NS, int BS, int R, bool kList, bool kShared = false>
__global__ void __launch_bounds__(NW * 32)
    paged_decode_kernel(const DecodeParams p, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap) {
  static_assert(R == 8 || R == 16, "8 or 16 rows");
  using G = TileGeom<D>;
  using SM = DecodeSmem<D, NW, NS>;
  constexpr bool kWide = R == 16;
  constexpr int kKSteps = D / 16;
  constexpr int kNTiles = D / 8;

  int h = blockIdx.x;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int group = p.group;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::kBarOffset);
  int32_t* table = reinterpret_cast<int32_t*>(smem + SM::kTableOffset);
  // Launched with programmatic stream serialization: the set-up above touches
  // only shared memory and kernel parameters; global memory waits for the
  // previous kernel.
  pdl_trigger();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
    for (int i = 0; i < NW * NS; ++i) mbar_init(&bars[i], 1);
    fence_barrier_init();
  }
  if constexpr (!kShared) pdl_wait();

  // Work units: one (sequence, partition) per CTA, or, for split-K, (kv head,
  // planned unit) pairs claimed one at a time (thread 0 claims the next while
  // the current one runs; the claimed index goes through a double-buffered
  // shared slot, so a barrier per unit suffices). Ring stages and barrier
  // phases carry over from one unit to the next (gbase = this warp's ring
  // iterations so far).
  __shared__ int claimed[2];
  int total = 0, next = 0;
  if constexpr (kList) {
    // A unit list planned for another step (a caller error) can hold more
    // entries than this launch's workspace holds, or sequences it does not
    // have: the count is clamped to the capacity and every entry is checked.
    const int cap = p.num_seqs * p.max_splits;
    total = min(max(*p.item_count, 0), cap) * p.num_kv_heads;
    if (threadIdx.x == 0) next = atomicAdd(p.item_next, 1);
  }
  uint32_t gbase = 0;
  for (int k = 0;; ++k) {
  int split, b;
  if constexpr (kList) {
    if (threadIdx.x == 0) {
      claimed[k & 1] = next;
      next = atomicAdd(p.item_next, 1);
    }
    __syncthreads();
    const int u = claimed[k & 1];
    if (u >= total) break;
    h = u % p.num_kv_heads;
    const int item = p.items[u / p.num_kv_heads];
    if (item < 0 || item >= p.num_seqs * p.max_splits) {
      if (threadIdx.x == 0) set_device_error(p.err, PS_DEVERR_LENGTH);
      continue;
    }
    split = item % p.max_splits;
    b = item / p.max_splits;
  } else {
    if (k > 0) break;
    split = blockIdx.y;
    b = ordered_seq(p, blockIdx.z);
    if (b < 0) break;
  }

  int ctx = p.ctx_lens[b];
  if (ctx > p.max_blocks * BS) {
    if (threadIdx.x == 0 && split == 0) set_device_error(p.err, PS_DEVERR_LENGTH);
    ctx = 0;
  }
  const bool any_keys = ctx > 0;
  int pre = 0;
  if constexpr (kShared) {
    // Also without keys: a prefix is longer than such a sequence.
    pre = shared_prefix(p, b, max(ctx, 0), threadIdx.x == 0);
    ctx -= pre;  // from here on: the sequence's own keys, behind the prefix
  }
  const int nsplit = (ctx + p.part_tokens - 1) / p.part_tokens;
  // Fused append: this (sequence, kv head)'s new K/V row goes to its slot, in
  // the last partition, which only this unit reads. Thread t < 2*D/8 moves 16 B.
  const bool writer = p.new_k != nullptr && split == (nsplit > 0 ? nsplit - 1 : 0);
  auto write_row = [&](int t) {
    constexpr int kPieces = D / 8;
    const int64_t slot = p.new_slots[b];
    if (slot >= p.num_slots) {
      if (t == 0) set_device_error(p.err, PS_DEVERR_SLOT);
      return false;
    }
    if (slot < 0 || t >= 2 * kPieces) return false;
    const bool is_v = t >= kPieces;
    const int piece = is_v ? t - kPieces : t;
    const int64_t blk = slot / BS;
    const int64_t row = ((blk * p.num_kv_heads + h) * BS + (slot - blk * BS)) * D + piece * 8;
    const T* src = static_cast<const T*>(is_v ? p.new_v : p.new_k) +
                   b * (is_v ? p.new_v_stride : p.new_k_stride) + static_cast<int64_t>(h) * D +
                   piece * 8;
    T* dst = static_cast<T*>(is_v ? p.v_pool_w : p.k_pool_w) + row;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
    return true;
  };
  if (!any_keys) {
    if constexpr (kShared) pdl_wait();
    if (writer) write_row(threadIdx.x);  // nothing of this launch reads it
    // No keys: the output is defined as zeros (nothing to attend to).
    if (split == 0) {
      T* o = static_cast<T*>(p.out) + b * p.out_stride + static_cast<int64_t>(h) * group * D;
      for (int i = threadIdx.x; i < group * D; i += blockDim.x) o[i] = from_f32<T>(0.f);
    }
    continue;
  }
  if (split >= max(nsplit, kShared ? 1 : 0)) continue;

  const int t_begin = split * p.part_tokens;
  const int t_end = min(ctx, t_begin + p.part_tokens);
  const int chunk_begin = t_begin / kChunk;
  const int nchunk = (t_end - t_begin + kChunk - 1) / kChunk;
  const int blk_begin = t_begin / BS;  // partitions start on block and chunk boundaries
  const int nblk = (t_end - t_begin + BS - 1) / BS;

  // Stage this partition's block ids, validated, in shared memory.
  const int32_t* bt = p.block_tables + static_cast<int64_t>(b) * p.bt_stride + blk_begin + pre / BS;
  for (int i = threadIdx.x; i < nblk; i += blockDim.x) {
    int32_t id = bt[i];
    if (id < 0 || id >= p.num_blocks) {
      set_device_error(p.err, PS_DEVERR_BLOCK_ID);
      id = 0;  // read a valid block instead of faulting; the error bit reports it
    }
    table[i] = id;
  }
  __syncthreads();
  if (writer && warp == (nchunk - 1) % NW) {
    // The warp that loads the last chunk writes the row, then hands it to its
    // own TMA issue (lane 0) through the proxy fence and a warp barrier.
    if (write_row(lane)) fence_proxy_async_global();
    __syncwarp();
  }

  uint8_t* ring = smem + warp * NS * SM::kStageBytes;
  uint64_t* wbar = bars + warp * NS;
  constexpr int kBox = BS < kChunk ? BS : kChunk;  // rows per TMA box
  constexpr int kBoxes = kChunk / kBox;            // boxes per 16-key chunk

  // Issue the TMA loads of warp-local iteration `it` (chunk warp + it*NW).
  auto issue = [&](int it) {
    const int j = warp + it * NW;
    const int st = (gbase + it) % NS;
    uint8_t* kdst = ring + st * SM::kStageBytes;
    uint8_t* vdst = kdst + G::kTileBytes;
    mbar_arrive_expect_tx(&wbar[st], SM::kStageBytes);
#pragma unroll
    for (int x = 0; x < kBoxes; ++x) {
      const int tok = j * kChunk + x * kBox;  // first key of the box, from t_begin
      // A box past the partition's last block re-reads that block (its keys are masked).
      const int bi = min(tok / BS, nblk - 1);
      const int32_t row = (table[bi] * p.num_kv_heads + h) * BS + tok % BS;
#pragma unroll
      for (int half = 0; half < G::kHalves; ++half) {
        tma_load_2d(kdst + half * G::kHalfBytes + x * kBox * 128, &kmap, &wbar[st], half * 64, row);
        tma_load_2d(vdst + half * G::kHalfBytes + x * kBox * 128, &vmap, &wbar[st], half * 64, row);
      }
    }
  };

  if (lane == 0) {
#pragma unroll
    for (int it = 0; it < NS; ++it)
      if (warp + it * NW < nchunk) issue(it);
  }

  // Q fragments: lane (r = lane/4, q4 = lane%4) holds rows r and r + 8 of the
  // head group (A registers a0/a2 and a1/a3 of the m16n8k16 layout).
  const int r = lane >> 2;
  const int q4 = lane & 3;
  uint32_t qa0[kKSteps], qa1[kKSteps], qa2[kKSteps], qa3[kKSteps];
  {
    const bool real = r < group;
    const T* qrow = static_cast<const T*>(p.q) + b * p.q_stride +
                    static_cast<int64_t>(h * group + (real ? r : 0)) * D;
    const bool real_hi = kWide && r + 8 < group;
    const T* qrow_hi = static_cast<const T*>(p.q) + b * p.q_stride +
                       static_cast<int64_t>(h * group + (real_hi ? r + 8 : 0)) * D;
#pragma unroll
    for (int kk = 0; kk < kKSteps; ++kk) {
      qa0[kk] = real ? *reinterpret_cast<const uint32_t*>(qrow + kk * 16 + 2 * q4) : 0u;
      qa2[kk] = real ? *reinterpret_cast<const uint32_t*>(qrow + kk * 16 + 8 + 2 * q4) : 0u;
      qa1[kk] = real_hi ? *reinterpret_cast<const uint32_t*>(qrow_hi + kk * 16 + 2 * q4) : 0u;
      qa3[kk] = real_hi ? *reinterpret_cast<const uint32_t*>(qrow_hi + kk * 16 + 8 + 2 * q4) : 0u;
    }
  }

  float o[kNTiles][4];
#pragma unroll
  for (int n = 0; n < kNTiles; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m_run = -INFINITY, m_hi = -INFINITY;  // rows r and r + 8
  float l_run = 0.f, l_hi = 0.f;
  int stuck_at = -1;  // warp-local iteration whose wait gave up

  // ldmatrix row/chunk selectors (see the fragment layouts above).
  const int qk_t = (lane & 7) + ((lane >> 4) << 3);
  const int qk_c = (lane >> 3) & 1;
  const int pv_t = (lane & 7) + (((lane >> 3) & 1) << 3);
  const int pv_c = lane >> 4;

  for (int it = 0; warp + it * NW < nchunk; ++it) {
    const int j = warp + it * NW;
    const int st = (gbase + it) % NS;
    if (!mbar_wait_bounded(&wbar[st], ((gbase + it) / NS) & 1)) {
      stuck_at = it;
      break;
    }
    const uint32_t kbase = smem_u32(ring + st * SM::kStageBytes);
    const uint32_t vbase = kbase + G::kTileBytes;

    // ---- S = Q K^T for the 16 keys of this block
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < kKSteps; ++kk) {
      uint32_t b00, b01, b10, b11;
      ldsm_x4(kbase + G::off(qk_t, 2 * kk + qk_c), b00, b01, b10, b11);
      Mma<T>::run(s0, qa0[kk], qa1[kk], qa2[kk], qa3[kk], b00, b01);
      Mma<T>::run(s1, qa0[kk], qa1[kk], qa2[kk], qa3[kk], b10, b11);
    }

    // ---- online softmax (log2 domain): row r lives in s0[0..1], s1[0..1],
    // row r + 8 in s0[2..3], s1[2..3]
    const int tok0 = (chunk_begin + j) * kChunk;
    float x[4] = {s0[0] * p.scale_log2, s0[1] * p.scale_log2, s1[0] * p.scale_log2,
                  s1[1] * p.scale_log2};
    float y[4] = {s0[2] * p.scale_log2, s0[3] * p.scale_log2, s1[2] * p.scale_log2,
                  s1[3] * p.scale_log2};
    if (tok0 + kChunk > t_end) {
      const int tk[4] = {2 * q4, 2 * q4 + 1, 8 + 2 * q4, 9 + 2 * q4};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tok0 + tk[e] >= t_end) x[e] = y[e] = -INFINITY;
      // Values behind the last key become 0 in shared memory: what their rows hold (NaN
      // among it) must not meet a probability of 0. (Masking the fragments of every chunk
      // instead: 17.9 against 16.9 us, small groups under short prefixes.)
      const int left = t_end - tok0;
      for (int i = lane; i < (kChunk - left) * (D / 8); i += 32)
        *reinterpret_cast<uint4*>(ring + st * SM::kStageBytes + G::kTileBytes +
                                  G::off(left + i / (D / 8), i % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }
    float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m_new = fmaxf(m_run, mx);
    const float alpha = exp2f(m_run - m_new);
    const uint32_t pa0 = pack2<T>(exp2f(x[0] - m_new), exp2f(x[1] - m_new));
    const uint32_t pa2 = pack2<T>(exp2f(x[2] - m_new), exp2f(x[3] - m_new));
    // Row sum of the rounded P the MMA consumes: normalisation matches the weights used.
    const float2 r0 = unpack2<T>(pa0);
    const float2 r1 = unpack2<T>(pa2);
    l_run = l_run * alpha + ((r0.x + r0.y) + (r1.x + r1.y));
    m_run = m_new;
    uint32_t pa1 = 0u, pa3 = 0u;
    float alpha_hi = 1.f;
    if constexpr (kWide) {
      float my = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
      my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 1));
      my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 2));
      const float mh_new = fmaxf(m_hi, my);
      alpha_hi = exp2f(m_hi - mh_new);
      pa1 = pack2<T>(exp2f(y[0] - mh_new), exp2f(y[1] - mh_new));
      pa3 = pack2<T>(exp2f(y[2] - mh_new), exp2f(y[3] - mh_new));
      const float2 h0 = unpack2<T>(pa1);
      const float2 h1 = unpack2<T>(pa3);
      l_hi = l_hi * alpha_hi + ((h0.x + h0.y) + (h1.x + h1.y));
      m_hi = mh_new;
    }
#pragma unroll
    for (int n = 0; n < kNTiles; ++n) {
      o[n][0] *= alpha;
      o[n][1] *= alpha;
      if constexpr (kWide) {
        o[n][2] *= alpha_hi;
        o[n][3] *= alpha_hi;
      }
    }

    // ---- O += P V
#pragma unroll
    for (int jj = 0; jj < kNTiles / 2; ++jj) {
      uint32_t b00, b01, b10, b11;
      ldsm_x4_t(vbase + G::off(pv_t, 2 * jj + pv_c), b00, b01, b10, b11);
      Mma<T>::run(o[2 * jj], pa0, pa1, pa2, pa3, b00, b01);
      Mma<T>::run(o[2 * jj + 1], pa0, pa1, pa2, pa3, b10, b11);
    }

    __syncwarp();
    if (lane == 0 && warp + (it + NS) * NW < nchunk) {
      fence_proxy_async_smem();  // our ldmatrix reads of this stage precede the refill
      issue(it + NS);
    }
  }

  if (stuck_at >= 0) {
    set_device_error(p.err, PS_DEVERR_TIMEOUT);
    // Drain this warp's copies still in flight (iterations stuck_at ..
    // stuck_at+NS-1 were issued, each wait bounded) before the CTA moves on.
    if (lane == 0) {
      for (int k = 0; k < NS; ++k) {
        const int i2 = stuck_at + k;
        if (warp + i2 * NW < nchunk)
          (void)mbar_wait_bounded(&wbar[(gbase + i2) % NS], ((gbase + i2) / NS) & 1);
      }
    }
  }
  __syncwarp();

  // Row sums across the quad (each lane summed only its own 4 keys).
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
  l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
  if constexpr (kWide) {
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
  }

  // ---- merge the NW warps' partial states through shared memory
  __syncthreads();  // every warp is done reading its ring; alias it as the merge area
  float* ms = reinterpret_cast<float*>(smem);   // [NW][R]
  float* ls = ms + NW * R;                      // [NW][R]
  float* os = ls + NW * R;                      // [NW][R][D]
  if (q4 == 0) {
    ms[warp * R + r] = m_run;
    ls[warp * R + r] = l_run;
    if constexpr (kWide) {
      ms[warp * R + r + 8] = m_hi;
      ls[warp * R + r + 8] = l_hi;
    }
  }
#pragma unroll
  for (int n = 0; n < kNTiles; ++n) {
    *reinterpret_cast<float2*>(&os[(warp * R + r) * D + n * 8 + 2 * q4]) =
        make_float2(o[n][0], o[n][1]);
    if constexpr (kWide)
      *reinterpret_cast<float2*>(&os[(warp * R + r + 8) * D + n * 8 + 2 * q4]) =
          make_float2(o[n][2], o[n][3]);
  }
  __syncthreads();

  const bool single = kShared ? nsplit <= 1 : nsplit == 1;
  // The prefix pass has left its pieces (and whatever runs after this kernel waits
  // for that pass too, since every CTA does).
  if constexpr (kShared) pdl_wait();
  const int npre = kShared && single ? shared_parts(p, pre) : 0;
  for (int idx = threadIdx.x; idx < group * (D / 4); idx += blockDim.x) {
    // kShared: neighbouring lanes take the heads, whose rows of a partial are neighbours.
    const int g = kShared ? idx % group : idx / (D / 4);
    const int d = (kShared ? idx / group : idx % (D / 4)) * 4;
    float mmax = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mmax = fmaxf(mmax, ms[w * R + g]);
    float lsum = 0.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = ms[w * R + g];
      const float sc = (mw == -INFINITY) ? 0.f : exp2f(mw - mmax);
      lsum += ls[w * R + g] * sc;
      const float4 ov = *reinterpret_cast<const float4*>(&os[(w * R + g) * D + d]);
      acc[0] += ov.x * sc;
      acc[1] += ov.y * sc;
      acc[2] += ov.z * sc;
      acc[3] += ov.w * sc;
    }
    if constexpr (kShared) merge_shared<D>(p, SharedRows(p, b, h, g), npre, d / 4, mmax, lsum, acc);
    const float inv = (lsum > 0.f) ? 1.f / lsum : 0.f;
    const int qh = h * group + g;
    if (single) {
      T* orow = static_cast<T*>(p.out) + b * p.out_stride + static_cast<int64_t>(qh) * D + d;
      uint2 packed;
      packed.x = pack2<T>(acc[0] * inv, acc[1] * inv);
      packed.y = pack2<T>(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<uint2*>(orow) = packed;
    } else {
      const int64_t slot = (static_cast<int64_t>(b) * p.max_splits + split) * p.num_q_heads + qh;
      *reinterpret_cast<float4*>(p.ws_o + slot * D + d) =
          make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      if (d == 0) p.ws_lse[slot] = (lsum > 0.f) ? mmax + log2f(lsum) : -INFINITY;
    }
  }
  // This warp's ring iterations in the unit (its chunks warp, warp + NW, ...).
  gbase += nchunk > warp ? static_cast<uint32_t>((nchunk - warp + NW - 1) / NW) : 0u;
  if constexpr (kList) {
    // The merge area aliases the ring: every thread is done with it before the
    // next unit's TMA writes it.
    fence_proxy_async_smem();
    __syncthreads();
  }
  }  // work units
  if constexpr (kShared) pdl_wait();  // also in CTAs that had no unit
}

// Longest-first order of the sequences for a decode launch: a counting sort of
// ctx_lens into 1024 buckets spanning [0, max ctx], buckets taken from the
// longest down (order inside a bucket is unspecified). One CTA.
__global__ void __launch_bounds__(1024) decode_order_kernel(const int32_t* ctx_lens, int n,
                                                            int32_t* order) {
  constexpr int kBuckets = 1024;
  __shared__ int hist[kBuckets];
  __shared__ int cursor[kBuckets];
  __shared__ int wmax[32];
  const int t = threadIdx.x;
  const int lane = t & 31;
  const int warp = t >> 5;
  hist[t] = 0;
  int mx = 0;
  for (int b = t; b < n; b += 1024) mx = max(mx, ctx_lens[b]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) wmax[warp] = mx;
  __syncthreads();
  if (warp == 0) {
    int m = wmax[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) wmax[0] = m;
  }
  __syncthreads();
  const int64_t span = static_cast<int64_t>(wmax[0]) + 1;
  auto bucket = [&](int ctx) -> int {
    const int c = max(ctx, 0);
    return static_cast<int>((static_cast<int64_t>(c) * kBuckets) / span);  // < kBuckets
  };
  for (int b = t; b < n; b += 1024) atomicAdd(&hist[bucket(ctx_lens[b])], 1);
  __syncthreads();
  // Start of bucket k = sequences in buckets above k: an exclusive scan over the
  // buckets in descending order (thread t owns bucket kBuckets - 1 - t).
  const int mine = hist[kBuckets - 1 - t];
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // hist read; wmax reused for warp totals
  if (lane == 31) wmax[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const int w = wmax[lane];
    int y = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    wmax[lane] = y - w;
  }
  __syncthreads();
  cursor[kBuckets - 1 - t] = wmax[warp] + x - mine;
  __syncthreads();
  for (int b = t; b < n; b += 1024) order[atomicAdd(&cursor[bucket(ctx_lens[b])], 1)] = b;
}

// ------------------------------------------------------------ host side
constexpr int kNW = 4;  // warps per CTA
constexpr int kNS = 2;  // TMA stages per warp
// Warps per CTA of the unsplit launch. One CTA streams one (sequence, KV head)
// through its warps' chunk loops, so the longest sequences' CTAs set a layer's
// length when the grid is one short wave; at head dim 64 a 16-token chunk is
// half the bytes, and eight warps keep those CTAs at the pace of the rest
// (Qwen2.5-0.5B geometry, 256 sequences: 54.4 against 60.6 us per layer;
// sixteen warps, one CTA per SM, 66 us). At head dim 128 four are faster
// (eight: 381 against 347 us per 8B layer).
template <int D>
constexpr int unsplit_warps() { return D == 64 ? 8 : kNW; }

template <typename T, int D, int BS, int R, bool kShared>
int launch_decode(const DecodeParams& p, const CUtensorMap& km, const CUtensorMap& vm,
                  cudaStream_t s, const SharedPrefix* prefix) {
  using SM = DecodeSmem<D, kNW, kNS>;
  const size_t smem = SM::bytes(p.table_cap);
  if (p.max_splits <= 1) {
    constexpr int NWU = unsplit_warps<D>();
    auto kern = paged_decode_kernel<T, D, NWU, kNS, BS, R, false, kShared>;
    static size_t configured[64] = {};
    const size_t smem_u = DecodeSmem<D, NWU, kNS>::bytes(p.table_cap);
    int st = reserve_smem(kern, smem_u, configured);
    if (st != PS_OK) return st;
    dim3 grid(p.num_kv_heads, 1, p.num_launch);
    if constexpr (kShared) {
      st = launch_shared_prefix(*prefix, s);
      if (st != PS_OK) return st;
    }
    const cudaError_t e = launch_pdl(kern, grid, dim3(NWU * 32), smem_u, s, p, km, vm);
    if (e != cudaSuccess)
      return fail(PS_ERR_CUDA, "ps_paged_decode: launch failed: %s", cudaGetErrorString(e));
    return check_launch("ps_paged_decode");
  }
  // Split-K: plan the (sequence, partition) units on the device, then one
  // persistent CTA per resident slot claims them; the grid does not depend on
  // the lengths, so the launch sequence can be captured in a CUDA graph.
  auto kern = paged_decode_kernel<T, D, kNW, kNS, BS, R, true, kShared>;
  static size_t configured[64] = {};
  int st = reserve_smem(kern, smem, configured);
  if (st != PS_OK) return st;
  static Resident cache[64];
  Resident res;
  st = resident_ctas(kern, "ps_paged_decode", kNW * 32, smem, cache, &res);
  if (st != PS_OK) return st;
  cudaError_t e = cudaSuccess;
  if (!p.planned) {
    e = launch_pdl(decode_plan_kernel<kShared>, dim3(1), dim3(1024), 0, s, p);
    if (e != cudaSuccess)
      return fail(PS_ERR_CUDA, "ps_paged_decode(plan): launch failed: %s", cudaGetErrorString(e));
  }
  if constexpr (kShared) {
    st = launch_shared_prefix(*prefix, s);
    if (st != PS_OK) return st;
  }
  e = launch_pdl(kern, dim3(res.per_sm * res.sms), dim3(kNW * 32), smem, s, p, km, vm);
  if (e != cudaSuccess)
    return fail(PS_ERR_CUDA, "ps_paged_decode: launch failed: %s", cudaGetErrorString(e));
  const int warps = p.num_launch * p.num_q_heads;
  e = launch_pdl(decode_combine_kernel<T, D, kShared>, dim3((warps + 3) / 4), dim3(128), 0, s, p);
  if (e != cudaSuccess)
    return fail(PS_ERR_CUDA, "ps_paged_decode(combine): launch failed: %s",
                cudaGetErrorString(e));
  return check_launch("ps_paged_decode(combine)");
}

template <typename T, int D, int R, bool kShared>
int dispatch_bs(const DecodeParams& p, const CUtensorMap& km, const CUtensorMap& vm,
                cudaStream_t s, int block_size, const SharedPrefix* prefix) {
  if (block_size == 8) return launch_decode<T, D, 8, R, kShared>(p, km, vm, s, prefix);
  if (block_size == 32) return launch_decode<T, D, 32, R, kShared>(p, km, vm, s, prefix);
  return launch_decode<T, D, 16, R, kShared>(p, km, vm, s, prefix);
}

template <typename T, int D, bool kShared>
int dispatch_rows(const DecodeParams& p, const CUtensorMap& km, const CUtensorMap& vm,
                  cudaStream_t s, int block_size, const SharedPrefix* prefix) {
  return p.group > 8 ? dispatch_bs<T, D, 16, kShared>(p, km, vm, s, block_size, prefix)
                     : dispatch_bs<T, D, 8, kShared>(p, km, vm, s, block_size, prefix);
}

template <bool kShared>
int dispatch_decode(const DecodeParams& p, const CUtensorMap& km, const CUtensorMap& vm,
                    cudaStream_t s, int dtype, int head_dim, int block_size,
                    const SharedPrefix* prefix = nullptr) {
  if (dtype == PS_DTYPE_BF16)
    return head_dim == 128
               ? dispatch_rows<__nv_bfloat16, 128, kShared>(p, km, vm, s, block_size, prefix)
               : dispatch_rows<__nv_bfloat16, 64, kShared>(p, km, vm, s, block_size, prefix);
  return head_dim == 128 ? dispatch_rows<__half, 128, kShared>(p, km, vm, s, block_size, prefix)
                         : dispatch_rows<__half, 64, kShared>(p, km, vm, s, block_size, prefix);
}

}  // namespace
}  // namespace ps

using namespace ps;

extern "C" int64_t ps_paged_decode_workspace_bytes(int num_seqs, int num_q_heads, int head_dim,
                                                   int block_size, int max_blocks_per_seq,
                                                   int split_tokens) {
  if (num_seqs <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_blocks_per_seq <= 0 ||
      block_size <= 0)
    return 0;
  const int part = split_tokens > 0 ? split_tokens : max_blocks_per_seq * block_size;
  const int64_t max_splits = (static_cast<int64_t>(max_blocks_per_seq) * block_size + part - 1) / part;
  if (max_splits <= 1) return 0;
  const int64_t rows = static_cast<int64_t>(num_seqs) * max_splits * num_q_heads;
  const int64_t o_bytes = ((rows * head_dim * 4) + 255) / 256 * 256;
  const int64_t lse_bytes = ((rows * 4) + 255) / 256 * 256;
  const int64_t item_bytes = ((static_cast<int64_t>(num_seqs) * max_splits * 4) + 255) / 256 * 256;
  return o_bytes + lse_bytes + item_bytes + 256;  // + the unit count
}

extern "C" int ps_paged_decode_order(const int32_t* ctx_lens, int num_seqs, int32_t* order,
                                     void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_order");
  const char* fn = "ps_paged_decode_order";
  if (num_seqs < 0 || num_seqs > 65535)
    return fail(PS_ERR_INVALID, "%s: num_seqs %d outside [0, 65535]", fn, num_seqs);
  if (num_seqs == 0) return PS_OK;
  if (!ctx_lens || !order) return fail(PS_ERR_INVALID, "%s: null pointer argument", fn);
  decode_order_kernel<<<1, 1024, 0, as_stream(stream)>>>(ctx_lens, num_seqs, order);
  return check_launch(fn);
}

extern "C" int ps_paged_decode(void* out, int64_t out_seq_stride, const void* query,
                               int64_t query_seq_stride, const void* k_pool, const void* v_pool,
                               int64_t num_blocks, const int32_t* block_tables,
                               int64_t block_table_stride, const int32_t* ctx_lens, int num_seqs,
                               int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                               int max_blocks_per_seq, float scale, int split_tokens,
                               void* workspace, int64_t workspace_bytes, int dtype,
                               int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode");
  return ps_paged_decode_ordered(out, out_seq_stride, query, query_seq_stride, k_pool, v_pool,
                                 num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                                 num_q_heads, num_kv_heads, head_dim, block_size,
                                 max_blocks_per_seq, scale, split_tokens, workspace,
                                 workspace_bytes, dtype, nullptr, device_error, stream);
}

namespace {
// The step's new token of each sequence, for the fused append.
struct NewToken {
  const void* key;
  int64_t key_stride;
  const void* value;
  int64_t value_stride;
  const int64_t* slots;
};

int decode_entry(const char* fn, void* out, int64_t out_seq_stride, const void* query,
                 int64_t query_seq_stride, const void* k_pool, const void* v_pool,
                 int64_t num_blocks, const int32_t* block_tables, int64_t block_table_stride,
                 const int32_t* ctx_lens, int num_seqs, int num_q_heads, int num_kv_heads,
                 int head_dim, int block_size, int max_blocks_per_seq, float scale,
                 int split_tokens, void* workspace, int64_t workspace_bytes, int dtype,
                 const int32_t* seq_order, const NewToken* nt, int32_t* device_error,
                 void* stream, int num_launch = -1, bool planned = false,
                 const SharedPrefix* shared = nullptr) {
  int part = 0, max_splits = 0, table_cap = 0;
  int vst = validate_decode(fn, out, out_seq_stride, query, query_seq_stride, k_pool, v_pool,
                            num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                            num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                            split_tokens, dtype, &part, &max_splits, &table_cap);
  if (vst != PS_OK || num_seqs == 0) return vst;
  if (num_launch < 0) num_launch = num_seqs;
  if (num_launch == 0) return PS_OK;
  const int group = num_q_heads / num_kv_heads;
  const int64_t rows = num_blocks * num_kv_heads * block_size;

  DecodeParams p{};
  if (max_splits > 1) {
    const int st = set_split_workspace(fn, &p, num_seqs, num_q_heads, head_dim, block_size,
                                       max_blocks_per_seq, split_tokens, max_splits, workspace,
                                       workspace_bytes);
    if (st != PS_OK) return st;
  }
  p.out = out;
  p.q = query;
  p.out_stride = out_seq_stride;
  p.q_stride = query_seq_stride;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.ctx_lens = ctx_lens;
  p.num_blocks = num_blocks;
  p.num_seqs = num_seqs;
  p.num_launch = num_launch;
  p.planned = planned;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = group;
  p.max_blocks = max_blocks_per_seq;
  p.block_size = block_size;
  p.part_tokens = part;
  p.max_splits = max_splits;
  p.table_cap = table_cap;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = device_error;
  p.seq_order = seq_order;
  if (nt) {
    if (!nt->key || !nt->value || !nt->slots)
      return fail(PS_ERR_INVALID, "%s: null key/value/slot_mapping", fn);
    if (nt->key_stride < static_cast<int64_t>(num_kv_heads) * head_dim ||
        nt->value_stride < static_cast<int64_t>(num_kv_heads) * head_dim ||
        (nt->key_stride % 8) || (nt->value_stride % 8) || !aligned(nt->key, 16) ||
        !aligned(nt->value, 16))
      return fail(PS_ERR_INVALID,
                  "%s: key/value must be 16-byte aligned with strides >= Hkv*D and %% 8", fn);
    if (num_blocks * block_size >= (int64_t(1) << 31))
      return fail(PS_ERR_INVALID, "%s: pool of %lld slots exceeds 2^31", fn,
                  (long long)(num_blocks * block_size));
    p.k_pool_w = const_cast<void*>(k_pool);
    p.v_pool_w = const_cast<void*>(v_pool);
    p.new_k = nt->key;
    p.new_v = nt->value;
    p.new_k_stride = nt->key_stride;
    p.new_v_stride = nt->value_stride;
    p.new_slots = nt->slots;
    p.num_slots = num_blocks * block_size;
  }

  CUtensorMap km, vm;
  const int box = block_size < kChunk ? block_size : kChunk;
  int st = get_pool_tmap(k_pool, static_cast<uint64_t>(rows), head_dim, box, &km);
  if (st != PS_OK) return st;
  st = get_pool_tmap(v_pool, static_cast<uint64_t>(rows), head_dim, box, &vm);
  if (st != PS_OK) return st;

  cudaStream_t s = as_stream(stream);
  if (shared) {
    p.shared_lens = shared->shared_lens;
    p.pre_o = shared->part_o;
    p.pre_ml = shared->part_ml;
    p.pre_keys = shared->piece_keys;
    p.pre_parts = shared->paired ? 2 : 1;
    p.pre_max = static_cast<int>(
        std::min<int64_t>(static_cast<int64_t>(shared->pieces) * shared->piece_keys, 0x7fffffff));
    return dispatch_decode<true>(p, km, vm, s, dtype, head_dim, block_size, shared);
  }
  return dispatch_decode<false>(p, km, vm, s, dtype, head_dim, block_size);
}
}  // namespace

extern "C" int ps_paged_decode_ordered(void* out, int64_t out_seq_stride, const void* query,
                                       int64_t query_seq_stride, const void* k_pool,
                                       const void* v_pool, int64_t num_blocks,
                                       const int32_t* block_tables, int64_t block_table_stride,
                                       const int32_t* ctx_lens, int num_seqs, int num_q_heads,
                                       int num_kv_heads, int head_dim, int block_size,
                                       int max_blocks_per_seq, float scale, int split_tokens,
                                       void* workspace, int64_t workspace_bytes, int dtype,
                                       const int32_t* seq_order, int32_t* device_error,
                                       void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_ordered");
  return decode_entry("ps_paged_decode", out, out_seq_stride, query, query_seq_stride, k_pool,
                      v_pool, num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                      num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, scale,
                      split_tokens, workspace, workspace_bytes, dtype, seq_order, nullptr,
                      device_error, stream);
}

extern "C" int ps_paged_decode_append(void* out, int64_t out_seq_stride, const void* query,
                                      int64_t query_seq_stride, const void* key,
                                      int64_t key_seq_stride, const void* value,
                                      int64_t value_seq_stride, const int64_t* slot_mapping,
                                      void* k_pool, void* v_pool, int64_t num_blocks,
                                      const int32_t* block_tables, int64_t block_table_stride,
                                      const int32_t* ctx_lens, int num_seqs, int num_q_heads,
                                      int num_kv_heads, int head_dim, int block_size,
                                      int max_blocks_per_seq, float scale, int split_tokens,
                                      void* workspace, int64_t workspace_bytes, int dtype,
                                      const int32_t* seq_order, int32_t* device_error,
                                      void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_append");
  const NewToken nt{key, key_seq_stride, value, value_seq_stride, slot_mapping};
  return decode_entry("ps_paged_decode_append", out, out_seq_stride, query, query_seq_stride,
                      k_pool, v_pool, num_blocks, block_tables, block_table_stride, ctx_lens,
                      num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                      max_blocks_per_seq, scale, split_tokens, workspace, workspace_bytes, dtype,
                      seq_order, &nt, device_error, stream);
}

extern "C" int ps_paged_decode_listed(void* out, int64_t out_seq_stride, const void* query,
                                      int64_t query_seq_stride, const void* k_pool,
                                      const void* v_pool, int64_t num_blocks,
                                      const int32_t* block_tables, int64_t block_table_stride,
                                      const int32_t* ctx_lens, int num_seqs,
                                      const int32_t* seq_list, int num_listed, int num_q_heads,
                                      int num_kv_heads, int head_dim, int block_size,
                                      int max_blocks_per_seq, float scale, int split_tokens,
                                      void* workspace, int64_t workspace_bytes, int dtype,
                                      int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_listed");
  const char* fn = "ps_paged_decode_listed";
  if (num_listed < 0 || num_listed > num_seqs)
    return fail(PS_ERR_INVALID, "%s: num_listed %d outside [0, num_seqs %d]", fn, num_listed,
                num_seqs);
  if (num_listed > 0 && !seq_list) return fail(PS_ERR_INVALID, "%s: null seq_list", fn);
  return decode_entry(fn, out, out_seq_stride, query, query_seq_stride, k_pool, v_pool,
                      num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                      num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, scale,
                      split_tokens, workspace, workspace_bytes, dtype, seq_list, nullptr,
                      device_error, stream, num_listed);
}

extern "C" int ps_paged_decode_plan(const int32_t* ctx_lens, int num_seqs,
                                    const int32_t* seq_order, int num_q_heads, int head_dim,
                                    int block_size, int max_blocks_per_seq, int split_tokens,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_plan");
  const char* fn = "ps_paged_decode_plan";
  if (num_seqs < 0 || num_seqs > 65535 || num_q_heads <= 0 || max_blocks_per_seq <= 0)
    return fail(PS_ERR_INVALID, "%s: bad sizes", fn);
  if (head_dim != 64 && head_dim != 128)
    return fail(PS_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", fn, head_dim);
  if (block_size != 8 && block_size != 16 && block_size != 32)
    return fail(PS_ERR_UNSUPPORTED, "%s: block_size %d unsupported (8, 16 or 32)", fn,
                block_size);
  const int unit = block_size > kChunk ? block_size : kChunk;
  if (split_tokens < 0 || (split_tokens % unit))
    return fail(PS_ERR_INVALID, "%s: split_tokens must be >= 0 and a multiple of %d", fn, unit);
  const int part = effective_part_tokens(split_tokens, max_blocks_per_seq, block_size);
  const int max_splits = (max_blocks_per_seq * block_size + part - 1) / part;
  if (num_seqs == 0 || max_splits <= 1) return PS_OK;  // nothing is split: no plan
  if (max_splits > 65535) return fail(PS_ERR_INVALID, "%s: too many partitions", fn);
  if (!ctx_lens) return fail(PS_ERR_INVALID, "%s: null ctx_lens", fn);
  DecodeParams p{};
  p.ctx_lens = ctx_lens;
  p.num_seqs = num_seqs;
  p.num_launch = num_seqs;
  p.max_blocks = max_blocks_per_seq;
  p.block_size = block_size;
  p.part_tokens = part;
  p.max_splits = max_splits;
  p.seq_order = seq_order;
  const int st = set_split_workspace(fn, &p, num_seqs, num_q_heads, head_dim, block_size,
                                     max_blocks_per_seq, split_tokens, max_splits, workspace,
                                     workspace_bytes);
  if (st != PS_OK) return st;
  const cudaError_t e =
      launch_pdl(decode_plan_kernel<false>, dim3(1), dim3(1024), 0, as_stream(stream), p);
  if (e != cudaSuccess) return fail(PS_ERR_CUDA, "%s: launch failed: %s", fn, cudaGetErrorString(e));
  return check_launch(fn);
}

extern "C" int ps_paged_decode_append_planned(
    void* out, int64_t out_seq_stride, const void* query, int64_t query_seq_stride,
    const void* key, int64_t key_seq_stride, const void* value, int64_t value_seq_stride,
    const int64_t* slot_mapping, void* k_pool, void* v_pool, int64_t num_blocks,
    const int32_t* block_tables, int64_t block_table_stride, const int32_t* ctx_lens,
    int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
    int max_blocks_per_seq, float scale, int split_tokens, void* workspace,
    int64_t workspace_bytes, int dtype, const int32_t* seq_order, int32_t* device_error,
    void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_append_planned");
  const NewToken nt{key, key_seq_stride, value, value_seq_stride, slot_mapping};
  return decode_entry("ps_paged_decode_append_planned", out, out_seq_stride, query,
                      query_seq_stride, k_pool, v_pool, num_blocks, block_tables,
                      block_table_stride, ctx_lens, num_seqs, num_q_heads, num_kv_heads, head_dim,
                      block_size, max_blocks_per_seq, scale, split_tokens, workspace,
                      workspace_bytes, dtype, seq_order, &nt, device_error, stream, -1, true);
}

// ------------------------------------------------------------ shared prefixes
namespace ps {
namespace {
// Pieces of the prefix pass and where a workspace holds their partials (outputs,
// then running maxima and sums, then the split-K workspace of the own keys).
struct SharedLayout {
  int piece_keys = 0;
  int pieces = 0;
  int64_t o_bytes = 0;
  int64_t ml_bytes = 0;
};

SharedLayout shared_layout(int num_seqs, int num_q_heads, int head_dim, int max_shared,
                           int split_keys) {
  SharedLayout l;
  if (max_shared <= 0) return l;
  const int64_t whole = (static_cast<int64_t>(max_shared) + 127) / 128 * 128;
  l.piece_keys = static_cast<int>(split_keys > 0 ? std::min<int64_t>(split_keys, whole)
                                                 : std::min<int64_t>(whole, 0x7fffff80));
  l.pieces = static_cast<int>((static_cast<int64_t>(max_shared) + l.piece_keys - 1) / l.piece_keys);
  // Room for two partials a piece: whether a piece leaves one or two depends on the
  // groups' sizes, which the workspace should not.
  const int64_t rows = 2 * static_cast<int64_t>(l.pieces) *
                       ((static_cast<int64_t>(num_seqs) * num_q_heads + 31) / 32 * 32);
  l.o_bytes = (rows * head_dim * 4 + 255) / 256 * 256;
  l.ml_bytes = (rows * 8 + 255) / 256 * 256;
  return l;
}
}  // namespace
}  // namespace ps

extern "C" int64_t ps_paged_decode_shared_workspace_bytes(int num_seqs, int num_q_heads,
                                                          int head_dim, int block_size,
                                                          int max_blocks_per_seq, int max_shared,
                                                          int split_keys, int split_tokens) {
  ps::NvtxRange nvtx_range("ps_paged_decode_shared_workspace_bytes");
  if (num_seqs <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_blocks_per_seq <= 0 ||
      block_size <= 0 || max_shared < 0 || max_shared > (1 << 30) || split_keys < 0 ||
      split_keys % 128)
    return 0;
  const SharedLayout l = shared_layout(num_seqs, num_q_heads, head_dim, max_shared, split_keys);
  return l.o_bytes + l.ml_bytes +
         ps_paged_decode_workspace_bytes(num_seqs, num_q_heads, head_dim, block_size,
                                         max_blocks_per_seq, split_tokens);
}

extern "C" int ps_paged_decode_shared(
    void* out, int64_t out_seq_stride, const void* query, int64_t query_seq_stride,
    const void* k_pool, const void* v_pool, int64_t num_blocks, const int32_t* block_tables,
    int64_t block_table_stride, const int32_t* ctx_lens, int num_seqs, const int32_t* group_starts,
    int num_groups, const int32_t* shared_lens, int max_group, int max_shared, int num_q_heads,
    int num_kv_heads, int head_dim, int block_size, int max_blocks_per_seq, float scale,
    int split_keys, int split_tokens, void* workspace, int64_t workspace_bytes, int dtype,
    const int32_t* seq_order, int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_shared");
  const char* fn = "ps_paged_decode_shared";
  int part = 0, max_splits = 0, table_cap = 0;
  const int vst = validate_decode(fn, out, out_seq_stride, query, query_seq_stride, k_pool, v_pool,
                                  num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                                  num_q_heads, num_kv_heads, head_dim, block_size,
                                  max_blocks_per_seq, split_tokens, dtype, &part, &max_splits,
                                  &table_cap);
  if (vst != PS_OK || num_seqs == 0) return vst;
  if (max_shared < 0 || max_shared > static_cast<int64_t>(max_blocks_per_seq) * block_size)
    return fail(PS_ERR_INVALID, "%s: max_shared %d outside [0, max_blocks_per_seq * block_size]",
                fn, max_shared);
  if (split_keys < 0 || split_keys % 128)
    return fail(PS_ERR_INVALID, "%s: split_keys %d must be a non-negative multiple of 128", fn,
                split_keys);
  if (num_groups < 0 || num_groups > num_seqs || max_group < 0 || max_group > num_seqs)
    return fail(PS_ERR_INVALID, "%s: num_groups %d and max_group %d must be in [0, num_seqs]", fn,
                num_groups, max_group);
  if (max_shared == 0 || num_groups == 0 || max_group == 0)  // nothing is shared
    return decode_entry(fn, out, out_seq_stride, query, query_seq_stride, k_pool, v_pool,
                        num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                        num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, scale,
                        split_tokens, workspace, workspace_bytes, dtype, seq_order, nullptr,
                        device_error, stream);
  if (!group_starts || !shared_lens)
    return fail(PS_ERR_INVALID, "%s: null group_starts/shared_lens", fn);
  const int64_t need = ps_paged_decode_shared_workspace_bytes(
      num_seqs, num_q_heads, head_dim, block_size, max_blocks_per_seq, max_shared, split_keys,
      split_tokens);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
    return fail(PS_ERR_INVALID, "%s: needs a 256-byte aligned workspace of %lld bytes", fn,
                (long long)need);
  const SharedLayout l = shared_layout(num_seqs, num_q_heads, head_dim, max_shared, split_keys);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  SharedPrefix a{};
  a.fn = fn;
  a.query = query;
  a.query_seq_stride = query_seq_stride;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.num_blocks = num_blocks;
  a.block_tables = block_tables;
  a.block_table_stride = block_table_stride;
  a.group_starts = group_starts;
  a.shared_lens = shared_lens;
  a.num_groups = num_groups;
  a.max_group = max_group;
  a.num_seqs = num_seqs;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.max_blocks = max_blocks_per_seq;
  a.pieces = l.pieces;
  a.piece_keys = l.piece_keys;
  a.paired = static_cast<int64_t>(max_group) * (num_q_heads / num_kv_heads) <= 128;
  a.scale = scale;
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + l.o_bytes);
  a.dtype = dtype;
  a.device_error = device_error;
  return decode_entry(fn, out, out_seq_stride, query, query_seq_stride, k_pool, v_pool, num_blocks,
                      block_tables, block_table_stride, ctx_lens, num_seqs, num_q_heads,
                      num_kv_heads, head_dim, block_size, max_blocks_per_seq, scale, split_tokens,
                      ws + l.o_bytes + l.ml_bytes, workspace_bytes - l.o_bytes - l.ml_bytes, dtype,
                      seq_order, nullptr, device_error, stream, -1, false, &a);
}

// ------------------------------------------------------------ allocation-free variant
// Split-K partials of ps_paged_decode_noalloc live in this file-scope device
// array instead of a caller-provided workspace. It is part of the library's
// device image, so every GPU that loads the library holds these bytes until
// the process exits, and all calls on a device share them.
namespace ps {
namespace {
constexpr int64_t kNoAllocScratchBytes = int64_t(64) << 20;  // 64 MiB per device
static __device__ __align__(256) uint8_t g_noalloc_scratch[kNoAllocScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex g_noalloc_mu;
void* g_noalloc_ptr[kMaxDevices] = {};
unsigned long long g_noalloc_ctx[kMaxDevices] = {};  // context id the address belongs to

// Driver calls that identify the calling thread's current context, fetched
// through the runtime (the library does not link libcuda directly).
using CtxGetCurrentFn = CUresult (*)(CUcontext*);
using CtxGetIdFn = CUresult (*)(CUcontext, unsigned long long*);
CtxGetCurrentFn g_ctx_get_current = nullptr;
CtxGetIdFn g_ctx_get_id = nullptr;
std::once_flag g_ctx_fns_once;

void load_ctx_fns() {
  cudaDriverEntryPointQueryResult q;
  void* fn = nullptr;
  if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &fn, cudaEnableDefault, &q) == cudaSuccess &&
      q == cudaDriverEntryPointSuccess)
    g_ctx_get_current = reinterpret_cast<CtxGetCurrentFn>(fn);
  fn = nullptr;
  if (cudaGetDriverEntryPoint("cuCtxGetId", &fn, cudaEnableDefault, &q) == cudaSuccess &&
      q == cudaDriverEntryPointSuccess)
    g_ctx_get_id = reinterpret_cast<CtxGetIdFn>(fn);
}

// Unique id of the calling thread's current context; 0 when none is current
// or the driver cannot say.
unsigned long long current_ctx_id() {
  std::call_once(g_ctx_fns_once, load_ctx_fns);
  if (!g_ctx_get_current || !g_ctx_get_id) return 0;
  CUcontext c = nullptr;
  unsigned long long id = 0;
  if (g_ctx_get_current(&c) != CUDA_SUCCESS || c == nullptr) return 0;
  if (g_ctx_get_id(c, &id) != CUDA_SUCCESS) return 0;
  return id;
}

// Device address of g_noalloc_scratch on the current device. In host code the
// symbol name is only a host-side handle, so the address is looked up with
// cudaGetSymbolAddress (with the device current) the first time a device
// needs it and cached. The cache is keyed by the device's context id: after
// cudaDeviceReset the context, and with it the array's address, is new, and
// the next call looks the address up again instead of using a stale one.
int noalloc_scratch(void** out) {
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess)
    return fail(PS_ERR_CUDA, "ps_paged_decode_noalloc: cudaGetDevice failed: %s",
                cudaGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices)
    return fail(PS_ERR_UNSUPPORTED, "ps_paged_decode_noalloc: device %d out of range", dev);
  const unsigned long long ctx = current_ctx_id();
  std::lock_guard<std::mutex> lock(g_noalloc_mu);
  if (g_noalloc_ptr[dev] == nullptr || ctx == 0 || ctx != g_noalloc_ctx[dev]) {
    void* p = nullptr;
    e = cudaGetSymbolAddress(&p, g_noalloc_scratch);
    if (e != cudaSuccess || p == nullptr)
      return fail(PS_ERR_CUDA, "ps_paged_decode_noalloc: cudaGetSymbolAddress failed: %s",
                  cudaGetErrorString(e));
    g_noalloc_ptr[dev] = p;
    g_noalloc_ctx[dev] = current_ctx_id();  // the lookup made the primary context current
  }
  *out = g_noalloc_ptr[dev];
  return PS_OK;
}
}  // namespace
}  // namespace ps

extern "C" int ps_paged_decode_noalloc(void* out, int64_t out_seq_stride, const void* query,
                                       int64_t query_seq_stride, const void* k_pool,
                                       const void* v_pool, int64_t num_blocks,
                                       const int32_t* block_tables, int64_t block_table_stride,
                                       const int32_t* ctx_lens, int num_seqs, int num_q_heads,
                                       int num_kv_heads, int head_dim, int block_size,
                                       int max_blocks_per_seq, float scale, int split_tokens,
                                       int dtype, int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_noalloc");
  const char* fn = "ps_paged_decode_noalloc";
  // The arguments are checked before the scratch is sized, so a bad argument
  // is reported as itself rather than as a request the scratch cannot hold.
  int part = 0, max_splits = 0, table_cap = 0;
  const int vst = validate_decode(fn, out, out_seq_stride, query, query_seq_stride, k_pool,
                                  v_pool, num_blocks, block_tables, block_table_stride, ctx_lens,
                                  num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                                  max_blocks_per_seq, split_tokens, dtype, &part, &max_splits,
                                  &table_cap);
  if (vst != PS_OK || num_seqs == 0) return vst;
  const int64_t need = max_splits > 1
                           ? ps_paged_decode_workspace_bytes(num_seqs, num_q_heads, head_dim,
                                                             block_size, max_blocks_per_seq,
                                                             split_tokens)
                           : 0;
  if (need > kNoAllocScratchBytes)
    return fail(PS_ERR_INVALID,
                "%s: split-K partials need %lld bytes, more than the %lld-byte built-in scratch; "
                "use fewer sequences, a larger split_tokens, or ps_paged_decode with a workspace",
                fn, (long long)need, (long long)kNoAllocScratchBytes);
  void* scratch = nullptr;
  if (need > 0) {
    const int st = noalloc_scratch(&scratch);
    if (st != PS_OK) return st;
  }
  // Nothing in the scratch needs clearing between calls: the plan kernel of
  // each call rewrites the unit list and count and resets the claim counter
  // before the decode reads them, and the combine reads only partials written
  // by the same call.
  return decode_entry(fn, out, out_seq_stride, query, query_seq_stride, k_pool, v_pool,
                      num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                      num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, scale,
                      split_tokens, scratch, need > 0 ? kNoAllocScratchBytes : 0, dtype, nullptr,
                      nullptr, device_error, stream);
}
