// Paged decode attention (one query token per sequence, GQA) over an 8-bit KV
// cache (quant.cuh) for sm_100a.
//
// With codes k, v and per-row scales a_n (K) and b_n (V) of key n:
//   s_n = scale * a_n * (q . k_n)     o = sum_n softmax(s)_n * b_n * v_n
// so both scales stay outside the matrix products: a_n multiplies a score, b_n a
// probability. The products run on fp16 warp MMAs: every e4m3 or int8 code is an
// fp16 value, so the probabilities are rounded (2^-11 relative), and the queries
// where a head's elements differ most: each head is first brought to [-2, 2) by a
// power of two, and there fp16's step is 2^-24 from 2^-14 down. Elements below 2^-14 (bf16
// queries, of fewer bits: 2^-17) of that range lose low bits, 2^-25 at most, and those
// below 2^-25 all of them: per product what fp32 sums of the larger ones lose too.
//
// A probability times b_n must fit fp16 too, whatever the b_n are, and keep its
// precision where the sum has its weight. So beside the running maximum m of the
// scores (for the softmax sum) each head has a running maximum M of
// s_n + log2 b_n, and the second product takes
//   P'_n = 2^(s_n + log2 b_n - M + 7)
// Both maxima move only when passed by 8 (2^8), so P' is below 2^15.2 and a term
// keeps fp16's full precision down to 2^-21 of the largest one; O is rescaled, in
// fp32, when M moves. P' is formed as (p_n F) (b_n H) with p_n = 2^(s_n - m) and
// F H = f = 2^(m - M + 7), F = max(f, 1): p_n is at most 2^8 and b_n below 2^121, so no
// factor overflows as long as f is at most 2^119. That is M >= m - 112, which M is held to:
// only where every value is below 2^-112 of what a probability of 1 weighs do terms start lower
// than 2^7. (b_n f in one product was infinite where the top key's values were zeros and
// others', far below it, were not, and a NaN where their p_n was 0.) A p_n below 2^-126 is 0.
//
// Work decomposition as in paged_decode.cu: one CTA per (KV head, sequence), or
// persistent CTAs claiming (KV head, partition) units; each warp owns a ring of
// stages of 32 keys filled by TMA (codes) and 16-byte asynchronous copies (scales). The group of
// query heads is the N side of the MMAs and the keys (for S) or the dims (for O)
// the M side, so eight heads fill a tile that would be half padding the other
// way round:
//   S^T[16 keys x 8 heads] = K[16 x D] . Q^T      (D/16 MMAs)
//   O^T[16 dims x 8 heads] += V^T[16 x 16 keys] . P^T
// The K codes of four neighbouring dims reach a lane as one 32-bit register; which
// of the MMA's k indices they stand for is free as long as Q is laid out alike.
//
// Bound by HBM, with half the bytes of the 16-bit cache to hide the same work behind:
// 256 sequences U[512,4096], Hq 32, Hkv 8, D 128, e4m3, blocks of 16 take 190-209 us by
// box for 1.293 GB (6,190-6,820 GB/s; the 16-bit cache takes 347 us). That is 0.96-1.05 of
// a copy's rate, which pays for writes too; of a plain read of as many bytes
// (ps_stream_read, 7,030-7,130 GB/s on the box of the 190 us) it is 0.96. A warp spends
// 1,200-1,500 cycles on a stage of 32 keys and about 800 on issuing the next one; twelve
// warps per SM hide both. Measured and not kept: 2 to 16 warps of 1 to 4 stages and stages of 16 keys (193 to 324 us); a producer warp per CTA
// feeding four others through a shared ring (870 cycles to issue a stage: 226 us with
// TMA, 202 us with 16-byte asynchronous copies); persistent CTAs taking over pending
// ones with the next unit's keys prefetched during the merge (no gain: the other CTAs of
// an SM cover a CTA's start). Partitions of 512 keys (64 sequences lognormal to 32768, Hq
// 64) take 78 us for 338 MB: a unit's lookup, queries and merge are a third of its time.
#include <cudaTypedefs.h>

#include "decode_common.cuh"
#include "quant.cuh"

namespace ps {
namespace {

constexpr int kKeys = 32;  // keys per stage

struct QuantDecodeParams {
  DecodeParams d;
  const float* k_scale;  // [num_blocks][Hkv][block_size]
  const float* v_scale;
};

template <int D, int NW, int NS>
struct QuantSmem {
  static constexpr int kTileBytes = kKeys * D;  // K or V codes of one stage
  static constexpr int kRingBytes = NW * NS * 2 * kTileBytes;
  static constexpr int kScaleOffset = kRingBytes;  // per stage: 32 K scales, 32 V scales
  static constexpr int kBarOffset = kScaleOffset + NW * NS * 2 * kKeys * 4;
  static constexpr int kTableOffset = kBarOffset + NW * NS * 8;
  static_assert(NW * 16 * (D + 2) * 4 <= kRingBytes, "merge area must fit in the ring");
  static size_t bytes(int table_cap) {
    return 1024 /*alignment slack*/ + kTableOffset + static_cast<size_t>(table_cap) * 4;
  }
  // Byte offset of 16-byte chunk c of key t inside a swizzled tile: a row of 128
  // bytes spreads over 8 rows (128-byte swizzle), one of 64 bytes over 4 pairs of
  // rows (64-byte swizzle); ldmatrix's 8 rows then hit 8 different groups of banks.
  __device__ __forceinline__ static uint32_t off(int t, int c) {
    return D == 128 ? t * 128 + ((c ^ (t & 7)) << 4) : t * 64 + ((c ^ ((t >> 1) & 3)) << 4);
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Asynchronous 16-byte copy to shared memory, and the arrival on `bar` of this thread's
// copies so far once they have landed (counted in the barrier's arrivals).
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Transposes an 8x8 matrix of 16-bit elements held two per lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// T = type of the queries and the output; C = code type; R = 8 or 16 head
// columns; kList as in paged_decode_kernel.
template <typename T, typename C, int D, int NW, int NS, int BS, int R, bool kList>
__global__ void __launch_bounds__(NW * 32)
    paged_decode_quant_kernel(const QuantDecodeParams qp, const __grid_constant__ CUtensorMap kmap,
                              const __grid_constant__ CUtensorMap vmap) {
  static_assert(R == 8 || R == 16, "8 or 16 head columns");
  using SM = QuantSmem<D, NW, NS>;
  const DecodeParams& p = qp.d;
  constexpr int kNT = R / 8;       // head tiles
  constexpr int kKSteps = D / 16;  // k steps of S, dim tiles of O
  constexpr int kBox = BS < kKeys ? BS : kKeys;
  constexpr int kBoxes = kKeys / kBox;

  int h = blockIdx.x;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int group = p.group;
  const int r = lane >> 2;  // key (S) or dim pair (O) row
  const int q4 = lane & 3;  // heads 2 q4, 2 q4 + 1 of a head tile

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::kBarOffset);
  int32_t* table = reinterpret_cast<int32_t*>(smem + SM::kTableOffset);
  pdl_trigger();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
    for (int i = 0; i < NW * NS; ++i) mbar_init(&bars[i], 33);  // the TMA bytes, and every lane's scales
    fence_barrier_init();
  }
  pdl_wait();

  // Work units as in paged_decode_kernel. kList: a CTA's first unit is its own index, those
  // past the grid are claimed from the counter one ahead (a launch with fewer units than
  // CTAs leaves it alone: the atomics to one address took 1 us of 12). Looking the next
  // unit up during this one's merge was 3% slower than at its start (more registers and
  // waits in the merge), claiming two ahead 5% (uneven work at the end).
  __shared__ int claimed[2];
  int total = 0, next = 0;
  if constexpr (kList) {
    // A unit list planned for another step (a caller error) can hold more entries than
    // this launch's workspace holds, or sequences it does not have: the count is clamped
    // to the capacity and every entry is checked.
    total = min(max(*p.item_count, 0), p.num_seqs * p.max_splits) * p.num_kv_heads;
  }
  uint32_t gbase = 0;  // this warp's ring iterations so far
  for (int k = 0;; ++k) {
    int split = 0, b;
    if constexpr (kList) {
      int u = blockIdx.x;
      if (k > 0) {
        if (threadIdx.x == 0) claimed[k & 1] = next;
        __syncthreads();
        u = claimed[k & 1];
      }
      if (u >= total) break;
      const int grid = static_cast<int>(gridDim.x);
      if (threadIdx.x == 0) next = total > grid ? grid + atomicAdd(p.item_next, 1) : total;
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
      b = ordered_seq(p, blockIdx.z);
      if (b < 0) break;
    }
    // The first block ids need not wait for the length: entries below max_blocks exist, and
    // those past the context are dropped.
    const int first_blk = split * p.part_tokens / BS;
    const int32_t* bt = p.block_tables + static_cast<int64_t>(b) * p.bt_stride + first_blk;
    const int32_t early = first_blk + static_cast<int>(threadIdx.x) < p.max_blocks ? bt[threadIdx.x] : 0;
    int ctx = p.ctx_lens[b];
    // The queries: loaded before the first stages' copies are issued where a CTA has one
    // unit (14.3 against 14.9 us, Qwen geometry), after them in a list (1 us of 80).
    uint2 qraw[kNT][kKSteps];
    auto load_q = [&]() {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        const bool real = nt * 8 + r < group;
        const T* qrow = static_cast<const T*>(p.q) + b * p.q_stride +
                        static_cast<int64_t>(h * group + (real ? nt * 8 + r : 0)) * D + 4 * q4;
#pragma unroll
        for (int kk = 0; kk < kKSteps; ++kk)
          qraw[nt][kk] = real ? *reinterpret_cast<const uint2*>(qrow + 16 * kk) : make_uint2(0u, 0u);
      }
    };
    if constexpr (!kList) load_q();
    if (ctx > p.max_blocks * BS) {
      if (threadIdx.x == 0 && split == 0) set_device_error(p.err, PS_DEVERR_LENGTH);
      ctx = 0;
    }
    const int nsplit = (ctx + p.part_tokens - 1) / p.part_tokens;
    if (ctx <= 0) {
      if (split == 0) {
        T* o = static_cast<T*>(p.out) + b * p.out_stride + static_cast<int64_t>(h) * group * D;
        for (int i = threadIdx.x; i < group * D; i += blockDim.x) o[i] = from_f32<T>(0.f);
      }
      continue;
    }
    if (split >= nsplit) continue;  // a stale list's entry

    const int t_begin = split * p.part_tokens;
    const int n_keys = min(ctx - t_begin, p.part_tokens);
    const int nchunk = (n_keys + kKeys - 1) / kKeys;
    const int nblk = (n_keys + BS - 1) / BS;
    for (int i = threadIdx.x; i < nblk; i += NW * 32) {
      int32_t id = i < NW * 32 ? early : bt[i];
      if (id < 0 || id >= p.num_blocks) {
        set_device_error(p.err, PS_DEVERR_BLOCK_ID);
        id = 0;  // read a valid block instead of faulting; the error bit reports it
      }
      table[i] = id;
    }
    __syncthreads();

    // Loads of warp-local iteration `it` (keys [32 j, 32 j + 32), j = warp + it NW): one
    // lane issues the rows' TMA copies, sixteen copy four scales each (a bulk copy per box
    // and scale pool would double the warp's issue time). A box past the partition's last
    // block re-reads that block (its keys are masked).
    auto issue = [&](int it) {
      const int j = warp + it * NW;
      const int st = warp * NS + (gbase + it) % NS;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[st], 2 * SM::kTileBytes);
#pragma unroll
        for (int x = 0; x < kBoxes; ++x) {
          const int tok = j * kKeys + x * kBox;
          const int32_t row =
              (table[min(tok / BS, nblk - 1)] * p.num_kv_heads + h) * BS + tok % BS;
          uint8_t* dst = smem + st * 2 * SM::kTileBytes + x * kBox * D;
          tma_load_2d(dst, &kmap, &bars[st], 0, row);
          tma_load_2d(dst + SM::kTileBytes, &vmap, &bars[st], 0, row);
        }
      }
      if (lane < 16) {
        const int tok = j * kKeys + (lane & 7) * 4;
        const int64_t row =
            static_cast<int64_t>(table[min(tok / BS, nblk - 1)] * p.num_kv_heads + h) * BS + tok % BS;
        cp_async16(smem + SM::kScaleOffset + st * 2 * kKeys * 4 + lane * 16,
                   (lane < 8 ? qp.k_scale : qp.v_scale) + row);
      }
      cp_async_arrive(&bars[st]);
    };
#pragma unroll
    for (int it = 0; it < NS; ++it)
      if (warp + it * NW < nchunk) issue(it);

    if constexpr (kList) load_q();
    // Q as the B operand: lane holds head n = lane/4 of each head tile, dims
    // 16 kk + 4 q4 .. + 3 of k step kk, as fp16 times 2^-e_head. The factor that
    // turns an S element of heads 2 q4, 2 q4 + 1 into log2 units goes to qs.
    uint32_t qb[kNT][kKSteps][2];
    float2 qs[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      float2 x[kKSteps][2];
      float mx = 0.f;
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) {
        x[kk][0] = unpack2<T>(qraw[nt][kk].x);
        x[kk][1] = unpack2<T>(qraw[nt][kk].y);
        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[kk][0].x), fabsf(x[kk][0].y)),
                             fmaxf(fabsf(x[kk][1].x), fabsf(x[kk][1].y))));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // Exponent of the head's largest |q|, clamped so that 2^-e is a normal number.
      const int e = min(max(static_cast<int>(__float_as_uint(mx) >> 23) - 127, -120), 120);
      const float down = pow2f(-e);
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) {
        qb[nt][kk][0] = pack2<__half>(x[kk][0].x * down, x[kk][0].y * down);
        qb[nt][kk][1] = pack2<__half>(x[kk][1].x * down, x[kk][1].y * down);
      }
      const float up = p.scale_log2 * pow2f(e);
      qs[nt].x = __shfl_sync(0xffffffffu, up, 8 * q4);      // a lane of head 2 q4
      qs[nt].y = __shfl_sync(0xffffffffu, up, 8 * q4 + 4);  // a lane of head 2 q4 + 1
    }

    float o[kNT][kKSteps][4];  // [dims 16 kk + 2 r (+1)][heads 2 q4, 2 q4 + 1]: {d0h0, d0h1, d1h0, d1h1}
    // Per head: running maxima of s (m) and s + log2 b (mv), the factor of P'
    // 2^(m - mv + 7), and this lane's part of the softmax sum.
    float2 m[kNT], mv[kNT], f[kNT], l[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk) o[nt][kk][0] = o[nt][kk][1] = o[nt][kk][2] = o[nt][kk][3] = 0.f;
      m[nt] = mv[nt] = make_float2(-INFINITY, -INFINITY);
      f[nt] = l[nt] = make_float2(0.f, 0.f);
    }
    int stuck_at = -1;

    const int row8 = (lane & 7) + ((lane >> 3) & 1) * 8;  // ldmatrix: row of this lane's address
    const int chunk1 = lane >> 4;                         // and its 16-byte chunk (0 or 1)

    // One stage: kTail when fewer than 32 of its keys belong to the partition. A lane's
    // two heads of a tile go through the softmax as packed pairs.
    auto step = [&](auto tail, uint32_t kbase, const float* ks, int left) {
      constexpr bool kTail = decltype(tail)::value;
      const uint32_t vbase = kbase + SM::kTileBytes;

      // ---- S^T: two key tiles of 16
      float s[2][kNT][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) s[kt][nt][0] = s[kt][nt][1] = s[kt][nt][2] = s[kt][nt][3] = 0.f;
      }
#pragma unroll
      for (int kk = 0; kk < kKSteps; kk += 2) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          uint32_t w[4];
          ldsm_x4(kbase + SM::off(kt * 16 + row8, kk + chunk1), w[0], w[1], w[2], w[3]);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t a0, a1, a2, a3;
            decode4<C>(w[2 * x], a0, a2);
            decode4<C>(w[2 * x + 1], a1, a3);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
              Mma<__half>::run(s[kt][nt], a0, a1, a2, a3, qb[nt][kk + x][0], qb[nt][kk + x][1]);
          }
        }
      }

      // ---- scores in log2 units; this lane's keys are r, r + 8, r + 16, r + 24
      float vs[4];
      float2 x[4][kNT];
      float2 top[kNT], topv[kNT];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = r + 8 * i;
        const bool live = !kTail || key < left;
        const float a = ks[key];
        vs[i] = live ? ks[kKeys + key] : 0.f;
        // log2 b to within 0.09: the bits of a float, read as an integer, are linear
        // in its logarithm between powers of two. Only the choice of M uses it.
        const float lb = fmaf(static_cast<float>(__float_as_int(vs[i])), 0x1p-23f, -127.f);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const float* sp = &s[i >> 1][nt][(i & 1) * 2];
          x[i][nt] = __fmul2_rn(make_float2(sp[0], sp[1]), __fmul2_rn(make_float2(a, a), qs[nt]));
          if (!live) x[i][nt] = make_float2(-INFINITY, -INFINITY);
          const float2 y = __fadd2_rn(x[i][nt], make_float2(lb, lb));
          top[nt].x = i ? fmaxf(top[nt].x, x[i][nt].x) : x[i][nt].x;
          top[nt].y = i ? fmaxf(top[nt].y, x[i][nt].y) : x[i][nt].y;
          topv[nt].x = i ? fmaxf(topv[nt].x, y.x) : y.x;
          topv[nt].y = i ? fmaxf(topv[nt].y, y.y) : y.y;
        }
      }
      // ---- running maxima, moved only when passed by 2^8
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
        move |= top[nt].x > m[nt].x + 8.f || top[nt].y > m[nt].y + 8.f ||
                topv[nt].x > mv[nt].x + 8.f || topv[nt].y > mv[nt].y + 8.f;
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          auto raise = [&](float t, float u, float& m_, float& mv_, float& l_, float& f_) {
#pragma unroll
            for (int o_ = 4; o_ < 32; o_ <<= 1) {
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o_));
              u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, o_));
            }
            const float m_new = fmaxf(m_, t);
            const float mv_new = fmaxf(fmaxf(mv_, u), m_new - 112.f);
            l_ *= m_new == -INFINITY ? 1.f : ex2(m_ - m_new);
            const float alpha = mv_new == -INFINITY ? 1.f : ex2(mv_ - mv_new);
            m_ = m_new;
            mv_ = mv_new;
            f_ = ex2(m_new - mv_new + 7.f);
            return alpha;
          };
          const float al0 = raise(top[nt].x, topv[nt].x, m[nt].x, mv[nt].x, l[nt].x, f[nt].x);
          const float al1 = raise(top[nt].y, topv[nt].y, m[nt].y, mv[nt].y, l[nt].y, f[nt].y);
#pragma unroll
          for (int kk = 0; kk < kKSteps; ++kk) {
            o[nt][kk][0] *= al0;
            o[nt][kk][1] *= al1;
            o[nt][kk][2] *= al0;
            o[nt][kk][3] *= al1;
          }
        }
      }

      // ---- P^T as the B operand: [kt][nt][keys 0-7 | 8-15]
      // P' is rounded to fp16: 2^-11 of a probability, an eighth of a bf16 output's own
      // rounding but all of an fp16 output's. There a second fp16 term holds what the first
      // one lost (one more MMA per tile; the tensor pipe is a fifth busy).
      constexpr bool kTwoTerms = std::is_same<T, __half>::value;
      uint32_t pb[2][kNT][2];
      [[maybe_unused]] uint32_t pl[2][kNT][2];
      float2 up[kNT], down[kNT];  // F and H
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        up[nt] = make_float2(fmaxf(f[nt].x, 1.f), fmaxf(f[nt].y, 1.f));
        down[nt] = make_float2(fminf(f[nt].x, 1.f), fminf(f[nt].y, 1.f));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const float2 z = __fadd2_rn(x[i][nt], make_float2(-m[nt].x, -m[nt].y));
          const float2 pr = make_float2(ex2(z.x), ex2(z.y));
          l[nt] = __fadd2_rn(l[nt], pr);
          const float2 pv = __fmul2_rn(__fmul2_rn(pr, up[nt]),
                                       __fmul2_rn(make_float2(vs[i], vs[i]), down[nt]));
          const uint32_t hi = pack2<__half>(pv);
          pb[i >> 1][nt][i & 1] = transpose8x8(hi);
          if constexpr (kTwoTerms) {
            const float2 back = unpack2<__half>(hi);
            pl[i >> 1][nt][i & 1] =
                transpose8x8(pack2<__half>(__fadd2_rn(pv, make_float2(-back.x, -back.y))));
          }
        }
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        // Codes of keys past the end become 0: what a block holds there (NaN codes
        // among it) must not meet a probability of 0. This lane's keys are
        // 2 q4, 2 q4 + 1 (low and high half of a register) and the same plus 8.
        uint32_t live0 = 0xffffffffu, live1 = 0xffffffffu;
        if constexpr (kTail) {
          const int k0 = left - kt * 16 - 2 * q4;
          live0 = k0 >= 2 ? 0xffffffffu : k0 == 1 ? 0x0000ffffu : 0u;
          live1 = k0 >= 10 ? 0xffffffffu : k0 == 9 ? 0x0000ffffu : 0u;
        }
#pragma unroll
        for (int kk = 0; kk < kKSteps; kk += 2) {
          uint32_t w[4];
          ldsm_x4_t(vbase + SM::off(kt * 16 + row8, kk + chunk1), w[0], w[1], w[2], w[3]);
#pragma unroll
          for (int x2 = 0; x2 < 2; ++x2) {
            // bytes (key0 dim0, key0 dim1, key1 dim0, key1 dim1) -> pairs of keys per dim
            uint32_t a0, a1, a2, a3;
            if constexpr (kTail) {
              w[2 * x2] &= live0;
              w[2 * x2 + 1] &= live1;
            }
            decode4<C>(__byte_perm(w[2 * x2], 0, 0x3120), a0, a1);
            decode4<C>(__byte_perm(w[2 * x2 + 1], 0, 0x3120), a2, a3);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
            {
              Mma<__half>::run(o[nt][kk + x2], a0, a1, a2, a3, pb[kt][nt][0], pb[kt][nt][1]);
              if constexpr (kTwoTerms)
                Mma<__half>::run(o[nt][kk + x2], a0, a1, a2, a3, pl[kt][nt][0], pl[kt][nt][1]);
            }
          }
        }
      }
    };

    for (int it = 0; warp + it * NW < nchunk; ++it) {
      const int st = warp * NS + (gbase + it) % NS;
      if (!mbar_wait_bounded(&bars[st], ((gbase + it) / NS) & 1)) {
        stuck_at = it;
        break;
      }
      const uint32_t kbase = smem_u32(smem + st * 2 * SM::kTileBytes);
      const float* ks = reinterpret_cast<const float*>(smem + SM::kScaleOffset + st * 2 * kKeys * 4);
      const int left = n_keys - (warp + it * NW) * kKeys;  // keys of the partition from here on
      if (left >= kKeys) step(std::false_type{}, kbase, ks, left);
      else step(std::true_type{}, kbase, ks, left);
      __syncwarp();
      if (warp + (it + NS) * NW < nchunk) {
        fence_proxy_async_smem();  // our reads of this stage precede the refill
        issue(it + NS);
      }
    }

    if (stuck_at >= 0) {
      set_device_error(p.err, PS_DEVERR_TIMEOUT);
      // Drain this warp's copies still in flight, each wait bounded.
      if (lane == 0) {
        for (int x = 0; x < NS; ++x) {
          const int i2 = stuck_at + x;
          if (warp + i2 * NW < nchunk)
            (void)mbar_wait_bounded(&bars[warp * NS + (gbase + i2) % NS], ((gbase + i2) / NS) & 1);
        }
      }
    }
    __syncwarp();

    // ---- merge the warps through shared memory
    __syncthreads();  // every warp is done reading its ring; alias it as the merge area
    float* ms = reinterpret_cast<float*>(smem);  // [NW][R]
    float* ls = ms + NW * R;                     // [NW][R]
    float* os = ls + NW * R;                     // [NW][R][D]
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = e ? l[nt].y : l[nt].x;  // each lane summed its own keys
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
        t += __shfl_xor_sync(0xffffffffu, t, 16);
        const int head = nt * 8 + 2 * q4 + e;
        const float fe = e ? f[nt].y : f[nt].x;
        const float unit = fe > 0.f ? 1.f / fe : 0.f;  // O / f is in units of 2^m, like l
        if (r == 0) {
          ms[warp * R + head] = e ? m[nt].y : m[nt].x;
          ls[warp * R + head] = t;
        }
#pragma unroll
        for (int kk = 0; kk < kKSteps; ++kk)
          *reinterpret_cast<float2*>(&os[(warp * R + head) * D + 16 * kk + 2 * r]) =
              make_float2(o[nt][kk][e] * unit, o[nt][kk][2 + e] * unit);
      }
    }
    __syncthreads();

    const bool single = nsplit == 1;
    for (int idx = threadIdx.x; idx < group * (D / 4); idx += blockDim.x) {
      const int g = idx / (D / 4);
      const int d = (idx % (D / 4)) * 4;
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
      // lsum is positive for finite scores; a NaN score leaves it NaN, and the output with it
      const float inv = 1.f / lsum;
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
        if (d == 0) p.ws_lse[slot] = mmax + log2f(lsum);
      }
    }
    gbase += nchunk > warp ? static_cast<uint32_t>((nchunk - warp + NW - 1) / NW) : 0u;
    if constexpr (kList) {
      // The merge area aliases the ring: every thread is done with it before the
      // next unit's copies write it.
      fence_proxy_async_smem();
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------ host side
constexpr int kNW = 4;  // warps per CTA
constexpr int kNS = 2;  // stages of 32 keys per warp
// Warps per CTA of the unsplit launch: at head dim 64 a stage is half the bytes, and a CTA's
// longest sequence sets the launch's length (96 sequences U[1,2000], Hq 14, Hkv 2, int8:
// 16.9 against 19.2 us); at head dim 128 eight are slower (256 sequences: 247 against 199).
template <int D>
constexpr int unsplit_warps() { return D == 64 ? 8 : kNW; }

template <typename T, typename C, int D, int BS, int R>
int launch_quant(const QuantDecodeParams& qp, const CUtensorMap& km, const CUtensorMap& vm,
                 cudaStream_t s) {
  const DecodeParams& p = qp.d;
  using SM = QuantSmem<D, kNW, kNS>;
  const size_t smem = SM::bytes(p.table_cap);
  const char* fn = "ps_paged_decode_quant";
  if (p.max_splits <= 1) {
    constexpr int NWU = unsplit_warps<D>();
    auto kern = paged_decode_quant_kernel<T, C, D, NWU, kNS, BS, R, false>;
    static size_t configured[64] = {};
    const size_t smem_u = QuantSmem<D, NWU, kNS>::bytes(p.table_cap);
    int st = reserve_smem(kern, smem_u, configured);
    if (st != PS_OK) return st;
    const cudaError_t e = launch_pdl(kern, dim3(p.num_kv_heads, 1, p.num_launch), dim3(NWU * 32),
                                     smem_u, s, qp, km, vm);
    if (e != cudaSuccess) return fail(PS_ERR_CUDA, "%s: launch failed: %s", fn, cudaGetErrorString(e));
    return check_launch(fn);
  }
  auto kern = paged_decode_quant_kernel<T, C, D, kNW, kNS, BS, R, true>;
  static size_t configured[64] = {};
  int st = reserve_smem(kern, smem, configured);
  if (st != PS_OK) return st;
  static Resident cache[64];
  Resident res;
  st = resident_ctas(kern, fn, kNW * 32, smem, cache, &res);
  if (st != PS_OK) return st;
  cudaError_t e = cudaSuccess;
  if (!p.planned) {
    e = launch_pdl(decode_plan_kernel<false>, dim3(1), dim3(1024), 0, s, p);
    if (e != cudaSuccess)
      return fail(PS_ERR_CUDA, "%s(plan): launch failed: %s", fn, cudaGetErrorString(e));
  }
  e = launch_pdl(kern, dim3(res.per_sm * res.sms), dim3(kNW * 32), smem, s, qp, km, vm);
  if (e != cudaSuccess) return fail(PS_ERR_CUDA, "%s: launch failed: %s", fn, cudaGetErrorString(e));
  const int warps = p.num_launch * p.num_q_heads;
  e = launch_pdl(decode_combine_kernel<T, D>, dim3((warps + 3) / 4), dim3(128), 0, s, p);
  if (e != cudaSuccess)
    return fail(PS_ERR_CUDA, "%s(combine): launch failed: %s", fn, cudaGetErrorString(e));
  return check_launch(fn);
}

// Nine heads and more take a second head tile (R 16): at head dim 128 its fragments and
// accumulators bring the kernel from 123-168 registers to 168-226, which leaves two CTAs an SM
// in place of three in all but a few forms. 256 sequences U[512,4096], Hkv 2, D 128, e4m3:
// 8 heads a KV head 58-59 us, 16 heads 64-65 (int8 78, blocks of 8 75) for the same keys,
// whose bytes take 50.5; in partitions of 512 keys 74-75 and 114.
template <typename T, typename C, int D>
int dispatch_geometry(const QuantDecodeParams& p, const CUtensorMap& km, const CUtensorMap& vm,
                      cudaStream_t s) {
  const bool wide = p.d.group > 8;
  if (p.d.block_size == 8)
    return wide ? launch_quant<T, C, D, 8, 16>(p, km, vm, s) : launch_quant<T, C, D, 8, 8>(p, km, vm, s);
  if (p.d.block_size == 32)
    return wide ? launch_quant<T, C, D, 32, 16>(p, km, vm, s) : launch_quant<T, C, D, 32, 8>(p, km, vm, s);
  return wide ? launch_quant<T, C, D, 16, 16>(p, km, vm, s) : launch_quant<T, C, D, 16, 8>(p, km, vm, s);
}

template <typename T>
int dispatch_code(const QuantDecodeParams& p, const CUtensorMap& km, const CUtensorMap& vm,
                  cudaStream_t s, int code, int head_dim) {
  if (code == PS_CODE_E4M3)
    return head_dim == 128 ? dispatch_geometry<T, CodeE4M3, 128>(p, km, vm, s)
                           : dispatch_geometry<T, CodeE4M3, 64>(p, km, vm, s);
  return head_dim == 128 ? dispatch_geometry<T, CodeInt8, 128>(p, km, vm, s)
                         : dispatch_geometry<T, CodeInt8, 64>(p, km, vm, s);
}

}  // namespace
}  // namespace ps

using namespace ps;

extern "C" int ps_paged_decode_quant(
    void* out, int64_t out_seq_stride, const void* query, int64_t query_seq_stride,
    const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
    int64_t num_blocks, const int32_t* block_tables, int64_t block_table_stride,
    const int32_t* ctx_lens, int num_seqs, const int32_t* seq_list, int num_listed, int num_q_heads,
    int num_kv_heads, int head_dim, int block_size, int max_blocks_per_seq, float scale,
    int split_tokens, int planned, void* workspace, int64_t workspace_bytes, int dtype, int code,
    int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_paged_decode_quant");
  const char* fn = "ps_paged_decode_quant";
  if (code != PS_CODE_E4M3 && code != PS_CODE_INT8)
    return fail(PS_ERR_UNSUPPORTED, "%s: code %d unsupported (e4m3 or int8)", fn, code);
  int part = 0, max_splits = 0, table_cap = 0;
  int st = validate_decode(fn, out, out_seq_stride, query, query_seq_stride, k_pool, v_pool,
                           num_blocks, block_tables, block_table_stride, ctx_lens, num_seqs,
                           num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                           split_tokens, dtype, &part, &max_splits, &table_cap);
  if (st != PS_OK || num_seqs == 0) return st;
  if (!k_scale || !v_scale || !aligned(k_scale, 16) || !aligned(v_scale, 16))
    return fail(PS_ERR_INVALID, "%s: k_scale/v_scale must be 16-byte aligned device pointers", fn);
  if (num_listed > num_seqs || (num_listed > 0 && !seq_list))
    return fail(PS_ERR_INVALID, "%s: num_listed %d needs a list of at most num_seqs %d entries", fn,
                num_listed, num_seqs);
  if (planned && num_listed >= 0)
    return fail(PS_ERR_INVALID, "%s: a plan covers all sequences; it cannot be combined with a list",
                fn);
  if (num_listed == 0) return PS_OK;
  QuantDecodeParams qp{};
  DecodeParams& p = qp.d;
  if (max_splits > 1) {
    st = set_split_workspace(fn, &p, num_seqs, num_q_heads, head_dim, block_size,
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
  p.num_launch = num_listed < 0 ? num_seqs : num_listed;
  p.planned = planned != 0;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.max_blocks = max_blocks_per_seq;
  p.block_size = block_size;
  p.part_tokens = part;
  p.max_splits = max_splits;
  p.table_cap = table_cap;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = device_error;
  p.seq_order = seq_list;
  qp.k_scale = k_scale;
  qp.v_scale = v_scale;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * num_kv_heads * block_size;
  CUtensorMap km, vm;
  const int box = block_size < kKeys ? block_size : kKeys;
  st = get_pool_tmap(k_pool, rows, head_dim, box, &km, 1);
  if (st != PS_OK) return st;
  st = get_pool_tmap(v_pool, rows, head_dim, box, &vm, 1);
  if (st != PS_OK) return st;
  cudaStream_t s = as_stream(stream);
  return dtype == PS_DTYPE_BF16 ? dispatch_code<__nv_bfloat16>(qp, km, vm, s, code, head_dim)
                                : dispatch_code<__half>(qp, km, vm, s, code, head_dim);
}
