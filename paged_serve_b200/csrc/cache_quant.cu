// Writing the 8-bit KV cache (optionally with RoPE on K) and reading it back.
//
// Both move bytes: the append reads 4 bytes and writes 2 for every (K, V) pair
// of values, the read back the other way round, plus 4 bytes of scale per row.
#include "capi_internal.h"
#include "common.cuh"
#include "quant.cuh"

namespace ps {
namespace {

struct AppendQuantParams {
  void* k_pool;
  void* v_pool;
  float* k_scale;
  float* v_scale;
  const void* key;
  const void* value;
  const int64_t* slots;
  const int64_t* positions;  // RoPE only
  const void* table;         // RoPE only: [table_positions][head_dim] (cos half | sin half)
  int64_t key_stride;
  int64_t value_stride;
  int64_t num_slots;
  int64_t table_positions;
  int num_kv_heads;
  int block_size;
  FastDiv div_heads;
  FastDiv div_block;
  int32_t* err;
};

// max |x| of the row's D/16 threads.
template <int kLanes>
__device__ __forceinline__ float row_max(float m) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// max |x| of eight values as two packed maxima (NaN when any is).
template <typename T>
__device__ __forceinline__ float max_abs8(const uint4& v);
template <>
__device__ __forceinline__ float max_abs8<__nv_bfloat16>(const uint4& v) {
  const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(w[0]), __habs2(w[1])),
                                       __hmax2_nan(__habs2(w[2]), __habs2(w[3])));
  return max_nan(__low2float(m), __high2float(m));
}
template <>
__device__ __forceinline__ float max_abs8<__half>(const uint4& v) {
  const __half2* w = reinterpret_cast<const __half2*>(&v);
  const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(w[0]), __habs2(w[1])),
                                __hmax2_nan(__habs2(w[2]), __habs2(w[3])));
  return max_nan(__low2float(m), __high2float(m));
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float2 (&x)[4]) {
  x[0] = unpack2<T>(v.x);
  x[1] = unpack2<T>(v.y);
  x[2] = unpack2<T>(v.z);
  x[3] = unpack2<T>(v.w);
}

// Quantises one thread's sixteen values of a row, m the largest of their |x|, and
// writes its codes (and, from the row's first thread, the scale).
template <typename C, int D>
__device__ __forceinline__ void quantise_row(float m, const float2 (&lo)[4], const float2 (&hi)[4],
                                             uint8_t* codes, float* scale_out, int c, bool store) {
  const float scale = row_scale<C>(row_max<D / 16>(m));
  if (!store) return;
  const float inv = __frcp_rn(scale);
  const float2 inv2 = make_float2(inv, inv);
  uint2 a, b;
  a.x = encode4<C>(__fmul2_rn(lo[0], inv2), __fmul2_rn(lo[1], inv2));
  a.y = encode4<C>(__fmul2_rn(lo[2], inv2), __fmul2_rn(lo[3], inv2));
  b.x = encode4<C>(__fmul2_rn(hi[0], inv2), __fmul2_rn(hi[1], inv2));
  b.y = encode4<C>(__fmul2_rn(hi[2], inv2), __fmul2_rn(hi[3], inv2));
  *reinterpret_cast<uint2*>(codes + c * 8) = a;
  *reinterpret_cast<uint2*>(codes + D / 2 + c * 8) = b;
  if (c == 0) *scale_out = scale;
}

// Row of the scale pool (and of the codes, times D) that `slot` names, for head h.
__device__ __forceinline__ int64_t pool_row(const AppendQuantParams& p, int64_t slot, int h) {
  const uint32_t blk = p.div_block.div(static_cast<uint32_t>(slot));
  const int off = static_cast<int>(static_cast<uint32_t>(slot) - blk * p.block_size);
  return (static_cast<int64_t>(blk) * p.num_kv_heads + h) * p.block_size + off;
}

// D/16 threads per (token, KV head) row; thread c owns elements [8c, 8c + 8) and
// [D/2 + 8c, D/2 + 8c + 8), the pairs that the rotation mixes, so RoPE needs no
// shuffles and the row's maximum three (D 128) or two (D 64). Without a rotation a
// thread takes its part of K and of V.
// 16,640 tokens of 8 heads, D 128, bf16 to e4m3: 17.9 us for 104 MB, 0.90 of
// the copy peak.
template <typename T, int D, typename C>
__global__ void __launch_bounds__(256)
    cache_append_quant_kernel(const AppendQuantParams p, uint32_t num_chunks) {
  constexpr int kThreadsPerRow = D / 16;
  pdl_trigger();
  pdl_wait();
  const uint32_t chunk = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t row = chunk / kThreadsPerRow;  // token * num_kv_heads + head
  const int c = static_cast<int>(chunk % kThreadsPerRow);
  // Rows never straddle num_chunks: a row's threads are all active or all past the end.
  bool store = chunk < num_chunks;
  uint4 k0 = {}, k1 = {}, v0 = {}, v1 = {};
  int64_t dst = 0;
  if (store) {
    const uint32_t t = p.div_heads.div(row);
    const int h = static_cast<int>(row - t * p.num_kv_heads);
    const int64_t slot = p.slots[t];
    const T* k = static_cast<const T*>(p.key) + t * p.key_stride + static_cast<int64_t>(h) * D + c * 8;
    const T* v = static_cast<const T*>(p.value) + t * p.value_stride + static_cast<int64_t>(h) * D + c * 8;
    k0 = __ldcs(reinterpret_cast<const uint4*>(k));
    k1 = __ldcs(reinterpret_cast<const uint4*>(k + D / 2));
    v0 = __ldcs(reinterpret_cast<const uint4*>(v));
    v1 = __ldcs(reinterpret_cast<const uint4*>(v + D / 2));
    store = slot >= 0 && slot < p.num_slots;  // negative: a padding token
    if (slot >= p.num_slots) set_device_error(p.err, PS_DEVERR_SLOT);
    if (store) dst = pool_row(p, slot, h);
  }
  float2 lo[4], hi[4];
  unpack8<T>(k0, lo);
  unpack8<T>(k1, hi);
  quantise_row<C, D>(max_nan(max_abs8<T>(k0), max_abs8<T>(k1)), lo, hi,
                     static_cast<uint8_t*>(p.k_pool) + dst * D, p.k_scale + dst, c, store);
  unpack8<T>(v0, lo);
  unpack8<T>(v1, hi);
  quantise_row<C, D>(max_nan(max_abs8<T>(v0), max_abs8<T>(v1)), lo, hi,
                     static_cast<uint8_t*>(p.v_pool) + dst * D, p.v_scale + dst, c, store);
}

// With RoPE on K: the CTAs of blockIdx.y 0 take the K rows, those of 1 the V rows. The
// rotation's chain of loads (position, then its cos and sin) wants more warps than the
// registers of both rows at once leave: 23.2 us against 24.6 in one thread (the sizes
// above; without a rotation the split costs 1.5 us). Position, slot, cos and sin are fetched
// and unpacked once per head: 70% of the issue slots, of which the rows' own work is a part.
// K is rotated in fp32: the products of two 16-bit values are exact there, so
// each rotated element is rounded once before it is quantised.
template <typename T, int D, typename C>
__global__ void __launch_bounds__(256)
    cache_append_rope_quant_kernel(const AppendQuantParams p, uint32_t num_chunks) {
  constexpr int kThreadsPerRow = D / 16;
  pdl_trigger();
  pdl_wait();
  const bool is_v = blockIdx.y != 0;
  const uint32_t chunk = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t row = chunk / kThreadsPerRow;  // token * num_kv_heads + head
  const int c = static_cast<int>(chunk % kThreadsPerRow);
  bool store = chunk < num_chunks;
  uint4 x0 = {}, x1 = {}, cv = {}, sv = {};
  int64_t dst = 0;
  if (store) {
    const uint32_t t = p.div_heads.div(row);
    const int h = static_cast<int>(row - t * p.num_kv_heads);
    const int64_t slot = p.slots[t];
    const int64_t pos = p.positions[t];
    const T* x = (is_v ? static_cast<const T*>(p.value) + t * p.value_stride
                       : static_cast<const T*>(p.key) + t * p.key_stride) +
                 static_cast<int64_t>(h) * D + c * 8;
    x0 = __ldcs(reinterpret_cast<const uint4*>(x));
    x1 = __ldcs(reinterpret_cast<const uint4*>(x + D / 2));
    store = slot >= 0 && slot < p.num_slots;  // negative: a padding token
    if (slot >= p.num_slots) {
      set_device_error(p.err, PS_DEVERR_SLOT);
    } else if (store && (pos < 0 || pos >= p.table_positions)) {
      set_device_error(p.err, PS_DEVERR_POSITION);
      store = false;  // neither K nor V is written
    }
    if (store) {
      dst = pool_row(p, slot, h);
      if (!is_v) {
        const T* cs = static_cast<const T*>(p.table) + pos * D + c * 8;
        cv = *reinterpret_cast<const uint4*>(cs);
        sv = *reinterpret_cast<const uint4*>(cs + D / 2);
      }
    }
  }
  float2 lo[4], hi[4];
  unpack8<T>(x0, lo);
  unpack8<T>(x1, hi);
  float m = 0.f;
  if (is_v) {
    m = max_nan(max_abs8<T>(x0), max_abs8<T>(x1));
  } else {
    float2 co[4], si[4];
    unpack8<T>(cv, co);
    unpack8<T>(sv, si);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = lo[i], b = hi[i];
      const float2 bs = __fmul2_rn(b, si[i]);  // exact, so the sums below round once
      lo[i] = __ffma2_rn(a, co[i], make_float2(-bs.x, -bs.y));
      hi[i] = __ffma2_rn(b, co[i], __fmul2_rn(a, si[i]));
      m = max3_abs_nan(m, lo[i].x, lo[i].y);
      m = max3_abs_nan(m, hi[i].x, hi[i].y);
    }
  }
  quantise_row<C, D>(m, lo, hi, static_cast<uint8_t*>(is_v ? p.v_pool : p.k_pool) + dst * D,
                     (is_v ? p.v_scale : p.k_scale) + dst, c, store);
}

template <typename T, int D, typename C, bool kRope>
cudaError_t launch_append(const AppendQuantParams& p, int64_t num_tokens, cudaStream_t s) {
  const uint32_t chunks = static_cast<uint32_t>(num_tokens * p.num_kv_heads * (D / 16));
  const unsigned grid = (chunks + 255) / 256;
  if constexpr (kRope)
    return launch_pdl(cache_append_rope_quant_kernel<T, D, C>, dim3(grid, 2), dim3(256), 0, s, p,
                      chunks);
  else
    return launch_pdl(cache_append_quant_kernel<T, D, C>, dim3(grid), dim3(256), 0, s, p, chunks);
}

template <typename T, bool kRope>
cudaError_t dispatch_append(const AppendQuantParams& p, int64_t n, int head_dim, int code,
                            cudaStream_t s) {
  if (code == PS_CODE_E4M3)
    return head_dim == 128 ? launch_append<T, 128, CodeE4M3, kRope>(p, n, s)
                           : launch_append<T, 64, CodeE4M3, kRope>(p, n, s);
  return head_dim == 128 ? launch_append<T, 128, CodeInt8, kRope>(p, n, s)
                         : launch_append<T, 64, CodeInt8, kRope>(p, n, s);
}

int append_quant_entry(const char* fn, bool rope, void* k_pool, void* v_pool, float* k_scale,
                       float* v_scale, const void* key, const void* value, const int64_t* slots,
                       const int64_t* positions, int64_t num_tokens, int64_t key_stride,
                       int64_t value_stride, int num_kv_heads, int head_dim, int block_size,
                       int64_t num_blocks, const void* table, int64_t table_positions,
                       int rope_dim, int dtype, int code, int32_t* err, void* stream) {
  if (dtype != PS_DTYPE_BF16 && dtype != PS_DTYPE_F16)
    return fail(PS_ERR_UNSUPPORTED, "%s: dtype %d unsupported (bf16/f16 only)", fn, dtype);
  if (code != PS_CODE_E4M3 && code != PS_CODE_INT8)
    return fail(PS_ERR_UNSUPPORTED, "%s: code %d unsupported (e4m3 or int8)", fn, code);
  if (head_dim != 64 && head_dim != 128)
    return fail(PS_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", fn, head_dim);
  if (num_tokens < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks <= 0)
    return fail(PS_ERR_INVALID, "%s: bad sizes (tokens %lld, kv heads %d, block %d, blocks %lld)",
                fn, (long long)num_tokens, num_kv_heads, block_size, (long long)num_blocks);
  if (rope && rope_dim != head_dim)
    return fail(PS_ERR_UNSUPPORTED, "%s: rope_dim %d != head_dim %d", fn, rope_dim, head_dim);
  if (num_tokens == 0) return PS_OK;
  if (!k_pool || !v_pool || !k_scale || !v_scale || !key || !value || !slots)
    return fail(PS_ERR_INVALID, "%s: null pointer argument", fn);
  if (key_stride < (int64_t)num_kv_heads * head_dim || value_stride < (int64_t)num_kv_heads * head_dim)
    return fail(PS_ERR_INVALID, "%s: token stride smaller than num_kv_heads*head_dim", fn);
  if ((key_stride % 8) || (value_stride % 8) || !aligned(key, 16) || !aligned(value, 16) ||
      !aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(k_scale, 16) ||
      !aligned(v_scale, 16))
    return fail(PS_ERR_INVALID,
                "%s: key/value/pools/scales must be 16-byte aligned with strides %% 8 == 0", fn);
  if (rope && (!positions || !table || table_positions <= 0))
    return fail(PS_ERR_INVALID, "%s: positions/table missing", fn);
  if (rope && !aligned(table, 16))
    return fail(PS_ERR_INVALID, "%s: cos_sin_table must be 16-byte aligned", fn);
  if (num_tokens > (int64_t(1) << 31) / num_kv_heads / (head_dim / 16) - 1)
    return fail(PS_ERR_INVALID, "%s: too many tokens for one launch", fn);
  if (num_blocks >= (int64_t(1) << 31) / block_size)
    return fail(PS_ERR_INVALID, "%s: pool of %lld blocks of %d slots exceeds 2^31", fn,
                (long long)num_blocks, block_size);
  AppendQuantParams p{};
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.key = key;
  p.value = value;
  p.slots = slots;
  p.positions = positions;
  p.table = table;
  p.key_stride = key_stride;
  p.value_stride = value_stride;
  p.num_slots = num_blocks * block_size;
  p.table_positions = table_positions;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.div_heads = FastDiv(static_cast<uint32_t>(num_kv_heads));
  p.div_block = FastDiv(static_cast<uint32_t>(block_size));
  p.err = err;
  cudaStream_t s = as_stream(stream);
  cudaError_t e;
  if (dtype == PS_DTYPE_BF16)
    e = rope ? dispatch_append<__nv_bfloat16, true>(p, num_tokens, head_dim, code, s)
             : dispatch_append<__nv_bfloat16, false>(p, num_tokens, head_dim, code, s);
  else
    e = rope ? dispatch_append<__half, true>(p, num_tokens, head_dim, code, s)
             : dispatch_append<__half, false>(p, num_tokens, head_dim, code, s);
  if (e != cudaSuccess) return fail(PS_ERR_CUDA, "%s: launch failed: %s", fn, cudaGetErrorString(e));
  return check_launch(fn);
}

// ------------------------------------------------------------- read back
struct ReadQuantParams {
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  const float* k_scale;
  const float* v_scale;
  void* k_out;
  void* v_out;
  const int32_t* tables;
  const int32_t* out_tables;
  int64_t table_stride;
  int64_t out_table_stride;
  const int32_t* ctx_lens;
  int64_t num_blocks;
  int64_t num_out_blocks;
  int max_blocks;
  int block_size;
  int vecs;  // 8-code vectors of one block: num_kv_heads * block_size * head_dim / 8
  FastDiv div_block;
  int32_t* err;
};

// One CTA per (block of a sequence): a block's codes are contiguous, and so are
// its values in the output block. A thread turns 8 codes of one row into 16 bytes
// (16 codes into two 16-byte stores leave half of each sector to the second store), four
// such loads in flight; rows past the sequence's last token are written as zeros, so what
// a freed block held before (NaN among it) never reaches a reader of whole tiles.
template <typename T, int D, typename C>
__global__ void __launch_bounds__(256) cache_read_quant_kernel(const ReadQuantParams p) {
  pdl_trigger();
  pdl_wait();
  const int j = blockIdx.x;
  const int b = blockIdx.y;
  const int ctx = p.ctx_lens[b];
  if (ctx > p.max_blocks * p.block_size) {
    if (j == 0 && threadIdx.x == 0) set_device_error(p.err, PS_DEVERR_LENGTH);
    return;
  }
  const int left = ctx - j * p.block_size;  // tokens of the sequence from this block on
  if (left <= 0) return;
  const int32_t src = p.tables[b * p.table_stride + j];
  const int32_t dst = p.out_tables[b * p.out_table_stride + j];
  if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.num_out_blocks) {
    if (threadIdx.x == 0) set_device_error(p.err, PS_DEVERR_BLOCK_ID);
    return;
  }
  constexpr int kUnroll = 4;
  const int64_t rows = static_cast<int64_t>(p.vecs) * 8 / D;
#pragma unroll
  for (int is_v = 0; is_v < 2; ++is_v) {
    const uint2* codes = reinterpret_cast<const uint2*>(is_v ? p.v_pool : p.k_pool) +
                         static_cast<int64_t>(src) * p.vecs;
    const float* scales = (is_v ? p.v_scale : p.k_scale) + src * rows;
    uint4* out = reinterpret_cast<uint4*>(is_v ? p.v_out : p.k_out) +
                 static_cast<int64_t>(dst) * p.vecs;
    for (int i0 = threadIdx.x; i0 < p.vecs; i0 += kUnroll * 256) {
      uint2 c[kUnroll];
      float s[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = i0 + u * 256;
        c[u] = make_uint2(0u, 0u);
        s[u] = 0.f;
        if (i < p.vecs) {
          const uint32_t row = static_cast<uint32_t>(i) / (D / 8);  // head * block_size + offset
          const int off = static_cast<int>(row - p.div_block.div(row) * p.block_size);
          if (off < left) {
            c[u] = __ldcs(codes + i);
            s[u] = scales[row];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = i0 + u * 256;
        uint32_t h[4];
        decode4<C>(c[u].x, h[0], h[1]);
        decode4<C>(c[u].y, h[2], h[3]);
        uint32_t o[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          o[x] = pack2<T>(__fmul2_rn(unpack2<__half>(h[x]), make_float2(s[u], s[u])));
        if (i < p.vecs) out[i] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
}

template <typename T, int D>
cudaError_t launch_read(const ReadQuantParams& p, int code, dim3 grid, cudaStream_t s) {
  return code == PS_CODE_E4M3
             ? launch_pdl(cache_read_quant_kernel<T, D, CodeE4M3>, grid, dim3(256), 0, s, p)
             : launch_pdl(cache_read_quant_kernel<T, D, CodeInt8>, grid, dim3(256), 0, s, p);
}

}  // namespace
}  // namespace ps

using namespace ps;

extern "C" int ps_cache_append_quant(void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                                     const void* key, const void* value,
                                     const int64_t* slot_mapping, int64_t num_tokens,
                                     int64_t key_token_stride, int64_t value_token_stride,
                                     int num_kv_heads, int head_dim, int block_size,
                                     int64_t num_blocks, int dtype, int code,
                                     int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_cache_append_quant");
  return append_quant_entry("ps_cache_append_quant", false, k_pool, v_pool, k_scale, v_scale, key,
                            value, slot_mapping, nullptr, num_tokens, key_token_stride,
                            value_token_stride, num_kv_heads, head_dim, block_size, num_blocks,
                            nullptr, 0, 0, dtype, code, device_error, stream);
}

extern "C" int ps_cache_append_rope_quant(
    void* k_pool, void* v_pool, float* k_scale, float* v_scale, const void* key, const void* value,
    const int64_t* slot_mapping, const int64_t* positions, int64_t num_tokens,
    int64_t key_token_stride, int64_t value_token_stride, int num_kv_heads, int head_dim,
    int block_size, int64_t num_blocks, const void* cos_sin_table, int64_t table_positions,
    int rope_dim, int dtype, int code, int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_cache_append_rope_quant");
  return append_quant_entry("ps_cache_append_rope_quant", true, k_pool, v_pool, k_scale, v_scale,
                            key, value, slot_mapping, positions, num_tokens, key_token_stride,
                            value_token_stride, num_kv_heads, head_dim, block_size, num_blocks,
                            cos_sin_table, table_positions, rope_dim, dtype, code, device_error,
                            stream);
}

extern "C" int ps_cache_read_quant(const void* k_pool, const void* v_pool, const float* k_scale,
                                   const float* v_scale, int64_t num_blocks, void* k_out,
                                   void* v_out, int64_t num_out_blocks,
                                   const int32_t* block_tables, int64_t block_table_stride,
                                   const int32_t* out_tables, int64_t out_table_stride,
                                   const int32_t* ctx_lens, int num_seqs, int num_kv_heads,
                                   int head_dim, int block_size, int max_blocks_per_seq, int dtype,
                                   int code, int32_t* device_error, void* stream) {
  ps::NvtxRange nvtx_range("ps_cache_read_quant");
  const char* fn = "ps_cache_read_quant";
  if (dtype != PS_DTYPE_BF16 && dtype != PS_DTYPE_F16)
    return fail(PS_ERR_UNSUPPORTED, "%s: dtype %d unsupported (bf16/f16 only)", fn, dtype);
  if (code != PS_CODE_E4M3 && code != PS_CODE_INT8)
    return fail(PS_ERR_UNSUPPORTED, "%s: code %d unsupported (e4m3 or int8)", fn, code);
  if (head_dim != 64 && head_dim != 128)
    return fail(PS_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", fn, head_dim);
  if (num_seqs < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks <= 0 ||
      num_out_blocks <= 0 || max_blocks_per_seq <= 0)
    return fail(PS_ERR_INVALID, "%s: bad sizes", fn);
  if (num_seqs == 0) return PS_OK;
  if (!k_pool || !v_pool || !k_scale || !v_scale || !k_out || !v_out || !block_tables ||
      !out_tables || !ctx_lens)
    return fail(PS_ERR_INVALID, "%s: null pointer argument", fn);
  if (block_table_stride < max_blocks_per_seq || out_table_stride < max_blocks_per_seq)
    return fail(PS_ERR_INVALID, "%s: table stride < max_blocks_per_seq", fn);
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(k_out, 16) || !aligned(v_out, 16) ||
      !aligned(k_scale, 16) || !aligned(v_scale, 16))
    return fail(PS_ERR_INVALID, "%s: pools and scales must be 16-byte aligned", fn);
  if (num_seqs > 65535) return fail(PS_ERR_INVALID, "%s: too many sequences for one launch", fn);
  if (static_cast<int64_t>(max_blocks_per_seq) * block_size >= (int64_t(1) << 31) ||
      static_cast<int64_t>(num_kv_heads) * block_size * (head_dim / 16) >= (int64_t(1) << 30))
    return fail(PS_ERR_INVALID, "%s: sequence or block too long", fn);
  ReadQuantParams p{};
  p.k_pool = static_cast<const uint8_t*>(k_pool);
  p.v_pool = static_cast<const uint8_t*>(v_pool);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.k_out = k_out;
  p.v_out = v_out;
  p.tables = block_tables;
  p.out_tables = out_tables;
  p.table_stride = block_table_stride;
  p.out_table_stride = out_table_stride;
  p.ctx_lens = ctx_lens;
  p.num_blocks = num_blocks;
  p.num_out_blocks = num_out_blocks;
  p.max_blocks = max_blocks_per_seq;
  p.block_size = block_size;
  p.vecs = num_kv_heads * block_size * (head_dim / 8);
  p.div_block = FastDiv(static_cast<uint32_t>(block_size));
  p.err = device_error;
  const dim3 grid(static_cast<unsigned>(max_blocks_per_seq), static_cast<unsigned>(num_seqs));
  cudaStream_t s = as_stream(stream);
  cudaError_t e;
  if (dtype == PS_DTYPE_BF16)
    e = head_dim == 128 ? launch_read<__nv_bfloat16, 128>(p, code, grid, s)
                        : launch_read<__nv_bfloat16, 64>(p, code, grid, s);
  else
    e = head_dim == 128 ? launch_read<__half, 128>(p, code, grid, s)
                        : launch_read<__half, 64>(p, code, grid, s);
  if (e != cudaSuccess) return fail(PS_ERR_CUDA, "%s: launch failed: %s", fn, cudaGetErrorString(e));
  return check_launch(fn);
}
