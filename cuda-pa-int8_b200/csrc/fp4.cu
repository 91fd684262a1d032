// Rows into and out of the 4-bit K/V cache (format and layout: fp4.cuh).
//
// Both directions are streams: a thread takes one 16-value block of one row (token, kv head, K
// or V), so a block's maximum needs no other lane, eight neighbouring threads cover a row, and a
// warp's loads and stores of values are contiguous. Every byte of the cache belongs to one
// token, so rows are written independently: a decode step's appends, a prompt through slots
// and rows in any order all take the same path.

#include "fp4.cuh"
#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_rows.cuh"

namespace pa {
namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerRow = 8;  // 128 head_dim values in blocks of 16

// Sixteen consecutive values as fp32 (p aligned to 16 bytes).
__device__ __forceinline__ void load16(const __half* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      x[8 * i + 2 * e] = f.x;
      x[8 * i + 2 * e + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void load16(const __nv_bfloat16* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[8 * i + 2 * e] = __uint_as_float(w[e] << 16);
      x[8 * i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
    x[4 * i] = f.x;
    x[4 * i + 1] = f.y;
    x[4 * i + 2] = f.z;
    x[4 * i + 3] = f.w;
  }
}

// Block b (16 values x) of token `off` of page row `page`: eight code bytes and the scale byte.
template <typename T>
__device__ __forceinline__ void put_block(const float (&x)[16], uint8_t* cache, bool is_v,
                                          size_t page, int off, int bs, int b) {
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 16; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  const uint32_t sb = fp4::scale_byte(m);
  const float s = fp4::scale_value(sb), inv = fp4::scale_inverse(sb);
  constexpr bool kWide = sizeof(T) == 4;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    w[e >> 2] |= fp4::code_pair(fp4::code_y<kWide>(x[2 * e], s, inv),
                                fp4::code_y<kWide>(x[2 * e + 1], s, inv))
                 << (8 * (e & 3));
  uint8_t* grp = cache + fp4::group_offset(page, off, bs);
  const int t = off % fp4::kGroupTokens;
  *reinterpret_cast<uint2*>(grp + t * fp4::kCodeRow + 8 * b) = make_uint2(w[0], w[1]);
  grp[fp4::scale_offset(is_v, t, b)] = (uint8_t)sb;
}

// Rows of a slot-mapped write; rows of one token are contiguous (kv_heads x 128 values).
template <typename T>
__global__ void __launch_bounds__(kThreads) write_fp4_kernel(
    const T* __restrict__ k, const T* __restrict__ v, long long token_stride,
    const int* __restrict__ slot_mapping, int N, int KVH, uint8_t* __restrict__ k_cache,
    uint8_t* __restrict__ v_cache, int NB, int bs, int* status) {
  const bool is_v = blockIdx.y != 0;
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = i >> 3;
  const int b = (int)(i & 7);
  if (row >= (long long)N * KVH) return;
  const int n = (int)(row / KVH);
  const int kvh = (int)(row - (long long)n * KVH);
  const int slot = __ldg(slot_mapping + n);
  if (slot < 0) return;  // padding token
  const int blk = slot / bs;
  if (blk >= NB) {
    flag_error(status, PA_ERR_SLOT);
    return;
  }
  float x[16];
  load16((is_v ? v : k) + (size_t)n * token_stride + (size_t)kvh * 128 + 16 * b, x);
  put_block<T>(x, is_v ? v_cache : k_cache, is_v, (size_t)blk * KVH + kvh, slot - blk * bs, bs,
               b);
}

// The decode step's new token: position context_lens[b] - 1 of sequence b, through its table.
template <typename T>
__global__ void __launch_bounds__(kThreads) step_fp4_kernel(
    const T* __restrict__ k, const T* __restrict__ v, long long token_stride,
    const int* __restrict__ block_table, const int* __restrict__ context_lens, int max_blocks,
    int B, int KVH, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, int NB, int bs,
    int* status) {
  const bool is_v = blockIdx.y != 0;
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = i >> 3;
  const int b = (int)(i & 7);
  if (row >= (long long)B * KVH) return;
  const int n = (int)(row / KVH);
  const int kvh = (int)(row - (long long)n * KVH);
  const int ctx = __ldg(context_lens + n);
  if (ctx < 1 || ctx > max_blocks * bs) return;  // the decode flags the length
  const int pos = ctx - 1;
  const int blk = __ldg(block_table + (size_t)n * max_blocks + pos / bs);
  if (blk < 0 || blk >= NB) {
    flag_error(status, PA_ERR_BLOCK_ID);
    return;
  }
  float x[16];
  load16((is_v ? v : k) + (size_t)n * token_stride + (size_t)kvh * 128 + 16 * b, x);
  put_block<T>(x, is_v ? v_cache : k_cache, is_v, (size_t)blk * KVH + kvh, pos % bs, bs, b);
}

// Sixteen held values as fp16 pairs, stored as T (exact: every held value is an fp16 and a bf16
// number; a NaN scale gives NaN).
__device__ __forceinline__ void store16(const uint32_t (&h)[8], __half* p) {
  reinterpret_cast<uint4*>(p)[0] = make_uint4(h[0], h[1], h[2], h[3]);
  reinterpret_cast<uint4*>(p)[1] = make_uint4(h[4], h[5], h[6], h[7]);
}
__device__ __forceinline__ void store16(const uint32_t (&h)[8], __nv_bfloat16* p) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const __nv_bfloat162 o = __floats2bfloat162_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const uint32_t*>(&o);
  }
  reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
__device__ __forceinline__ void store16(const uint32_t (&h)[8], float* p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[2 * i]));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h[2 * i + 1]));
    reinterpret_cast<float4*>(p)[i] = make_float4(a.x, a.y, b.x, b.y);
  }
}

// Rows read back: out rows of tokens with a negative or out-of-range slot are left as they are.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_fp4_kernel(
    T* __restrict__ k_out, T* __restrict__ v_out, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const int* __restrict__ slot_mapping, int N, int KVH,
    int NB, int bs, int* status) {
  const bool is_v = blockIdx.y != 0;
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long row = i >> 3;
  const int b = (int)(i & 7);
  if (row >= (long long)N * KVH) return;
  const int n = (int)(row / KVH);
  const int kvh = (int)(row - (long long)n * KVH);
  const int slot = __ldg(slot_mapping + n);
  if (slot < 0) return;
  const int blk = slot / bs;
  if (blk >= NB) {
    flag_error(status, PA_ERR_SLOT);
    return;
  }
  const int off = slot - blk * bs, t = off % fp4::kGroupTokens;
  const uint8_t* grp = (is_v ? v_cache : k_cache) +
                       fp4::group_offset((size_t)blk * KVH + kvh, off, bs);
  const uint2 c = *reinterpret_cast<const uint2*>(grp + t * fp4::kCodeRow + 8 * b);
  const uint32_t s = (uint32_t)grp[fp4::scale_offset(is_v, t, b)] * 0x00800080u;  // twice << 7
  uint32_t h[8];
  fp4::codes_to_f16x2(c.x, h[0], h[1], h[2], h[3]);
  fp4::codes_to_f16x2(c.y, h[4], h[5], h[6], h[7]);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = fp4::hmul2(h[e], s);
  store16(h, (is_v ? v_out : k_out) + (size_t)row * 128 + 16 * b);
}

// Threads of N x KVH rows, eight each; 0 when there are none, -1 when a grid cannot hold them.
long long grid_of(long long rows) {
  const long long g = (rows * kBlocksPerRow + kThreads - 1) / kThreads;
  return g > 0x7fffffffLL ? -1 : g;
}

template <typename T>
cudaError_t write_t(const void* k, const void* v, long long ts, const int* slots, int N, int KVH,
                    void* kc, void* vc, int NB, int bs, int* status, cudaStream_t st) {
  const long long g = grid_of((long long)N * KVH);
  if (g < 0) return cudaErrorInvalidValue;
  if (g == 0) return cudaSuccess;
  write_fp4_kernel<T><<<dim3((unsigned)g, 2), kThreads, 0, st>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), ts, slots, N, KVH,
      static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), NB, bs, status);
  return cudaGetLastError();
}

template <typename T>
cudaError_t step_t(const void* k, const void* v, long long ts, const int* bt, const int* cl,
                   int max_blocks, int B, int KVH, void* kc, void* vc, int NB, int bs,
                   int* status, cudaStream_t st) {
  const long long g = grid_of((long long)B * KVH);
  if (g < 0) return cudaErrorInvalidValue;
  if (g == 0) return cudaSuccess;
  step_fp4_kernel<T><<<dim3((unsigned)g, 2), kThreads, 0, st>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), ts, bt, cl, max_blocks, B, KVH,
      static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), NB, bs, status);
  return cudaGetLastError();
}

template <typename T>
cudaError_t read_t(void* k, void* v, const void* kc, const void* vc, const int* slots, int N,
                   int KVH, int NB, int bs, int* status, cudaStream_t st) {
  const long long g = grid_of((long long)N * KVH);
  if (g < 0) return cudaErrorInvalidValue;
  if (g == 0) return cudaSuccess;
  read_fp4_kernel<T><<<dim3((unsigned)g, 2), kThreads, 0, st>>>(
      static_cast<T*>(k), static_cast<T*>(v), static_cast<const uint8_t*>(kc),
      static_cast<const uint8_t*>(vc), slots, N, KVH, NB, bs, status);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_write_fp4(int in_dtype, const void* k, const void* v, long long ts,
                             const int* slots, int N, int KVH, void* kc, void* vc, int NB, int bs,
                             int* status, cudaStream_t st) {
  switch (in_dtype) {
    case PA_DTYPE_F16: return write_t<__half>(k, v, ts, slots, N, KVH, kc, vc, NB, bs, status, st);
    case PA_DTYPE_BF16:
      return write_t<__nv_bfloat16>(k, v, ts, slots, N, KVH, kc, vc, NB, bs, status, st);
    case PA_DTYPE_F32: return write_t<float>(k, v, ts, slots, N, KVH, kc, vc, NB, bs, status, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_step_fp4(int in_dtype, const void* k, const void* v, long long ts,
                            const int* bt, const int* cl, int max_blocks, int B, int KVH,
                            void* kc, void* vc, int NB, int bs, int* status, cudaStream_t st) {
  switch (in_dtype) {
    case PA_DTYPE_F16:
      return step_t<__half>(k, v, ts, bt, cl, max_blocks, B, KVH, kc, vc, NB, bs, status, st);
    case PA_DTYPE_BF16:
      return step_t<__nv_bfloat16>(k, v, ts, bt, cl, max_blocks, B, KVH, kc, vc, NB, bs, status,
                                   st);
    case PA_DTYPE_F32:
      return step_t<float>(k, v, ts, bt, cl, max_blocks, B, KVH, kc, vc, NB, bs, status, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_read_fp4(int out_dtype, void* k, void* v, const void* kc, const void* vc,
                            const int* slots, int N, int KVH, int NB, int bs, int* status,
                            cudaStream_t st) {
  switch (out_dtype) {
    case PA_DTYPE_F16: return read_t<__half>(k, v, kc, vc, slots, N, KVH, NB, bs, status, st);
    case PA_DTYPE_BF16:
      return read_t<__nv_bfloat16>(k, v, kc, vc, slots, N, KVH, NB, bs, status, st);
    case PA_DTYPE_F32: return read_t<float>(k, v, kc, vc, slots, N, KVH, NB, bs, status, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace pa
