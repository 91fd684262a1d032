// Rows into and out of the 4-bit K/V cache (format and layout: fp4.cuh).
//
// Both directions are streams of rows (token, kv head, K or V), bound by memory once their
// instructions per row are few: the kv head and K or V come from the block index (no division),
// the write gives a thread a whole 16-value block (its maximum needs no other lane), the read
// eight values (one 16-byte store a thread, contiguous over the warp), and each thread takes
// several tokens at once so that their loads overlap. Every byte of the cache belongs to one token,
// so rows are written independently: a decode step's appends, a prompt through slots and rows in
// any order all take the same path.

#include "fp4.cuh"
#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_rows.cuh"

namespace pa {
namespace {

constexpr int kThreads = 256;
constexpr int kWriteRow = 8;   // threads of a row in the write: 128 values in blocks of 16
constexpr int kReadRow = 16;   // in the read: eight values each
// Tokens a thread takes. 1.05 M rows of K and of V: write 125 us with one, 111 with two or four;
// read 157 with two, 143 with four, 164 with eight.
constexpr int kWriteTokens = 2;
constexpr int kReadTokens = 4;

// Where the groups of a cache are. Group indices fit 32 bits: 2^32 groups would be 4.9 TB.
struct Cache {
  int NB, KVH;
  int shift;  // log2 of the block size (16 .. 128)
};
// Group index of `slot` and kv head kvh; the token of the group in t.
__device__ __forceinline__ uint32_t group_of(const Cache& c, int blk, int slot, int kvh, int& t) {
  t = slot & (fp4::kGroupTokens - 1);
  const uint32_t page = (uint32_t)blk * (uint32_t)c.KVH + (uint32_t)kvh;
  return (page << (c.shift - 4)) | (((uint32_t)slot & ((1u << c.shift) - 1u)) >> 4);
}

// Sixteen consecutive values (p aligned to 16 bytes) as loaded: 16-bit values packed in pairs.
template <typename T> struct Block { uint32_t w[8]; };
template <> struct Block<float> { uint32_t w[16]; };

template <typename T>
__device__ __forceinline__ void load_block(const T* p, Block<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {  // 32 or 64 bytes
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
    r.w[4 * i] = u.x;
    r.w[4 * i + 1] = u.y;
    r.w[4 * i + 2] = u.z;
    r.w[4 * i + 3] = u.w;
  }
}
// Bit pattern of the largest magnitude as fp32. Bit patterns without the sign order as the
// magnitudes do, NaN above infinity, so the 16-bit types compare two at a time as integers.
__device__ __forceinline__ uint32_t max_bits(const Block<float>& r) {
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 16; ++e) m = max(m, r.w[e] & 0x7fffffffu);
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t max_pair(const Block<T>& r) {
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = __vmaxu2(m, r.w[e] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}
__device__ __forceinline__ uint32_t max_bits(const Block<__half>& r) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max_pair(r))));
}
__device__ __forceinline__ uint32_t max_bits(const Block<__nv_bfloat16>& r) {
  return max_pair(r) << 16;
}
// Values 2e and 2e + 1.
__device__ __forceinline__ float2 pair_of(const Block<float>& r, int e) {
  return make_float2(__uint_as_float(r.w[2 * e]), __uint_as_float(r.w[2 * e + 1]));
}
__device__ __forceinline__ float2 pair_of(const Block<__half>& r, int e) {
  return __half22float2(*reinterpret_cast<const __half2*>(&r.w[e]));
}
__device__ __forceinline__ float2 pair_of(const Block<__nv_bfloat16>& r, int e) {
  return make_float2(__uint_as_float(r.w[e] << 16), __uint_as_float(r.w[e] & 0xffff0000u));
}

// Block b of token t of a group: eight code bytes and the scale byte.
template <typename T>
__device__ __forceinline__ void put_block(const Block<T>& r, uint8_t* grp, bool is_v, int t,
                                          int b) {
  constexpr bool kWide = sizeof(T) == 4;
  const uint32_t sb = fp4::scale_byte<kWide>(max_bits(r));
  const float s = fp4::scale_value(sb), inv = fp4::scale_inverse<kWide>(sb);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 v = pair_of(r, 4 * h + e);
      if constexpr (kWide) {
        v = make_float2(fp4::code_y<true>(v.x, s, inv), fp4::code_y<true>(v.y, s, inv));
      } else {  // fp4::code_y<false>, two values at a time
        v = add2(fma2(v, make_float2(inv, inv), make_float2(96.f, 96.f)),
                 make_float2(-96.f, -96.f));
      }
      y[2 * e] = v.x;
      y[2 * e + 1] = v.y;
    }
    w[h] = fp4::code_word(y);
  }
  *reinterpret_cast<uint2*>(grp + t * fp4::kCodeRow + 8 * b) = make_uint2(w[0], w[1]);
  grp[fp4::scale_offset(is_v, t, b)] = (uint8_t)sb;
}

// Rows of a slot-mapped write; rows of one token are contiguous (kv_heads x 128 values). Block
// row y of the grid: kv head y / 2, K (even) or V.
template <typename T>
__global__ void __launch_bounds__(kThreads) write_fp4_kernel(
    const T* __restrict__ k, const T* __restrict__ v, long long token_stride,
    const int* __restrict__ slot_mapping, int N, uint8_t* __restrict__ k_cache,
    uint8_t* __restrict__ v_cache, const Cache c, int* status) {
  constexpr int kTokens = kThreads / kWriteRow;  // tokens of a CTA's round
  const bool is_v = (blockIdx.y & 1) != 0;
  const int kvh = blockIdx.y >> 1;
  const int b = threadIdx.x % kWriteRow;
  const unsigned n0 = blockIdx.x * (unsigned)(kTokens * kWriteTokens) + threadIdx.x / kWriteRow;
  const T* src = (is_v ? v : k) + kvh * 128 + 16 * b;
  uint8_t* cache = is_v ? v_cache : k_cache;
  int slot[kWriteTokens];
#pragma unroll
  for (int i = 0; i < kWriteTokens; ++i) {
    const unsigned n = n0 + i * kTokens;
    slot[i] = n < (unsigned)N ? __ldg(slot_mapping + n) : -1;  // negative: padding token
  }
  Block<T> r[kWriteTokens];
#pragma unroll
  for (int i = 0; i < kWriteTokens; ++i)
    if (slot[i] >= 0) load_block(src + (n0 + i * kTokens) * token_stride, r[i]);
#pragma unroll
  for (int i = 0; i < kWriteTokens; ++i) {
    if (slot[i] < 0) continue;
    const int blk = slot[i] >> c.shift;
    if (blk >= c.NB) {
      flag_error(status, PA_ERR_SLOT);
      continue;
    }
    int t;
    const uint32_t g = group_of(c, blk, slot[i], kvh, t);
    put_block<T>(r[i], cache + (size_t)g * fp4::kGroupBytes, is_v, t, b);
  }
}

// The decode step's new token: position context_lens[b] - 1 of sequence b, through its table.
template <typename T>
__global__ void __launch_bounds__(kThreads) step_fp4_kernel(
    const T* __restrict__ k, const T* __restrict__ v, long long token_stride,
    const int* __restrict__ block_table, const int* __restrict__ context_lens, int max_blocks,
    int B, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, const Cache c,
    int* status) {
  const bool is_v = (blockIdx.y & 1) != 0;
  const int kvh = blockIdx.y >> 1;
  const int b = threadIdx.x % kWriteRow;
  const int n = blockIdx.x * (kThreads / kWriteRow) + threadIdx.x / kWriteRow;
  if (n >= B) return;
  const int ctx = __ldg(context_lens + n);
  if (ctx < 1 || ctx > max_blocks << c.shift) return;  // the decode flags the length
  const int pos = ctx - 1;
  const int blk = __ldg(block_table + (size_t)n * max_blocks + (pos >> c.shift));
  if (blk < 0 || blk >= c.NB) {
    flag_error(status, PA_ERR_BLOCK_ID);
    return;
  }
  Block<T> r;
  load_block((is_v ? v : k) + n * token_stride + kvh * 128 + 16 * b, r);
  int t;
  const uint32_t g = group_of(c, blk, pos, kvh, t);
  put_block<T>(r, (is_v ? v_cache : k_cache) + (size_t)g * fp4::kGroupBytes, is_v, t, b);
}

// Eight held values as fp16 pairs, stored as T (exact: every held value is an fp16 and a bf16
// number; a NaN scale gives NaN). Streaming stores: the read is bound by its writes (1.05 M rows
// of 128 fp16 values, K and V: 139.6 us with them, 143.5 without, 143.5 for filling the same
// memory with a constant).
__device__ __forceinline__ void store8(const uint32_t (&h)[4], __half* p) {
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(h[0], h[1], h[2], h[3]));
}
__device__ __forceinline__ void store8(const uint32_t (&h)[4], __nv_bfloat16* p) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const __nv_bfloat162 o = __floats2bfloat162_rn(f.x, f.y);
    w[i] = *reinterpret_cast<const uint32_t*>(&o);
  }
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ void store8(const uint32_t (&h)[4], float* p) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[2 * i]));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h[2 * i + 1]));
    __stcs(reinterpret_cast<float4*>(p) + i, make_float4(a.x, a.y, b.x, b.y));
  }
}

// Rows read back: out rows of tokens with a negative or out-of-range slot are left as they are.
template <typename T>
__global__ void __launch_bounds__(kThreads) read_fp4_kernel(
    T* __restrict__ k_out, T* __restrict__ v_out, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const int* __restrict__ slot_mapping, int N,
    const Cache c, int* status) {
  constexpr int kTokens = kThreads / kReadRow;
  const bool is_v = (blockIdx.y & 1) != 0;
  const int kvh = blockIdx.y >> 1;
  const int c8 = threadIdx.x % kReadRow;
  const unsigned n0 = blockIdx.x * (unsigned)(kTokens * kReadTokens) + threadIdx.x / kReadRow;
  const uint8_t* cache = is_v ? v_cache : k_cache;
  T* out = (is_v ? v_out : k_out) + kvh * 128 + 8 * c8;
  const long long row = (long long)c.KVH * 128;
  int slot[kReadTokens];
#pragma unroll
  for (int i = 0; i < kReadTokens; ++i) {
    const unsigned n = n0 + i * kTokens;
    slot[i] = n < (unsigned)N ? __ldg(slot_mapping + n) : -1;
  }
  uint32_t w[kReadTokens], s[kReadTokens];
#pragma unroll
  for (int i = 0; i < kReadTokens; ++i) {
    const int blk = slot[i] >> c.shift;
    if (blk >= c.NB) {
      flag_error(status, PA_ERR_SLOT);
      slot[i] = -1;
    }
    if (slot[i] >= 0) {
      int t;
      const uint32_t g = group_of(c, blk, slot[i], kvh, t);
      const uint8_t* grp = cache + (size_t)g * fp4::kGroupBytes;
      w[i] = __ldg(reinterpret_cast<const uint32_t*>(grp + t * fp4::kCodeRow + 4 * c8));
      s[i] = __ldg(grp + fp4::scale_offset(is_v, t, c8 >> 1));
    }
  }
#pragma unroll
  for (int i = 0; i < kReadTokens; ++i) {
    if (slot[i] < 0) continue;
    uint32_t h[4];
    fp4::codes_to_f16x2(w[i], h[0], h[1], h[2], h[3]);
    const uint32_t s2 = s[i] * 0x00800080u;  // twice byte << 7
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = fp4::hmul2(h[e], s2);
    store8(h, out + (n0 + i * kTokens) * row);
  }
}

Cache cache_of(int NB, int KVH, int bs) {
  int shift = 4;
  while ((1 << shift) < bs) ++shift;
  return Cache{NB, KVH, shift};
}

// Grid of `tokens` tokens, per_cta of them to a CTA, for K and V of every kv head (the grid's
// second dimension holds 65535).
bool grid_of(long long tokens, int per_cta, int KVH, dim3* g) {
  if (KVH > 32767) return false;
  *g = dim3((unsigned)((tokens + per_cta - 1) / per_cta), 2u * (unsigned)KVH);
  return true;
}

template <typename T>
cudaError_t write_t(const void* k, const void* v, long long ts, const int* slots, int N, int KVH,
                    void* kc, void* vc, int NB, int bs, int* status, cudaStream_t st) {
  dim3 g;
  if (!grid_of(N, kThreads / kWriteRow * kWriteTokens, KVH, &g)) return cudaErrorInvalidValue;
  write_fp4_kernel<T><<<g, kThreads, 0, st>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), ts, slots, N,
      static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), cache_of(NB, KVH, bs), status);
  return cudaGetLastError();
}

template <typename T>
cudaError_t step_t(const void* k, const void* v, long long ts, const int* bt, const int* cl,
                   int max_blocks, int B, int KVH, void* kc, void* vc, int NB, int bs,
                   int* status, cudaStream_t st) {
  dim3 g;
  if (!grid_of(B, kThreads / kWriteRow, KVH, &g)) return cudaErrorInvalidValue;
  step_fp4_kernel<T><<<g, kThreads, 0, st>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), ts, bt, cl, max_blocks, B,
      static_cast<uint8_t*>(kc), static_cast<uint8_t*>(vc), cache_of(NB, KVH, bs), status);
  return cudaGetLastError();
}

template <typename T>
cudaError_t read_t(void* k, void* v, const void* kc, const void* vc, const int* slots, int N,
                   int KVH, int NB, int bs, int* status, cudaStream_t st) {
  dim3 g;
  if (!grid_of(N, kThreads / kReadRow * kReadTokens, KVH, &g)) return cudaErrorInvalidValue;
  read_fp4_kernel<T><<<g, kThreads, 0, st>>>(
      static_cast<T*>(k), static_cast<T*>(v), static_cast<const uint8_t*>(kc),
      static_cast<const uint8_t*>(vc), slots, N, cache_of(NB, KVH, bs), status);
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
