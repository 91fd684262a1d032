// RMS norm of every q and k head and the position rotation in one pass, with K and V optionally
// going straight into the paged cache.
//
// Per row x (one head of one token, 128 values):
//   y = x * rsqrt(mean(x^2) + eps) * w          (left out when there is no weight)
//   (a, b) -> (a c - b s, b c + a s)            over the first rot values, pairs (i, i + rot/2)
//                                               or, interleaved, (2i, 2i + 1)
// with c, s = the cosine and sine of the token's position, read from the caller's table. All of
// it in fp32, rounded once to the rows' type.
//
// Sixteen lanes hold a row, eight neighbouring values each (one 16-byte access for 16-bit rows), so a
// warp works on two heads at a time: four shuffles sum the squares, and a pair's other half is
// a neighbour value (interleaved) or eight lanes' exchange (rot / 16 lanes away). A warp stays
// with one token and takes kHeads heads per half-warp, all loaded before the first is used: the
// token's cosines and sines are read once for them and the loads overlap.
//
// The cache forms (kCache) round K to the rows' type first, so caches are bit for bit those of
// the separate calls, then quantise as the cache writes do: the 4-bit format's blocks are two
// lanes, the one-byte formats' row maximum is a half-warp's. One launch less for a step, and
// K's rows never go to memory and back.

#include "fp4.cuh"
#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_rows.cuh"

namespace pa {
namespace {

constexpr int kThreads = 128;
constexpr int kVals = 8;  // values of a lane

template <typename T> struct Row8 { uint4 u; };
template <> struct Row8<float> { float4 a, b; };

template <typename T>
__device__ __forceinline__ Row8<T> load8(const T* p) {
  return Row8<T>{__ldg(reinterpret_cast<const uint4*>(p))};
}
template <>
__device__ __forceinline__ Row8<float> load8<float>(const float* p) {
  return Row8<float>{__ldg(reinterpret_cast<const float4*>(p)),
                     __ldg(reinterpret_cast<const float4*>(p) + 1)};
}
__device__ __forceinline__ void widen(const Row8<__half>& r, float (&x)[kVals]) {
  const uint32_t w[4] = {r.u.x, r.u.y, r.u.z, r.u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
}
__device__ __forceinline__ void widen(const Row8<__nv_bfloat16>& r, float (&x)[kVals]) {
  const uint32_t w[4] = {r.u.x, r.u.y, r.u.z, r.u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(w[e] << 16);
    x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void widen(const Row8<float>& r, float (&x)[kVals]) {
  x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
  x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
}
__device__ __forceinline__ uint32_t pair_bits(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pair_bits(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[kVals]) {
  const T* tag = nullptr;
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pair_bits(x[0], x[1], tag), pair_bits(x[2], x[3], tag),
                 pair_bits(x[4], x[5], tag), pair_bits(x[6], x[7], tag));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[kVals]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Eight values of a row into the cache: lane l of the row's sixteen holds values 8l .. 8l + 7.
// All sixteen lanes call this together (`mask`: the lanes of the warp that do).
template <typename T, int KIND>
__device__ __forceinline__ void cache_row(const float (&x)[kVals], int l, unsigned mask,
                                          bool is_v, void* cache, float* scales, size_t page,
                                          int off, int bs) {
  if constexpr (KIND == kRowsFP4) {
    uint32_t m = 0u;
#pragma unroll
    for (int e = 0; e < kVals; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(mask, m, 1));
    const uint32_t sb = fp4::scale_byte(m);
    const float s = fp4::scale_value(sb), inv = fp4::scale_inverse(sb);
    constexpr bool kWide = sizeof(T) == 4;
    uint32_t w = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w |= fp4::code_pair(fp4::code_y<kWide>(x[2 * e], s, inv),
                          fp4::code_y<kWide>(x[2 * e + 1], s, inv))
           << (8 * e);
    uint8_t* grp = static_cast<uint8_t*>(cache) + fp4::group_offset(page, off, bs);
    const int t = off % fp4::kGroupTokens;
    *reinterpret_cast<uint32_t*>(grp + t * fp4::kCodeRow + 4 * l) = w;
    if ((l & 1) == 0) grp[fp4::scale_offset(is_v, t, l >> 1)] = (uint8_t)sb;
  } else {
    uint32_t w[4];  // fp16: eight halves; one byte: eight bytes in w[0], w[1]
    float s = 0.f;
    if constexpr (KIND == kRowsF16) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = pair_bits(x[2 * e], x[2 * e + 1], static_cast<const __half*>(nullptr));
    } else {
      float am = 0.f;
#pragma unroll
      for (int e = 0; e < kVals; ++e) am = fmaxf(am, fabsf(x[e]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(mask, am, o));
      s = KIND == kRowsI8 ? token_scale<T>(am) : __fdiv_rn(am, 448.f);
      const float inv = KIND == kRowsI8 ? __frcp_rn(s) : 0.f;
      w[0] = w[1] = 0u;
#pragma unroll
      for (int e = 0; e < kVals; ++e) {
        uint32_t q;
        if constexpr (KIND == kRowsI8) {
          q = (uint8_t)quant_fast(x[e], s, inv);
        } else {
          q = s > 0.f ? (uint32_t)(uint8_t)__nv_cvt_float_to_fp8(__fdiv_rn(x[e], s),
                                                                 __NV_SATFINITE, __NV_E4M3)
                      : 0u;
        }
        w[e >> 2] |= q << (8 * (e & 3));
      }
    }
    constexpr int ES = KIND == kRowsF16 ? 2 : 1;
    uint8_t* c = static_cast<uint8_t*>(cache);
    if (!is_v) {  // K page [D/8][bs][8]: a lane's values are one chunk
      uint8_t* dst = c + ((page * 16 + l) * (size_t)bs + off) * 8 * ES;
      if constexpr (KIND == kRowsF16) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      }
    } else {  // V page [D][bs]
#pragma unroll
      for (int e = 0; e < kVals; ++e) {
        const size_t i = (page * 128 + 8 * l + e) * bs + off;
        if constexpr (KIND == kRowsF16) {
          reinterpret_cast<uint16_t*>(c)[i] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        } else {
          c[i] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
        }
      }
    }
    if (KIND != kRowsF16 && l == 0) scales[page * bs + off] = s;
  }
}

// kCache: the cache's RowKind, or -1 for k rows written to k_out (and no V).
template <typename T, int kCache, int kHeads>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const RopeArgs a) {
  const int lane = threadIdx.x & 31;
  const int l = lane & 15;  // lane of the row
  const int half = lane >> 4;
  const unsigned mask = 0xffffu << (16 * half);
  const int heads = a.H + a.KVH + (kCache >= 0 ? a.KVH : 0);
  const int per_token = (heads + 2 * kHeads - 1) / (2 * kHeads);  // warps of a token
  const long long gw = ((long long)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const long long n = gw / per_token;
  if (n >= a.N) return;
  const int h0 = (int)(gw - n * per_token) * 2 * kHeads + half;

  // This half-warp's heads: h0, h0 + 2, ... (q heads, then k, then v).
  Row8<T> raw[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + 2 * i;
    const T* src;
    if (h < a.H) {
      src = static_cast<const T*>(a.q) + n * a.q_stride + (size_t)h * 128;
    } else if (h < a.H + a.KVH) {
      src = static_cast<const T*>(a.k) + n * a.k_stride + (size_t)(h - a.H) * 128;
    } else if (h < heads) {
      src = static_cast<const T*>(a.v) + n * a.v_stride + (size_t)(h - a.H - a.KVH) * 128;
    } else {
      break;
    }
    raw[i] = load8(src + kVals * l);
  }

  const int pos = __ldg(a.positions + n);
  if (pos < 0) return;  // padding token
  if (pos >= a.table_len) {
    if (lane == 0 && h0 == 0) flag_error(a.status, PA_ERR_POSITION);
    return;
  }
  // This token's place in the cache: page row of kv head 0, or none.
  long long page0 = -1;
  int off = 0;
  if constexpr (kCache >= 0) {
    const int slot = __ldg(a.slots + n);
    if (slot >= 0) {
      const int blk = slot / a.bs;
      if (blk < a.NB) {
        page0 = (long long)blk * a.KVH;
        off = slot - blk * a.bs;
      } else if (lane == 0 && h0 == 0) {
        flag_error(a.status, PA_ERR_SLOT);
      }
    }
  }

  // Cosines and sines of the lane's values: pairs share an angle, so the values 8l .. 8l + 7
  // need angles (8l .. 8l + 7) mod rot/2, or 4l .. 4l + 3 interleaved. Lanes past rot turn by
  // angle zero.
  const int rl = a.rot >> 3;      // lanes that turn
  const int hl = a.rot >> 4;      // lanes between a pair's halves (not interleaved)
  float c[kVals], s[kVals];
#pragma unroll
  for (int e = 0; e < kVals; ++e) {
    c[e] = 1.f;
    s[e] = 0.f;
  }
  if (l < rl) {
    const float* row = a.table + (size_t)pos * a.rot;
    if (a.interleaved) {
      const float4 c4 = __ldg(reinterpret_cast<const float4*>(row + 4 * l));
      const float4 s4 = __ldg(reinterpret_cast<const float4*>(row + a.rot / 2 + 4 * l));
      const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int e = 0; e < kVals; ++e) {
        c[e] = cc[e >> 1];
        s[e] = (e & 1) ? ss[e >> 1] : -ss[e >> 1];
      }
    } else {
      const bool up = l >= hl;  // second halves of the pairs: b c + a s, else a c - b s
      const float4* p = reinterpret_cast<const float4*>(row + 8 * (up ? l - hl : l));
      const float4* q = reinterpret_cast<const float4*>(row + a.rot / 2 + 8 * (up ? l - hl : l));
      const float4 c0 = __ldg(p), c1 = __ldg(p + 1), s0 = __ldg(q), s1 = __ldg(q + 1);
      const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
      for (int e = 0; e < kVals; ++e) {
        c[e] = cc[e];
        s[e] = up ? ss[e] : -ss[e];
      }
    }
  }
  // The lane holding the other halves (itself where nothing turns).
  const int other = (lane & 16) | (l < hl ? l + hl : (l < rl ? l - hl : l));

#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + 2 * i;
    if (h >= heads) break;
    float x[kVals];
    widen(raw[i], x);
    const bool is_q = h < a.H;
    const bool is_v = kCache >= 0 && h >= a.H + a.KVH;
    if (!is_v) {
      const T* w = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
      if (w != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < kVals; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
        const float inv = __frcp_rn(__fsqrt_rn(fmaf(sum, 1.f / 128.f, a.eps)));
        float wv[kVals];
        widen(load8(w + kVals * l), wv);
#pragma unroll
        for (int e = 0; e < kVals; ++e) x[e] = x[e] * inv * wv[e];
      }
      float y[kVals];
#pragma unroll
      for (int e = 0; e < kVals; ++e) {
        const float o = a.interleaved ? x[e ^ 1] : __shfl_sync(mask, x[e], other);
        y[e] = fmaf(x[e], c[e], o * s[e]);
      }
#pragma unroll
      for (int e = 0; e < kVals; ++e) x[e] = y[e];
    }
    if (is_q) {
      store8(static_cast<T*>(a.q_out) + n * a.qo_stride + (size_t)h * 128 + kVals * l, x);
    } else if constexpr (kCache < 0) {
      store8(static_cast<T*>(a.k_out) + n * a.ko_stride + (size_t)(h - a.H) * 128 + kVals * l,
             x);
    } else if (page0 >= 0) {
      const int kvh = h - a.H - (is_v ? a.KVH : 0);
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < kVals; ++e) x[e] = In<T>::round_t(x[e]);
      }
      cache_row<T, kCache>(x, l, mask, is_v, is_v ? a.v_cache : a.k_cache,
                           is_v ? a.v_scales : a.k_scales, (size_t)page0 + kvh, off, a.bs);
    }
  }
}

template <typename T, int kCache>
cudaError_t launch_t(const RopeArgs& a, int sms, cudaStream_t st) {
  const long long heads = a.H + a.KVH + (kCache >= 0 ? a.KVH : 0);
  // Four heads per half-warp where that still gives every SM sixteen warps, else one.
  const long long w4 = (long long)a.N * ((heads + 7) / 8);
  const bool few = w4 < 16LL * sms;
  const long long warps = few ? (long long)a.N * ((heads + 1) / 2) : w4;
  const long long grid = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (few) {
    norm_rope_kernel<T, kCache, 1><<<(int)grid, kThreads, 0, st>>>(a);
  } else {
    norm_rope_kernel<T, kCache, 4><<<(int)grid, kThreads, 0, st>>>(a);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_kind(int kind, const RopeArgs& a, int sms, cudaStream_t st) {
  switch (kind) {
    case -1: return launch_t<T, -1>(a, sms, st);
    case kRowsF16: return launch_t<T, kRowsF16>(a, sms, st);
    case kRowsI8: return launch_t<T, kRowsI8>(a, sms, st);
    case kRowsFP8: return launch_t<T, kRowsFP8>(a, sms, st);
    case kRowsFP4: return launch_t<T, kRowsFP4>(a, sms, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_norm_rope(int dtype, int kind, const RopeArgs& a, int sms, cudaStream_t st) {
  switch (dtype) {
    case PA_DTYPE_F16: return launch_kind<__half>(kind, a, sms, st);
    case PA_DTYPE_BF16: return launch_kind<__nv_bfloat16>(kind, a, sms, st);
    case PA_DTYPE_F32: return launch_kind<float>(kind, a, sms, st);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace pa
