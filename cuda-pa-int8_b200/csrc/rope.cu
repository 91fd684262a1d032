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
// Bound by memory for many tokens (each row read and written once), by latency for few. What kept
// a first version from that bound was its instruction count (104 a row), so:
//  * sixteen lanes hold a row, two chunks of four neighbouring values each, and a pair's two
//    halves sit in the same lane: chunk a holds values 4l .., chunk b the values rot/2 further on
//    (interleaved, and past rot: eight neighbouring values), so the rotation needs no exchange;
//  * a warp stays with one token and one kind of row (q, k or v) and takes kHeads heads per
//    half-warp, all loaded before the first is used. It folds the weights into the token's
//    cosines and sines once: a' = r (a (c w_a) - b (s w_b)), r = 1/rms, three operations a value.
//
// Measured on a B200 (graph replay): 16384 tokens, 32/8 heads, bf16: 62.4-65.5 us from one B200 to
// the next, 5.3-5.5 TB/s, 0.80-0.84 of the measured copy bandwidth (memory and issue slots both
// two thirds busy); 64 tokens: 2.4 us after another kernel of its graph, 4.2 as a graph of its
// own, a launch and two dependent loads. With the same kernel at 63.7 us, CTAs of 256 threads
// instead of 128: 71; 40 registers a thread for full occupancy: 76 (spills); four rows' sums
// reduced together, with fewer shuffles but all rows waited for at once: 65.6.
//
// The cache forms (kCache) round K to the rows' type first, so caches are bit for bit those of
// the separate calls, then quantise as the cache writes do. One launch less for a step, and K's
// rows never go to memory and back. A lane has eight values of a row, so V's page layout takes it
// eight stores where the token write has 16-byte ones for runs of slots: for few tokens this form
// is faster than the separate calls, for many slower. bf16, fused and separate, us:
//   28/4 heads, 16 tokens     4-bit 3.1  4.1   fp16 3.1  4.6   int8 3.6  5.2
//   28/4 heads, 1024 tokens   4-bit 7.2  7.2   fp16 12.3 13.3  int8 12.9 13.3
//   28/4 heads, 4096 tokens   4-bit 19.5 16.9  fp16 30.9 35.8  int8 36.0 33.4
//   32/8 heads, 16384 tokens  4-bit 99.9 76.8  fp16 179 91     int8 214 92 (prompts; 184 226 and
//                             197 213 at scattered slots)
// The int8 and fp8 kernels of four 16-bit heads a half-warp spill 8 to 24 bytes.

#include "fp4.cuh"
#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_rows.cuh"

#include <type_traits>

namespace pa {
namespace {

constexpr int kThreads = 128;

// Four neighbouring values as loaded (8 bytes for 16-bit rows, 16 for fp32).
template <typename T> struct Raw { using type = uint2; };
template <> struct Raw<float> { using type = float4; };

template <typename T>
__device__ __forceinline__ typename Raw<T>::type load4(const T* p) {
  return __ldg(reinterpret_cast<const typename Raw<T>::type*>(p));
}
// Of q, k and v rows: a plain load, since the outputs may be the inputs and __ldg is for memory
// that nothing writes during the launch.
template <typename T>
__device__ __forceinline__ typename Raw<T>::type load4_row(const T* p) {
  return *reinterpret_cast<const typename Raw<T>::type*>(p);
}
__device__ __forceinline__ void widen(uint2 u, const __half*, float2 (&x)[2]) {
  x[0] = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  x[1] = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
}
__device__ __forceinline__ void widen(uint2 u, const __nv_bfloat16*, float2 (&x)[2]) {
  x[0] = make_float2(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u));
  x[1] = make_float2(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void widen(float4 u, const float*, float2 (&x)[2]) {
  x[0] = make_float2(u.x, u.y);
  x[1] = make_float2(u.z, u.w);
}
__device__ __forceinline__ uint32_t pair_bits(float2 v, const __half*) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pair_bits(float2 v, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float2 (&x)[2]) {
  const T* tag = nullptr;
  *reinterpret_cast<uint2*>(p) = make_uint2(pair_bits(x[0], tag), pair_bits(x[1], tag));
}
template <>
__device__ __forceinline__ void store4<float>(float* p, const float2 (&x)[2]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
}

// a * b + c where `on`, else c, without a branch.
__device__ __forceinline__ float2 fma2_if(bool on, float2 a, float2 b, float2 c) {
  asm("{\n\t.reg .pred t;\n\t.reg .b64 x, y, z;\n\t"
      "setp.ne.s32 t, %6, 0;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%0, %1};\n\t"
      "@t fma.rn.f32x2 z, x, y, z;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "+f"(c.x), "+f"(c.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "r"((int)on));
  return c;
}

// CTAs an SM of the partly turned kernels of many 16-bit tokens, so that they keep to the 56
// registers of the others (4099 tokens, 28/4 heads, half the head, interleaved: 18.3 us without the
// bound, 17.6 with it).
template <typename T, int kCache, int kHeads, bool kWhole>
constexpr int kMinCtas = !kWhole && kCache < 0 && kHeads == 4 && sizeof(T) == 2 ? 9 : 0;

// A row into the cache. The lane's chunks: values oa .. oa + 3 (x[0], x[1]) and ob .. ob + 3
// (x[2], x[3]); `apart`: the chunks lie in different 16-value blocks, each shared by four
// neighbouring lanes (else both in one block of two lanes; for the 4-bit cache rot is a multiple
// of 32, so four neighbouring lanes agree). All lanes of the warp call this together; rows with
// `ok` false are not stored.
template <typename T, int KIND>
__device__ __forceinline__ void cache_row(const float2 (&x)[4], int l, int oa, int ob, bool apart,
                                          bool ok, bool is_v, void* cache, float* scales,
                                          size_t page, int off, int bs) {
  const float v[8] = {x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
  if constexpr (KIND == kRowsFP4) {
    uint32_t m[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e >> 2] = max(m[e >> 2], __float_as_uint(v[e]) & 0x7fffffffu);
    if (!apart) m[0] = m[1] = max(m[0], m[1]);
    uint8_t* grp = static_cast<uint8_t*>(cache) + fp4::group_offset(page, off, bs);
    const int t = off % fp4::kGroupTokens;
    constexpr bool kWide = sizeof(T) == 4;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t mc = max(m[c], __shfl_xor_sync(0xffffffffu, m[c], 1));
      const uint32_t far = __shfl_xor_sync(0xffffffffu, mc, 2);
      if (apart) mc = max(mc, far);
      const uint32_t sb = fp4::scale_byte<kWide>(mc);
      const float s = fp4::scale_value(sb), inv = fp4::scale_inverse<kWide>(sb);
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fp4::code_y<kWide>(v[4 * c + e], s, inv);
      const int o = c ? ob : oa;
      const uint32_t w = fp4::code_pair(y[0], y[1]) | (fp4::code_pair(y[2], y[3]) << 8);
      if (ok) *reinterpret_cast<uint16_t*>(grp + t * fp4::kCodeRow + o / 2) = (uint16_t)w;
      if (ok && (o & 15) == 0) grp[fp4::scale_offset(is_v, t, o / 16)] = (uint8_t)sb;
    }
  } else {
    float s = 0.f, inv = 0.f;
    if constexpr (KIND != kRowsF16) {
      float am = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(v[e]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
      s = KIND == kRowsI8 ? token_scale<T>(am) : __fdiv_rn(am, 448.f);
      inv = KIND == kRowsI8 ? __frcp_rn(s) : 0.f;
    }
    if (!ok) return;
    constexpr int ES = KIND == kRowsF16 ? 2 : 1;
    uint8_t* c8 = static_cast<uint8_t*>(cache);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int o = c ? ob : oa;
      uint32_t w[2] = {0u, 0u};  // fp16: four halves; one byte: four bytes in w[0]
      if constexpr (KIND == kRowsF16) {
        w[0] = pair_bits(x[2 * c], static_cast<const __half*>(nullptr));
        w[1] = pair_bits(x[2 * c + 1], static_cast<const __half*>(nullptr));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t q;
          if constexpr (KIND == kRowsI8) {
            q = (uint8_t)quant_fast(v[4 * c + e], s, inv);
          } else {
            q = s > 0.f ? (uint32_t)(uint8_t)__nv_cvt_float_to_fp8(__fdiv_rn(v[4 * c + e], s),
                                                                   __NV_SATFINITE, __NV_E4M3)
                        : 0u;
          }
          w[0] |= q << (8 * e);
        }
      }
      if (!is_v) {  // K page [D/8][bs][8]
        uint8_t* dst = c8 + ((page * 16 + o / 8) * (size_t)bs + off) * 8 * ES + (o & 7) * ES;
        if constexpr (KIND == kRowsF16) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
        } else {
          *reinterpret_cast<uint32_t*>(dst) = w[0];
        }
      } else {  // V page [D][bs]
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const size_t i = (page * 128 + o + e) * bs + off;
          if constexpr (KIND == kRowsF16) {
            reinterpret_cast<uint16_t*>(c8)[i] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
          } else {
            c8[i] = (uint8_t)(w[0] >> (8 * e));
          }
        }
      }
    }
    if (KIND != kRowsF16 && l == 0) scales[page * bs + off] = s;
  }
}

// kCache: the cache's RowKind, or -1 for k rows written to k_out (and no V). kInter: pairs
// (2i, 2i + 1). kWhole: rot is 128, every lane's values turn. Where rot is less, the other lanes'
// values are only scaled: with a sine of zero instead, a neighbour's infinity would make them NaN.
// 16384 tokens, 32/8 heads, bf16, half the head: 64-66 us with a branch, 67.6 with a predicate
// (interleaved, with the predicate, 62.7-65), 62-64 with the zero; whole heads, which need neither,
// 62.4 and, by a kernel for both, 65-71.
template <typename T, int kCache, int kHeads, bool kInter, bool kWhole>
__global__ void __launch_bounds__(kThreads, kMinCtas<T, kCache, kHeads, kWhole>)
norm_rope_kernel(const RopeArgs a) {
  using R = typename Raw<T>::type;
  const int lane = threadIdx.x & 31;
  const int l = lane & 15;  // lane of the row
  const int half = lane >> 4;
  // Warps of a token: those of its q rows, then k, then v.
  const int qw = (a.H + 2 * kHeads - 1) / (2 * kHeads);
  const int kw = (a.KVH + 2 * kHeads - 1) / (2 * kHeads);
  const unsigned per_token = qw + (kCache >= 0 ? 2 : 1) * kw;
  const unsigned gw = blockIdx.x * (unsigned)(kThreads / 32) + (threadIdx.x >> 5);
  const unsigned n = gw / per_token;
  if (n >= (unsigned)a.N) return;
  int w = (int)(gw - n * per_token);
  const bool is_q = w < qw;
  const bool is_v = w >= qw + kw;
  if (!is_q) w -= is_v ? qw + kw : qw;
  const int heads = is_q ? a.H : a.KVH;
  const int h0 = w * 2 * kHeads + half;  // this half-warp's heads: h0, h0 + 2, ...

  // The lane's chunks.
  const int turning = is_v ? 0 : a.rot >> 3;  // lanes whose values turn
  const bool turns = l < turning;
  const bool apart = !kInter && turns;
  const int oa = apart ? 4 * l : 8 * l;
  const int ob = apart ? (a.rot >> 1) + 4 * l : 8 * l + 4;

  const int pos = __ldg(a.positions + n);  // first: the table's row waits for it
  const T* src = static_cast<const T*>(is_q ? a.q : (is_v ? a.v : a.k)) +
                 (size_t)n * (is_q ? a.q_stride : (is_v ? a.v_stride : a.k_stride));
  R ra[kHeads], rb[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + 2 * i;
    ra[i] = rb[i] = R{};  // the half-warp past an odd last head goes along with zeros
    if (h < heads) {
      ra[i] = load4_row(src + h * 128 + oa);
      rb[i] = load4_row(src + h * 128 + ob);
    }
  }

  if (pos < 0) return;  // padding token
  if (pos >= a.table_len) {
    if (lane == 0 && w == 0 && is_q == (a.H > 0)) flag_error(a.status, PA_ERR_POSITION);
    return;
  }
  // This token's place in the cache: page row of kv head 0, or none.
  long long page0 = -1;
  int off = 0;
  if constexpr (kCache >= 0) {
    if (!is_q) {
      const int slot = __ldg(a.slots + n);
      if (slot >= 0) {
        const int blk = slot / a.bs;
        if (blk < a.NB) {
          page0 = (long long)blk * a.KVH;
          off = slot - blk * a.bs;
        } else if (lane == 0 && w == 0 && !is_v) {
          flag_error(a.status, PA_ERR_SLOT);
        }
      }
      if (page0 < 0) return;
    }
  }

  // Rotation coefficients with the weights folded in. Not interleaved: (a, b) = (chunk a, chunk b)
  // value by value; interleaved: (even, odd) values of the two chunks.
  //   u = a (c w_a) - b (s w_b),  v = b (c w_b) + a (s w_a)
  float2 cu[2], su[2], cv[2], sv[2];
  const T* wt = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
  const bool norm = !is_v && wt != nullptr;
  if (!is_v) {
    float2 wa[2], wb[2];
    if (norm) {
      widen(load4(wt + oa), static_cast<const T*>(nullptr), wa);
      widen(load4(wt + ob), static_cast<const T*>(nullptr), wb);
    } else {
      wa[0] = wa[1] = wb[0] = wb[1] = make_float2(1.f, 1.f);
    }
    float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (turns) {
      const float* row = a.table + (size_t)pos * a.rot + 4 * l;
      c = __ldg(reinterpret_cast<const float4*>(row));
      s = __ldg(reinterpret_cast<const float4*>(row + (a.rot >> 1)));
    }
    const float2 c2[2] = {make_float2(c.x, c.y), make_float2(c.z, c.w)};
    const float2 s2[2] = {make_float2(s.x, s.y), make_float2(s.z, s.w)};
    if constexpr (kInter) {
      // The pair's a-values: even values of the lane's eight; w likewise.
      const float2 we[2] = {make_float2(wa[0].x, wa[1].x), make_float2(wb[0].x, wb[1].x)};
      const float2 wo[2] = {make_float2(wa[0].y, wa[1].y), make_float2(wb[0].y, wb[1].y)};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cu[i] = mul2(c2[i], we[i]);
        su[i] = mul2(make_float2(-s2[i].x, -s2[i].y), wo[i]);
        cv[i] = mul2(c2[i], wo[i]);
        sv[i] = mul2(s2[i], we[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cu[i] = mul2(c2[i], wa[i]);
        su[i] = mul2(make_float2(-s2[i].x, -s2[i].y), wb[i]);
        cv[i] = mul2(c2[i], wb[i]);
        sv[i] = mul2(s2[i], wa[i]);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + 2 * i;
    if (h - half >= heads) break;
    const bool ok = h < heads;
    float2 x[4];  // chunk a, chunk b
    {
      float2 xa[2], xb[2];
      widen(ra[i], static_cast<const T*>(nullptr), xa);
      widen(rb[i], static_cast<const T*>(nullptr), xb);
      x[0] = xa[0]; x[1] = xa[1]; x[2] = xb[0]; x[3] = xb[1];
    }
    if (!is_v) {
      if (norm) {
        float2 q2 = mul2(x[0], x[0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) q2 = fma2(x[e], x[e], q2);
        float sum = q2.x + q2.y;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float r = rsqrtf(fmaf(sum, 1.f / 128.f, a.eps));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = mul2(x[e], make_float2(r, r));
      }
      if constexpr (kInter) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 p = make_float2(x[2 * e].x, x[2 * e + 1].x);
          const float2 q = make_float2(x[2 * e].y, x[2 * e + 1].y);
          const float2 u = kWhole ? fma2(q, su[e], mul2(p, cu[e]))
                                  : fma2_if(turns, q, su[e], mul2(p, cu[e]));
          const float2 v = kWhole ? fma2(p, sv[e], mul2(q, cv[e]))
                                  : fma2_if(turns, p, sv[e], mul2(q, cv[e]));
          x[2 * e] = make_float2(u.x, v.x);
          x[2 * e + 1] = make_float2(u.y, v.y);
        }
      } else if (!kWhole && !turns) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = mul2(x[e], cu[e]);
          x[2 + e] = mul2(x[2 + e], cv[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 u = fma2(x[2 + e], su[e], mul2(x[e], cu[e]));
          const float2 v = fma2(x[e], sv[e], mul2(x[2 + e], cv[e]));
          x[e] = u;
          x[2 + e] = v;
        }
      }
    }
    if (kCache < 0 || is_q) {
      T* dst = is_q ? static_cast<T*>(a.q_out) + (size_t)n * a.qo_stride + h * 128
                    : static_cast<T*>(a.k_out) + (size_t)n * a.ko_stride + h * 128;
      const float2 lo[2] = {x[0], x[1]}, hi[2] = {x[2], x[3]};
      if (ok) {
        store4(dst + oa, lo);
        store4(dst + ob, hi);
      }
    } else if constexpr (kCache >= 0) {
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = make_float2(In<T>::round_t(x[e].x), In<T>::round_t(x[e].y));
      }
      cache_row<T, kCache>(x, l, oa, ob, apart, ok, is_v, is_v ? a.v_cache : a.k_cache,
                           is_v ? a.v_scales : a.k_scales, (size_t)page0 + h, off, a.bs);
    }
  }
}

template <typename T, int kCache, int kHeads>
cudaError_t launch_heads(const RopeArgs& a, long long warps, cudaStream_t st) {
  const long long grid = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (warps > 0x7fffffffLL) return cudaErrorInvalidValue;
  auto launch = [&](auto inter, auto whole) {
    norm_rope_kernel<T, kCache, kHeads, decltype(inter)::value, decltype(whole)::value>
        <<<(int)grid, kThreads, 0, st>>>(a);
  };
  using Yes = std::true_type;
  using No = std::false_type;
  if (a.rot == 128) {
    if (a.interleaved) launch(Yes{}, Yes{}); else launch(No{}, Yes{});
  } else {
    if (a.interleaved) launch(Yes{}, No{}); else launch(No{}, No{});
  }
  return cudaGetLastError();
}

template <typename T, int kCache>
cudaError_t launch_t(const RopeArgs& a, int sms, cudaStream_t st) {
  auto warps = [&](int heads) {  // of the launch with `heads` heads a half-warp
    auto of = [&](int h) { return (h + 2LL * heads - 1) / (2 * heads); };
    return a.N * (of(a.H) + (kCache >= 0 ? 2 : 1) * of(a.KVH));
  };
  // Four heads per half-warp where that still gives every SM sixteen warps, else one (each warp's
  // chain is then shorter). 32/8 heads, bf16, one and four heads: 256 tokens (1280 warps of four)
  // 2.9 and 3.1 us, 512 tokens (2560) 4.5 and 3.8, 16384 tokens 102 and 62 (of 28 and 4 heads four
  // leave a fifth of the row slots empty).
  if (warps(4) >= 16LL * sms) return launch_heads<T, kCache, 4>(a, warps(4), st);
  return launch_heads<T, kCache, 1>(a, warps(1), st);
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
