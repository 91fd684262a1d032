// The 4-bit K/V cache format: device helpers shared by its writes and reads (fp4.cu), the
// norm-and-rotation kernel (rope.cu) and the decode kernel (decode_fp4.cu).
//
// A value is code * scale. Codes are e2m1 (sign, two exponent bits, one mantissa bit: 0, .5, 1,
// 1.5, 2, 3, 4, 6); sixteen neighbouring head_dim values of a row share one scale byte, an
// unsigned float of five exponent bits (bias 15) and three mantissa bits, so that byte << 7 is
// its fp16 bit pattern. The largest scale written is 10240 (0xE2): 6 * 10240 = 61440 is the
// largest magnitude the format holds, and every code * scale product (at most six significant
// bits, a multiple of 2^-18) is an exact fp16 and bf16 number, so pages convert to MMA operands
// without rounding. A block that holds a NaN or an infinity gets scale byte 0xFF, a NaN, and
// reads as NaN throughout.
//
// Why a scale per 16 values and not per row: the rows carry outlier channels (20 times the
// others in this library's own stress rows), and with one scale for all 128 values fifteen
// levels leave nothing of the rest. Why five exponent bits: 2^-17 .. 10240 covers what fp16 rows
// can hold, so no second scale per row has to be stored, read and multiplied in.
//
// Layout: 16 tokens of one block and kv head form a group of 1152 bytes,
//   cache [num_blocks][kv_heads][block_size / 16][1152] (uint8),
//   group: codes [16 tokens][64 bytes], byte j = head_dim 2j (low half) and 2j + 1 (high half);
//          scales: K [16 tokens][8], V [8][16 tokens].
// A token owns whole bytes (no two tokens share one), so tokens of a group are written
// independently. A group is one contiguous copy for the decode kernel. The code rows are what a
// lane of the QK MMA reads as 16 bytes; the V scales' order lets a lane of the PV MMA read its
// four tokens' scales as one word.
#pragma once

#include "pa_common.cuh"

namespace pa {
namespace fp4 {

constexpr int kGroupTokens = 16;
constexpr int kCodeRow = 64;                              // code bytes of one token
constexpr int kCodes = kGroupTokens * kCodeRow;           // 1024: offset of the scales
constexpr int kGroupBytes = kCodes + kGroupTokens * 8;    // 1152
constexpr uint32_t kScaleMax = 0xE2u;                     // 10240 = 1.25 * 2^13
constexpr uint32_t kScaleNan = 0xFFu;

// Byte offset of the group holding token `off` of page row `page` (= block * kv_heads + head).
__device__ __forceinline__ size_t group_offset(size_t page, int off, int bs) {
  return (page * (size_t)(bs / kGroupTokens) + off / kGroupTokens) * kGroupBytes;
}
// Offset inside the group of scale b of token t.
__device__ __forceinline__ int scale_offset(bool is_v, int t, int b) {
  return kCodes + (is_v ? b * kGroupTokens + t : t * 8 + b);
}

// Scale byte of a block from the bit pattern of its largest magnitude (as an unsigned integer:
// NaN and infinities compare above every finite value): the nearest representable to amax / 6,
// ties to even.
// fp32 inputs (kWide): the IEEE quotient, which reaches a midpoint between two scales (five
// significant bits) only where the exact one does.
// 16-bit inputs: amax times 1/6, two roundings off by at most 2^-23 of it, then rounded to 17
// significant bits. A quotient on a midpoint comes out as the midpoint; any other quotient of an
// 11-bit amax by 6 is at least 2^-13 of its value away from it.
template <bool kWide>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kScaleNan;
  const float amax = __uint_as_float(amax_bits);
  uint32_t u;
  if constexpr (kWide) {
    u = __float_as_uint(__fdiv_rn(amax, 6.f));
  } else {
    u = (__float_as_uint(__fmul_rn(amax, 1.f / 6.f)) + 0x40u) & ~0x7fu;
  }
  const float t = __uint_as_float(u);
  // From 2^-14 up: round to four significant bits; the exponent field moves from bias 127 to 15.
  const uint32_t normal = ((u + 0x7ffffu + ((u >> 20) & 1u)) >> 20) - (112u << 3);
  // Below: steps of 2^-17 (adding 96 rounds to that grid, ties to even).
  const uint32_t small = __float_as_uint(__fadd_rn(t, 96.f)) & 0xffu;
  return min(t < 0x1p-14f ? small : normal, kScaleMax);
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __half2float(__ushort_as_half((unsigned short)(byte << 7)));
}

// Factor for code_y below: 1 / scale; 0 for the zero scale (zero codes) and for NaN, where the
// codes mean nothing. 16-bit inputs take the hardware's approximate reciprocal (2^-23 off at most).
template <bool kWide>
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
  if (byte == 0u || byte == kScaleNan) return 0.f;
  if constexpr (kWide) return __frcp_rn(scale_value(byte));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale_value(byte)));
  return r;
}

// x / scale, close enough to round to the same code as the exact quotient.
// 16-bit inputs (kWide false): fma(x, 1/scale, 96) - 96 puts the quotient on a grid of 2^-17.
// The borders between codes (.25 .75 1.25 1.75 2.5 3.5 5) lie on that grid, the product is within
// 2^-20 of the quotient there, so a quotient on a border comes out as the border; any other
// quotient of an 11-bit x and a 4-bit scale is at least 2^-13 away from it.
// fp32 inputs: the IEEE quotient, which reaches a border only where the exact one does.
template <bool kWide>
__device__ __forceinline__ float code_y(float x, float s, float inv) {
  if constexpr (kWide) {
    return inv == 0.f ? 0.f : __fdiv_rn(x, s);
  } else {
    return __fadd_rn(__fmaf_rn(x, inv, 96.f), -96.f);
  }
}

// Two e2m1 codes, the nearest to a (low half of the byte) and b (high half), ties to the even
// code, magnitudes above 6 as 6.
__device__ __forceinline__ uint32_t code_pair(float a, float b) {
  uint32_t r;
  asm("{\n\t.reg .b8 c;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n\t"
      "cvt.u32.u8 %0, c;\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b));
  return r;
}
// Eight codes, y[0] in the lowest four bits.
__device__ __forceinline__ uint32_t code_word(const float (&y)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c3, %8, %7;\n\t"
      "mov.b32 %0, {c0, c1, c2, c3};\n\t}"
      : "=r"(r)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}

// Four code bytes as four fp16 pairs (low half of the byte in the low half of the pair), exact.
__device__ __forceinline__ void codes_to_f16x2(uint32_t w, uint32_t& h0, uint32_t& h1,
                                               uint32_t& h2, uint32_t& h3) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h0), "=r"(h1), "=r"(h2), "=r"(h3)
      : "r"(w));
}

// Two scale bytes of z as two fp16 scales: bytes 0 and 1, or 2 and 3 with sel 0x3424.
__device__ __forceinline__ uint32_t scale_pair(uint32_t z, uint32_t sel = 0x1404u) {
  return prmt(z, 0u, sel) >> 1;  // b << 8 in each half, shifted down to b << 7
}

// a times the low or the high half of s (the multiply takes the half as an operand modifier).
template <bool kHigh>
__device__ __forceinline__ uint32_t hmul2_half(uint32_t a, uint32_t s) {
  const __half2 s2 = *reinterpret_cast<const __half2*>(&s);
  const __half2 d = __hmul2(*reinterpret_cast<const __half2*>(&a),
                            kHigh ? __high2half2(s2) : __low2half2(s2));
  return *reinterpret_cast<const uint32_t*>(&d);
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// One row by one warp: lane l holds values 4l .. 4l + 3. Returns the lane's two code bytes; all
// lanes get their block's scale byte (block l / 4).
template <bool kWide>
__device__ __forceinline__ uint32_t warp_quantize4(const float (&x)[4], uint32_t& scale) {
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  scale = scale_byte<kWide>(m);
  const float s = scale_value(scale), inv = scale_inverse<kWide>(scale);
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = code_y<kWide>(x[e], s, inv);
  return code_pair(y[0], y[1]) | (code_pair(y[2], y[3]) << 8);
}

}  // namespace fp4
}  // namespace pa
