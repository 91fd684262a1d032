// Paged-attention decode over the 4-bit K/V cache (format and layout: fp4.cuh).
//
// The work is cut as in decode.cu: one warp per equal range of 16-token pages of the flattened
// sequence x kv head x head tile x page list. A segment cut between warps leaves partials; those of
// one CTA are merged in its shared memory, those of several CTAs by the one that arrives last, in
// page order, so results do not depend on timing. (A partial of every warp in the workspace, as
// decode.cu has it, cost 2.5 us a launch and, where few sequences have many pages, much more:
// 1 x 8192 tokens, 12/2 heads, 58 us instead of 16.)
// The page loop is its own, because at 144 bytes a token and kv head it is bound by what the four
// schedulers of an SM can issue, not by memory:
//  * two pages a step, copied by all lanes of the warp (16-byte asynchronous copies into the
//    warp's ring), so a step's fixed costs are shared by 32 tokens;
//  * S^T = K Q^T with tokens on the MMA's 16 rows and the (up to 8) heads of a kv head on its
//    columns: half the MMAs of heads on rows. The weights' 8 x 8 tiles are transposed in registers
//    (movmatrix) into the B fragments of O^T = V^T P^T;
//  * codes convert two at a time (cvt e2m1x2 -> f16x2) and are multiplied by their block's scale,
//    exactly, before the MMA: a lane's 32 K values are two blocks of one token, its 64 V values
//    one block of four tokens;
//  * a running maximum that moves only when a score passes it by 2^8, so most steps need no
//    reduction over the lanes and no rescale;
//  * weights enter PV as two fp16 parts, as in decode.cu: one rounding to fp16 would add as much
//    error as the output's own.
//  * steps of two full pages run in a loop with nothing to check; a step's scale and maximum are
//    one multiply-add before the exponential (raw scores are compared with a threshold).
// 281 warp instructions a page (479 with decode.cu's loop): 64 conversions, 64 multiplies, 24
// MMAs, 16 to pair the codes of neighbouring tokens for PV, the rest softmax, copies and loop.
// Measured on a B200 (graph replay): 64 x 8192 tokens, 12/2 heads 41.2 us (3.68 TB/s); 8 x 64-128
// K, 64/8 heads 167 us in a short run (5.44 TB/s, 0.83 of the measured copy bandwidth), 189-201 in
// a loop of seconds, at the power cap of 1000 W and 1.65-1.75 GHz. That is 463 cycles a page
// and scheduler, of which ALU instructions (conversions, logic) take 249, MMAs 192 and the FMA pipe
// up to 189; they hardly overlap (a group of one MMA and three conversions and multiplies takes
// 18.6 cycles where the MMA alone takes 8 and the others 8). Shifts turned into multiplies, the
// QK of the next step issued between the PV of this one, two chains of QK MMAs a page instead of
// one, and a choice of refill inside one loop for all full pages measured no better.

#include "fp4.cuh"
#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_rows.cuh"

#include <atomic>
#include <type_traits>

namespace pa {
namespace {

// log2 of the factor by which the softmax weights are formed (as in decode.cu: keeps the fp16
// parts of the weights normal; it cancels in O / l and is taken out of partials).
constexpr float kPExp = 6.f;

template <int D, int GT, int DEPTH, int WARPS>
struct Tile {
  static constexpr int NS = D / 32;          // words of eight codes a lane reads of a K token
  static constexpr int MT = D / 16;          // PV m-tiles (head_dim rows)
  static constexpr int NT = GT / 8;          // head tiles of eight
  static constexpr int SLOT = (D + 2) * GT;  // partial slot floats
  static constexpr int PT = fp4::kGroupBytes;
  static constexpr int STAGE = 4 * PT;       // two pages: K, K, V, V
  static constexpr size_t RING = (size_t)WARPS * DEPTH * STAGE;
  // A piece's partial as it lies in shared memory: rows of GT heads, four floats of padding every
  // sixteen rows (the lanes that store a column of rows then meet in a bank two at a time instead
  // of eight), maxima, sums.
  static constexpr int PIECE = SLOT + D / 4;
  static constexpr size_t EARLY = (size_t)WARPS * PIECE * sizeof(float);
  static constexpr size_t SMEM = 128 + RING + EARLY;
  static_assert((size_t)DEPTH * STAGE >= PIECE * sizeof(float),
                "a warp's ring holds its last piece");
};

// Merges take bf16 output rows too, and pass NaN on (a block of the cache that holds one) instead
// of taking it for an empty sequence. This file shares no code with decode.cu's: sharing it through a
// header left its kernels' resources as they were but made the FP8 decode 2 % slower (66.3 -> 67.5
// us at 64 x 8192 tokens, 12/2 heads).
//
// One output value, as fp16 or bf16.
__device__ __forceinline__ void store_out(__half* p, float v, bool bf) {
  if (bf) {
    *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v);
  } else {
    *p = __float2half_rn(v);
  }
}

// ---------------------------------------------------------------------------------------
// Log-sum-exp merge of rows `slice` * D / kSlices .. of `np` partials by one warp: m = max m_k,
// o = sum 2^(m_k - m) o_k, l likewise. piece(k) is partial k, in shared memory (SMEM, with its
// padding) or a global slot [D][GT], [GT] maxima, [GT] sums. Four partials are in flight at once,
// and they enter in the order of k, so the bits do not depend on timing. The result is the
// normalised output rows (out_rows, fp16 or with bf bf16), or a slot (out_slot).
// ---------------------------------------------------------------------------------------
constexpr int kSlices = 4;

template <int D, int GT, bool SMEM, typename PieceFn>
__device__ __forceinline__ void merge_rows(PieceFn piece, int np, int slice, int lane, int hcnt,
                                           __half* out_rows, bool bf, float* out_slot,
                                           int* status) {
  constexpr int ROWS = D / kSlices;
  constexpr int O4 = ROWS * GT / 4 / 32;  // float4 outputs of a lane
  constexpr int U = 4;
  constexpr int ML = D * GT + (SMEM ? D / 4 : 0);  // where the maxima are
  static_assert(ROWS * GT / 4 % 32 == 0, "outputs must tile the warp");
  auto load = [](const float* s) {
    float4 v;
    if constexpr (SMEM) v = *reinterpret_cast<const float4*>(s);
    else v = __ldcg(reinterpret_cast<const float4*>(s));
    return v;
  };
  // Output i: row d_of(i), heads h0 .. h0 + 3.
  const int h0 = 4 * (lane % (GT / 4));
  auto d_of = [&](int i) { return slice * ROWS + (lane + 32 * i) / (GT / 4); };
  float M[4], L[4], acc[O4][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    M[e] = neg_inf();
    L[e] = 0.f;
#pragma unroll
    for (int i = 0; i < O4; ++i) acc[i][e] = 0.f;
  }
  for (int k0 = 0; k0 < np; k0 += U) {
    float4 m[U], l[U], v[U][O4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* s = piece(min(k0 + u, np - 1));
      m[u] = load(s + ML + h0);
      l[u] = load(s + ML + GT + h0);
#pragma unroll
      for (int i = 0; i < O4; ++i)
        v[u][i] = load(s + d_of(i) * GT + (SMEM ? d_of(i) / 16 * 4 : 0) + h0);
      if (k0 + u >= np) m[u] = make_float4(neg_inf(), neg_inf(), neg_inf(), neg_inf());
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      auto at = [&](const float4& x) { return e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w; };
      float mn = M[e];
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, at(m[u]));
      const float from = mn == neg_inf() ? 0.f : mn;
      const float c = ex2(M[e] - from);
      M[e] = mn;
      L[e] *= c;
#pragma unroll
      for (int i = 0; i < O4; ++i) acc[i][e] *= c;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = ex2(at(m[u]) - from);
        L[e] = fmaf(w, at(l[u]), L[e]);
#pragma unroll
        for (int i = 0; i < O4; ++i) acc[i][e] = fmaf(w, at(v[u][i]), acc[i][e]);
      }
    }
  }
  if (out_rows != nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (h0 + e >= hcnt) continue;
      const float inv = L[e] == 0.f ? 0.f : 1.f / L[e];
      if (L[e] == 0.f) flag_error(status, PA_ERR_EMPTY_CONTEXT);
#pragma unroll
      for (int i = 0; i < O4; ++i)
        store_out(out_rows + (size_t)(h0 + e) * D + d_of(i), acc[i][e] * inv, bf);
    }
  } else {
#pragma unroll
    for (int i = 0; i < O4; ++i)
      *reinterpret_cast<float4*>(out_slot + d_of(i) * GT + h0) =
          make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    if (slice == 0 && lane < GT / 4) {
      *reinterpret_cast<float4*>(out_slot + D * GT + h0) = make_float4(M[0], M[1], M[2], M[3]);
      *reinterpret_cast<float4*>(out_slot + D * GT + GT + h0) =
          make_float4(L[0], L[1], L[2], L[3]);
    }
  }
}

// ---------------------------------------------------------------------------------------
// CTA-cooperative log-sum-exp merge of `np` partial slots (all NTHR threads of the block take
// part; scratch is shared memory). Pass 1 forms the maxima, the per-piece weights (kept in
// shared memory) and the denominators with every thread reading a different piece; pass 2
// gives each thread one float4 of the [D][GT] output and U pieces' loads in flight per step,
// so a merge costs a handful of dependent L2 round trips however many pieces there are.
// ---------------------------------------------------------------------------------------
template <int D, int GT, int NTHR, int U>
struct Coop {
  static constexpr int OUT4 = D * GT / 4;                        // float4 outputs
  static constexpr int PG = NTHR >= OUT4 ? NTHR / OUT4 : 1;      // piece groups
  static constexpr int OPT = NTHR >= OUT4 ? 1 : OUT4 / NTHR;     // outputs per thread
  static constexpr int NW = NTHR / 32;
  // Scratch floats needed for np pieces.
  __host__ __device__ static constexpr size_t floats(int np) {
    return 2 * GT + NW * GT + ((size_t)np * GT + 3) / 4 * 4 + (size_t)PG * OUT4 * 4;
  }
};

template <int D, int GT, int NTHR, int U, typename PieceFn>
__device__ __forceinline__ void coop_combine(PieceFn piece, int np, int hcnt, __half* out_rows,
                                             bool bf, float* out_slot, int* status,
                                             float* sm) {
  using CC = Coop<D, GT, NTHR, U>;
  static_assert(NTHR >= CC::OUT4 || CC::OUT4 % NTHR == 0, "outputs must tile the block");
  const int tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5;
  float* sM = sm;
  float* sL = sm + GT;
  float* sRed = sm + 2 * GT;
  float* sW = sRed + CC::NW * GT;
  float4* sAcc = reinterpret_cast<float4*>(sW + ((size_t)np * GT + 3) / 4 * 4);

  float mx[GT];
#pragma unroll
  for (int h = 0; h < GT; ++h) mx[h] = neg_inf();
  for (int k = tid; k < np; k += NTHR) {
    const float4* mk = reinterpret_cast<const float4*>(piece(k) + D * GT);
#pragma unroll
    for (int h4 = 0; h4 < GT / 4; ++h4) {
      const float4 v = __ldcg(mk + h4);
      mx[4 * h4 + 0] = fmaxf(mx[4 * h4 + 0], v.x);
      mx[4 * h4 + 1] = fmaxf(mx[4 * h4 + 1], v.y);
      mx[4 * h4 + 2] = fmaxf(mx[4 * h4 + 2], v.z);
      mx[4 * h4 + 3] = fmaxf(mx[4 * h4 + 3], v.w);
    }
  }
#pragma unroll
  for (int h = 0; h < GT; ++h) {
    const float v = warp_max(mx[h]);
    if (lane == 0) sRed[warp * GT + h] = v;
  }
  __syncthreads();
  if (tid < GT) {
    float v = neg_inf();
    for (int w = 0; w < CC::NW; ++w) v = fmaxf(v, sRed[w * GT + tid]);
    sM[tid] = v;
  }
  __syncthreads();
  float ls[GT];
#pragma unroll
  for (int h = 0; h < GT; ++h) ls[h] = 0.f;
  for (int k = tid; k < np; k += NTHR) {
    const float4* mk = reinterpret_cast<const float4*>(piece(k) + D * GT);
#pragma unroll
    for (int h4 = 0; h4 < GT / 4; ++h4) {
      const float4 m4 = __ldcg(mk + h4);
      const float4 l4 = __ldcg(mk + GT / 4 + h4);
      const float mm[4] = {m4.x, m4.y, m4.z, m4.w};
      const float ll[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int h = 4 * h4 + e;
        const float M = sM[h];
        const float w = (M == neg_inf()) ? 0.f : ex2(mm[e] - M);
        sW[(size_t)k * GT + h] = w;
        ls[h] += w * ll[e];
      }
    }
  }
#pragma unroll
  for (int h = 0; h < GT; ++h) {
    float v = ls[h];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sRed[warp * GT + h] = v;
  }
  __syncthreads();
  if (tid < GT) {
    float v = 0.f;
    for (int w = 0; w < CC::NW; ++w) v += sRed[w * GT + tid];
    sL[tid] = v;
  }
  __syncthreads();

  const int pg = (NTHR >= CC::OUT4) ? tid / CC::OUT4 : 0;
  float4 acc[CC::OPT];
#pragma unroll
  for (int i = 0; i < CC::OPT; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (pg < CC::PG) {
#pragma unroll
    for (int i = 0; i < CC::OPT; ++i) {
      const int o = (NTHR >= CC::OUT4) ? tid % CC::OUT4 : tid + i * NTHR;
      const int h0 = (o % (GT / 4)) * 4;
      for (int k0 = pg; k0 < np; k0 += CC::PG * U) {
        float4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = k0 + u * CC::PG;
          v[u] = (k < np) ? __ldcg(reinterpret_cast<const float4*>(piece(k)) + o)
                          : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = k0 + u * CC::PG;
          if (k < np) {
            const float* w = sW + (size_t)k * GT + h0;
            acc[i].x += w[0] * v[u].x;
            acc[i].y += w[1] * v[u].y;
            acc[i].z += w[2] * v[u].z;
            acc[i].w += w[3] * v[u].w;
          }
        }
      }
    }
  }
  if constexpr (CC::PG > 1) {
    if (pg < CC::PG) sAcc[pg * CC::OUT4 + tid % CC::OUT4] = acc[0];
    __syncthreads();
    if (pg == 0) {
      for (int g2 = 1; g2 < CC::PG; ++g2) {
        const float4 t = sAcc[g2 * CC::OUT4 + tid];
        acc[0].x += t.x;
        acc[0].y += t.y;
        acc[0].z += t.z;
        acc[0].w += t.w;
      }
    }
  }
  if (pg == 0) {
#pragma unroll
    for (int i = 0; i < CC::OPT; ++i) {
      const int o = (NTHR >= CC::OUT4) ? tid : tid + i * NTHR;
      const int d = o / (GT / 4);
      const int h0 = (o % (GT / 4)) * 4;
      const float a4[4] = {acc[i].x, acc[i].y, acc[i].z, acc[i].w};
      if (out_rows != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = h0 + e;
          if (h < hcnt) {
            const float L = sL[h];
            store_out(out_rows + (size_t)h * D + d, L == 0.f ? 0.f : a4[e] / L, bf);
          }
        }
      } else {
        reinterpret_cast<float4*>(out_slot)[o] = acc[i];
      }
    }
  }
  if (tid < GT) {
    if (out_slot != nullptr) {
      out_slot[D * GT + tid] = sM[tid];
      out_slot[D * GT + GT + tid] = sL[tid];
    } else if (tid < hcnt && sL[tid] == 0.f) {
      flag_error(status, PA_ERR_EMPTY_CONTEXT);
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------
// Decode step over a 4-bit cache: one warp quantises the new token's K and V rows (16-bit, at
// src_k / src_v) and stores them into the cache, at token `off` of page row `row`, before it
// loads the page. Only the calling warp reads the page.
// ---------------------------------------------------------------------------------------
template <int D>
__device__ __noinline__ void store_new_token_fp4(const uint8_t* src_k, const uint8_t* src_v,
                                                 int new_dtype, uint8_t* kc, uint8_t* vc,
                                                 size_t row, int off, int bs, int lane) {
  static_assert(D == 128, "one lane per four head_dim values");
  const size_t grp = fp4::group_offset(row, off, bs);
  const int t = off % fp4::kGroupTokens;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint8_t* src = which ? src_v : src_k;
    float x[4];
    if (new_dtype == PA_DTYPE_BF16) {
      load_vals<__nv_bfloat16, 4>(reinterpret_cast<const __nv_bfloat16*>(src) + 4 * lane, x);
    } else {
      load_vals<__half, 4>(reinterpret_cast<const __half*>(src) + 4 * lane, x);
    }
    uint32_t sb;
    const uint32_t w = fp4::warp_quantize4<false>(x, sb);
    uint8_t* dst = (which ? vc : kc) + grp;
    *reinterpret_cast<uint16_t*>(dst + t * fp4::kCodeRow + 2 * lane) = (uint16_t)w;
    if ((lane & 3) == 0) dst[fp4::scale_offset(which != 0, t, lane >> 2)] = (uint8_t)sb;
  }
  __syncwarp();
}

// ---------------------------------------------------------------------------------------
// The decode kernel.
// ---------------------------------------------------------------------------------------
// PACK (kv heads of at most four q heads): the PV MMA's columns 0-3 take the weights' high parts
// and columns 4-7 their low parts, one MMA instead of two; the two halves of O are added at the
// end of a piece.
template <int D, int GT, bool PACK, int DEPTH, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) decode_fp4_kernel(const DecodeFp4Args a) {
  static_assert(!PACK || GT == 8, "packed weights need the idle columns of one head tile");
  using C = Tile<D, GT, DEPTH, WARPS>;
  constexpr int NS = C::NS;
  constexpr int MT = C::MT;
  constexpr int NT = C::NT;
  constexpr int SLOT = C::SLOT;
  constexpr int NTHR = WARPS * 32;

  __shared__ int s_pre[kBMax + 1];
  __shared__ int s_ctx[kBMax];
  __shared__ int s_tmp[32];
  __shared__ int s_empty;
  __shared__ unsigned s_over[kBMax / 32];  // sequences whose context exceeds the table
  __shared__ int s_pend[WARPS][2][6];   // a warp's partials: see the piece epilogue
  __shared__ int s_npend[WARPS];
  __shared__ int s_last[2];
  __shared__ int s_nblk[WARPS][32];     // block ids of a warp's next batch of pages
  __shared__ int s_nmeta[WARPS][32];    // their (kv_head << 3) | subpage
  __shared__ int s_nwr[WARPS][32];      // their decode-step new-token sequence, or -1
  extern __shared__ __align__(16) uint8_t dsm_raw[];
  uint8_t* ring = dsm_raw + ((128u - (smem_u32(dsm_raw) & 127u)) & 127u);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;  // MMA group (row / column index)
  const int r = lane & 3;   // position inside the group

  if (threadIdx.x == 0) {
    s_empty = 0;
    // This CTA's share of the block tables and q rows into L2, so the first block-id and q
    // reads after the scan do not each wait for DRAM.
    prefetch_l2_share(a.block_table, (size_t)a.B * a.max_blocks * sizeof(int), blockIdx.x,
                      gridDim.x);
    prefetch_l2_share(a.q, (size_t)a.B * a.H * D * sizeof(__half), blockIdx.x, gridDim.x);
  }

  // ---- 1. Scan of per-sequence page counts (all CTAs, identical result) -------------------
  const int SEGS = a.KVH * a.HT;
  const int cap = a.max_blocks * a.bs;
  int carry = 0;
  for (int i = threadIdx.x; i < kBMax / 32; i += NTHR) s_over[i] = 0u;
  __syncthreads();
  for (int base = 0; base < a.B; base += NTHR) {
    const int b = base + threadIdx.x;
    int w = 0;
    if (b < a.B) {
      int c = __ldg(a.context_lens + b);
      if (c < 1) {
        if (blockIdx.x == 0 && a.mode != kModePartial) flag_error(a.status, PA_ERR_EMPTY_CONTEXT);
        if (blockIdx.x == 0 && c < 0) flag_error(a.status, PA_ERR_CONTEXT_RANGE);
        s_empty = 1;
        c = 0;
      }
      if (c > cap) {
        if (blockIdx.x == 0) flag_error(a.status, PA_ERR_CONTEXT_RANGE);
        atomicOr(&s_over[b >> 5], 1u << (b & 31));
        c = cap;
      }
      s_ctx[b] = c;
      w = ((c + kSubTokens - 1) / kSubTokens) * SEGS;
    }
    int v = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += t;
    }
    if (lane == 31) s_tmp[warp] = v;
    __syncthreads();
    if (warp == 0) {
      int t = (lane < WARPS) ? s_tmp[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += u;
      }
      if (lane < WARPS) s_tmp[lane] = t;
    }
    __syncthreads();
    if (b < a.B) s_pre[b] = carry + (warp ? s_tmp[warp - 1] : 0) + v - w;
    carry += s_tmp[WARPS - 1];
    __syncthreads();
  }
  if (threadIdx.x == 0) s_pre[a.B] = carry;
  __syncthreads();
  const int T = carry;

  // Sequences with no tokens: zero output (stream) or an empty partial (partial mode).
  if (blockIdx.x == 0 && s_empty) {
    if (a.mode == kModeStream) {
      const int per_b = a.H * D / 8;
      for (int i = threadIdx.x; i < a.B * per_b; i += NTHR) {
        const int b = i / per_b;
        if (s_ctx[b] == 0)
          reinterpret_cast<uint4*>(a.out + (size_t)b * a.H * D)[i - b * per_b] =
              make_uint4(0u, 0u, 0u, 0u);
      }
    } else if (a.mode == kModePartial) {
      for (int i = threadIdx.x; i < a.B * SEGS * SLOT; i += NTHR) {
        const int segid = i / SLOT;
        const int b = segid / SEGS;
        if (s_ctx[b] == 0) {
          const int k = i - segid * SLOT;
          a.part_out[i] = (k >= D * GT && k < D * GT + GT) ? neg_inf() : 0.f;
        }
      }
    }
  }
  if (T == 0) return;

  auto pages_of = [&](int b) { return (s_ctx[b] + kSubTokens - 1) / kSubTokens; };
  // Flattened page index -> (sequence, segment inside the sequence, subpage).
  auto locate = [&](int p, int& b, int& seg, int& sp) {
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_pre[mid] <= p) lo = mid; else hi = mid - 1;
    }
    b = lo;
    const int rel = p - s_pre[b];
    const int pg = pages_of(b);
    seg = rel / pg;
    sp = rel - seg * pg;
  };
  // ---- 2. This warp's page range ------------------------------------------------------------
  const long long Wt = min((long long)a.total_warps, (long long)T);
  const int wg = blockIdx.x * WARPS + warp;
  long long p0 = 0, p1 = 0;
  if (wg < Wt) {
    p0 = (long long)wg * T / Wt;
    p1 = (long long)(wg + 1) * T / Wt;
  }
  const int n = (int)(p1 - p0);
  int nrec = 0;  // partials of segments shared with other warps
  if (n > 0) {

  // ---- 3. Consumer position and the first piece's q rows --------------------------------------
  int cb, cseg, csp;
  locate((int)p0, cb, cseg, csp);
  int cpg = pages_of(cb);
  int cctx = s_ctx[cb];
  // Scores are taken times |scale| log2 e; a negative scale turns q's signs. (A zero scale becomes
  // one whose scores vanish against each other all the same.)
  const float qs = fmaxf(fabsf(a.qk_scale_log2), 1e-30f);
  const uint32_t qsign = a.qk_scale_log2 < 0.f ? 0x80008000u : 0u;

  // Q as the B fragments of the QK MMA (fp16): values 32r .. 32r + 31 of head g (qa) and, with 16
  // heads to a tile, of head g + 8 (qb).
  uint4 qa[NS], qb[NS];
  uint4 ra[NS], rb[NS];  // q rows fetched ahead of the piece that uses them
  int q_b = -1, q_seg = -1;

  auto fetch_q = [&](int b, int seg) {
    const int kvh = seg / a.HT;
    const int ht = seg - kvh * a.HT;
    const int hl = ht * GT + g;
    const __half* qrow = a.q + ((size_t)b * a.H + (size_t)kvh * a.G + hl) * D + 32 * r;
#pragma unroll
    for (int si = 0; si < NS; ++si) {
      ra[si] = (hl < a.G) ? __ldg(reinterpret_cast<const uint4*>(qrow) + si)
                          : make_uint4(0u, 0u, 0u, 0u);
      rb[si] = make_uint4(0u, 0u, 0u, 0u);
      if (GT == 16 && hl + 8 < a.G)
        rb[si] = __ldg(reinterpret_cast<const uint4*>(qrow + 8 * D) + si);
    }
  };
  // Eight bf16 values as fp16: exact inside the fp16 normal range; larger magnitudes saturate and
  // are flagged, as by the conversion kernel of pa_decode_bf16q.
  auto bf16_to_f16 = [&](uint4 v) {
    const uint32_t src[4] = {v.x, v.y, v.z, v.w};
    uint32_t dst[4];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float lo = __uint_as_float(src[e] << 16), hi = __uint_as_float(src[e] & 0xffff0000u);
      if (fabsf(lo) > 65504.f) {
        bad = true;
        lo = copysignf(65504.f, lo);
      }
      if (fabsf(hi) > 65504.f) {
        bad = true;
        hi = copysignf(65504.f, hi);
      }
      dst[e] = pack_f16x2(lo, hi);
    }
    if (bad) flag_error(a.status, PA_ERR_Q_RANGE);
    return make_uint4(dst[0], dst[1], dst[2], dst[3]);
  };
  auto convert_q = [&]() {
    auto turn = [&](uint4 v) {
      if (a.act_bf16) v = bf16_to_f16(v);
      return make_uint4(v.x ^ qsign, v.y ^ qsign, v.z ^ qsign, v.w ^ qsign);
    };
#pragma unroll
    for (int si = 0; si < NS; ++si) {
      qa[si] = turn(ra[si]);
      if constexpr (NT == 2) qb[si] = turn(rb[si]);
    }
  };
  // The first piece's q rows are requested before the page copies, so their latency overlaps
  // the block-table reads and the first copies rather than queueing behind them.
  fetch_q(cb, cseg);
  q_b = cb;
  q_seg = cseg;

  // ---- 4. Producer: the group indices of 32 upcoming pages, one per lane. With a decode step, wr
  // receives the sequence whose new token lies in the page (the last page of a segment whose
  // context and block id are valid), else -1.
  const bool step_write = a.new_k != nullptr;
  const uint64_t pol = l2_policy_evict_first();
  // Page jbase + lane of the range: the address of its block id, its (kv_head << 3) | subpage
  // and, for a decode step, the sequence whose new token it holds (else -1).
  auto page_ref = [&](int jbase, int& meta, int& wr) -> const int* {
    meta = 0;
    wr = -1;
    const int jj = jbase + lane;
    if (jj >= n) return nullptr;
    int b, seg, sp;
    locate((int)(p0 + jj), b, seg, sp);
    const int bi = sp / a.subs;
    meta = ((seg / a.HT) << 3) | (sp - bi * a.subs);
    if (step_write && sp == pages_of(b) - 1 && !((s_over[b >> 5] >> (b & 31)) & 1u)) wr = b;
    return a.block_table + (size_t)b * a.max_blocks + bi;
  };
  // Group index of a page (below 2^31); a block id outside the cache is flagged and read as block
  // 0, and its new token (if any) is not written.
  auto pack_page = [&](int blk, int meta, int& wr) -> uint32_t {
    if (blk < 0 || blk >= a.NB) {
      flag_error(a.status, PA_ERR_BLOCK_ID);
      blk = 0;
      wr = -1;
    }
    return (uint32_t)((blk * a.KVH + (meta >> 3)) * a.subs + (meta & 7));
  };
  int curw, meta0;
  const int* bref0 = page_ref(0, meta0, curw);
  const int blk0 = bref0 != nullptr ? __ldg(bref0) : 0;
  uint32_t cur = pack_page(blk0, meta0, curw);

  // Decode step: the new token in the page of group gi, if it holds one (sequence wb >= 0), is
  // written into the cache before the page is copied.
  auto write_new = [&](uint32_t gi, int wb) {
    if (wb < 0) return;
    const uint32_t row = gi / (uint32_t)a.subs;
    const size_t so = ((size_t)wb * a.new_stride + (size_t)(row % (uint32_t)a.KVH) * D) * 2;
    store_new_token_fp4<D>(static_cast<const uint8_t*>(a.new_k) + so,
                           static_cast<const uint8_t*>(a.new_v) + so, a.new_dtype, a.k_write,
                           a.v_write, row, (s_ctx[wb] - 1) % a.bs, a.bs, lane);
    __threadfence();  // the copies read what the warp's lanes have just written, from L2
    __syncwarp();
  };
  // The warp's ring is filled by 16-byte asynchronous copies of all its lanes, one commit group
  // per stage of two pages. (Four bulk copies per stage, issued by one lane, cost 87 of the step's
  // 640 instructions; nine copies a lane and their addresses cost about 25.) A page's K and V
  // groups are 72 chunks each: two rounds of the warp, and the last eight chunks of all four
  // groups in one more round.
  const uint32_t my_ring = smem_u32(ring) + (uint32_t)(warp * DEPTH) * (uint32_t)C::STAGE;
  const uint8_t* k_lane = a.k_cache + 16 * lane;
  const uint8_t* v_lane = a.v_cache + 16 * lane;
  const uint8_t* rest_lane = ((lane & 16) ? a.v_cache : a.k_cache) + 1024 + 16 * (lane & 7);
  const uint32_t rest_off =
      (uint32_t)(lane >> 3) * (uint32_t)C::PT + 1024u + 16u * (uint32_t)(lane & 7);
  auto copy_pair = [&](uint32_t g0, uint32_t g1, int s) {
    const uint32_t st = my_ring + (uint32_t)s * (uint32_t)C::STAGE;
    const uint32_t sl = st + 16u * (uint32_t)lane;
    const size_t o0 = (size_t)g0 * C::PT, o1 = (size_t)g1 * C::PT;
    cp_async_16_hint(sl, k_lane + o0, pol);
    cp_async_16_hint(sl + 512, k_lane + o0 + 512, pol);
    cp_async_16_hint(sl + C::PT, k_lane + o1, pol);
    cp_async_16_hint(sl + C::PT + 512, k_lane + o1 + 512, pol);
    cp_async_16_hint(sl + 2 * C::PT, v_lane + o0, pol);
    cp_async_16_hint(sl + 2 * C::PT + 512, v_lane + o0 + 512, pol);
    cp_async_16_hint(sl + 3 * C::PT, v_lane + o1, pol);
    cp_async_16_hint(sl + 3 * C::PT + 512, v_lane + o1 + 512, pol);
    cp_async_16_hint(st + rest_off, rest_lane + (size_t)((lane & 8) ? g1 : g0) * C::PT, pol);
  };
  // Pages jj and jj + 1 (jj even; asked for in order) into stage s; past the range's end the
  // group is empty, and a missing second page is the first once more. The ids of the next 32
  // pages come along with a batch's first stage, sixteen groups before they are needed.
  static_assert(2 * DEPTH < 32, "a batch's ids must arrive before the batch begins");
  auto issue_pair = [&](int jj, int s) {
    if (jj < n) {
      if ((jj & 31) == 0) {
        if (jj > 0) {
          curw = s_nwr[warp][lane];
          cur = pack_page(s_nblk[warp][lane], s_nmeta[warp][lane], curw);
        }
        int meta, wr;
        const int* p = page_ref(jj + 32, meta, wr);
        s_nmeta[warp][lane] = meta;
        s_nwr[warp][lane] = wr;
        if (p != nullptr) {
          cp_async_4(&s_nblk[warp][lane], p);
        } else {
          s_nblk[warp][lane] = 0;  // past the range: any valid id
        }
      }
      const int i1 = (jj & 31) + (jj + 1 < n ? 1 : 0);
      const uint32_t g0 = __shfl_sync(0xffffffffu, cur, jj & 31);
      const uint32_t g1 = __shfl_sync(0xffffffffu, cur, i1);
      if (step_write) {
        write_new(g0, __shfl_sync(0xffffffffu, curw, jj & 31));
        write_new(g1, __shfl_sync(0xffffffffu, curw, i1));
      }
      copy_pair(g0, g1, s);
    }
    cp_async_commit();
  };
  __syncwarp();
  for (int j = 0; j < DEPTH; ++j) issue_pair(2 * j, j);
  convert_q();

  // Of heads nt * 8 + 2r and the next: the reference maximum m (a whole number, so that rescaling
  // by a change of it is exact) as fmb = kPExp - m, the score at which it moves, and the sum.
  float fmb[NT][2], thr[NT][2], fl[NT][2];
  float oacc[MT][NT][4];
  const int tau = 4 * (g >> 1) + (g & 1);  // token of K row g (row g + 8: + 2)

  int s = 0;  // ring stage of page j
  int j = 0;
  while (j < n) {
    // ---- one piece: the pages of this warp's range inside one segment, pages
    // [csp, csp + len) of sequence cb, segment cseg.
    const int piece_sp0 = csp;
    const int len = min(cpg - csp, n - j);
    if (q_b != cb || q_seg != cseg) {
      fetch_q(cb, cseg);
      convert_q();
      q_b = cb;
      q_seg = cseg;
    }
    // When this piece ends its segment and the range goes on, the next segment's q rows are
    // brought into L1 while this piece runs, so the next piece's q fetch does not wait on L2.
    if (csp + len == cpg && j + len < n) {
      int nb = cb, ns = cseg + 1;
      if (ns == SEGS) {
        ns = 0;
        do { ++nb; } while (pages_of(nb) == 0);
      }
      const int kvh = ns / a.HT;
      const int hl = (ns - kvh * a.HT) * GT + (lane >> 1);
      if (lane < 2 * GT && hl < a.G)
        prefetch_l1(a.q + ((size_t)nb * a.H + (size_t)kvh * a.G + hl) * D + (lane & 1) * (D / 2));
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) oacc[i][nt][e] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        fmb[nt][e] = -neg_inf();
        thr[nt][e] = neg_inf();
        fl[nt][e] = 0.f;
      }
    bool far = false;  // a maximum is far from zero: see the step
    // One step: the two pages of stage s. FULL: all their tokens count; else valid0 and valid1 of
    // them do (where a piece begins or ends inside a stage, the page that is not its own has
    // none, and is met again by the other piece). False: nothing was done, the step needs !FULL.
    auto step = [&](auto full, int s, int valid0, int valid1) -> bool {
      constexpr bool FULL = decltype(full)::value;
      const uint32_t st = my_ring + (uint32_t)s * (uint32_t)C::STAGE;
      const uint32_t ka = st + tau * fp4::kCodeRow + 16 * r;
      const uint32_t ksa = st + fp4::kCodes + tau * 8 + 2 * r;
      const uint32_t va = st + 2 * C::PT + 4 * r * fp4::kCodeRow + 8 * g;
      const uint32_t vsa = st + 2 * C::PT + fp4::kCodes + 16 * g + 4 * r;

      // S^T = K Q^T: rows = tokens (row g: token tau, row g + 8: tau + 2), columns = heads, so
      // that eight heads fill the MMA. A lane reads the 32 codes 32r .. 32r + 31 of its two
      // tokens; codes -> fp16, times the block scale, is exact (fp4.cuh).
      float x[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 c0 = lds128(ka + u * C::PT), c1 = lds128(ka + u * C::PT + 2 * fp4::kCodeRow);
        const uint32_t z0 = lds16(ksa + u * C::PT), z1 = lds16(ksa + u * C::PT + 16);
        const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
        const uint32_t s0 = fp4::scale_pair(z0), s1 = fp4::scale_pair(z1);
        float acc[NT][4];
        auto mma = [](bool begin, float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                      uint32_t a3, uint32_t b0, uint32_t b1) {
          if (begin) mma_16816_zero(d, a0, a1, a2, a3, b0, b1);
          else mma_16816(d, a0, a1, a2, a3, b0, b1);
        };
#pragma unroll
        for (int si = 0; si < NS; ++si) {
          uint32_t h[4], i4[4];
          fp4::codes_to_f16x2(w0[si], h[0], h[1], h[2], h[3]);
          fp4::codes_to_f16x2(w1[si], i4[0], i4[1], i4[2], i4[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[e] = si < NS / 2 ? fp4::hmul2_half<false>(h[e], s0)
                               : fp4::hmul2_half<true>(h[e], s0);
            i4[e] = si < NS / 2 ? fp4::hmul2_half<false>(i4[e], s1)
                                : fp4::hmul2_half<true>(i4[e], s1);
          }
          mma(si == 0, acc[0], h[0], i4[0], h[1], i4[1], qa[si].x, qa[si].y);
          mma(false, acc[0], h[2], i4[2], h[3], i4[3], qa[si].z, qa[si].w);
          if constexpr (NT == 2) {
            mma(si == 0, acc[1], h[0], i4[0], h[1], i4[1], qb[si].x, qb[si].y);
            mma(false, acc[1], h[2], i4[2], h[3], i4[3], qb[si].z, qb[si].w);
          }
        }
        // Raw scores: heads nt * 8 + 2r + (e & 1) of token tau (e < 2) and tau + 2.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][nt][e] = acc[nt][e];
      }
      if constexpr (!FULL) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int vd = u ? valid1 : valid0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (tau + (e & 2) >= vd) x[u][nt][e] = neg_inf();
        }
      }
      // The reference maximum moves only when a score passes it by 2^kLazy: weights then stay
      // below 2^(kPExp + kLazy) (far inside fp16), O and l carry the same factor, and most
      // steps need neither a reduction over the lanes nor a rescale.
      // Far from zero the weights' one multiply-add fails: fp32 scores of 2^27 have no bits below 1
      // left, so the unrounded product may be off the rounded maximum by any power of two, and the
      // threshold's own rounding lets as much through. Once a score that moves a maximum is 2^18
      // (`far`, until the piece ends) the products are rounded as the maxima are, and every larger
      // score moves its maximum. Steps of full pages leave that to the others: they stop before
      // they have changed anything. (Heads of one tile: no time lost; of 9-16 heads 1-2 %, 12/1 5 %.
      // With the branch inside them, one tile 0.4-2 %, 9-16 heads 4-9 %; two operations for every
      // score 0.3-1.7 % of one tile.)
      constexpr float kLazy = 8.f, kFar = 0x1p18f;
      float tm[NT][2];
      bool up = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          tm[nt][e] = fmaxf(fmaxf(x[0][nt][e], x[0][nt][2 + e]),
                            fmaxf(x[1][nt][e], x[1][nt][2 + e]));
          up = up || tm[nt][e] > thr[nt][e];
        }
      if (__any_sync(0xffffffffu, up)) {
        bool is_far = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float h = fabsf(tm[nt][e] * qs);
            is_far = is_far || (h >= kFar && h != -neg_inf());
          }
        if (__any_sync(0xffffffffu, is_far)) {
          far = true;
          if constexpr (FULL) return false;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = tm[nt][e];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            if constexpr (FULL) {
              const float m = kPExp - fmb[nt][e], mn = fmaxf(m, ceilf(v * qs));
              c[e] = mn > m ? ex2(m - mn) : 1.f;
              fmb[nt][e] = kPExp - mn;
              thr[nt][e] = __fdividef(mn + kLazy, qs);
            } else {  // the maximum moves up, fmb down
              const float f = fminf(fmb[nt][e], kPExp - ceilf(__fmul_rn(v, qs)));
              c[e] = f < fmb[nt][e] ? ex2(f - fmb[nt][e]) : 1.f;
              fmb[nt][e] = f;
              thr[nt][e] = far ? fmaxf(thr[nt][e], v) : __fdividef(kPExp - f + kLazy, qs);
            }
            fl[nt][e] *= c[e];
            if constexpr (PACK) {  // columns 4-7 belong to the heads of columns 0-3
              const float other = __shfl_xor_sync(0xffffffffu, c[e], 2);
              if (r >= 2) c[e] = other;
            }
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) {  // O's columns are the lane's own heads
            oacc[i][nt][0] *= c[0];
            oacc[i][nt][1] *= c[1];
            oacc[i][nt][2] *= c[0];
            oacc[i][nt][3] *= c[1];
          }
        }
      }

      auto weight_arg = [&](float a, float b, int nt) {
        const float2 f = make_float2(fmb[nt][0], fmb[nt][1]);
        // (Scalar multiplications: packed ones and the addition would be fused.)
        if (!FULL && far) return add2(make_float2(__fmul_rn(a, qs), __fmul_rn(b, qs)), f);
        return fma2(make_float2(a, b), make_float2(qs, qs), f);
      };
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // Weights, as two fp16 parts each (about 22 significant bits, as for the other
        // caches); the transposed 8 x 8 tiles are the PV MMA's B fragments.
        uint32_t ph0[NT], ph1[NT], pl0[NT], pl1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 v = weight_arg(x[u][nt][e], x[u][nt][e + 1], nt);
            p[e] = ex2(v.x);
            p[e + 1] = ex2(v.y);
            const float2 l = add2(make_float2(fl[nt][0], fl[nt][1]),
                                  make_float2(p[e], p[e + 1]));
            fl[nt][0] = l.x;
            fl[nt][1] = l.y;
          }
          split_f16x2_packed(p[0], p[1], ph0[nt], pl0[nt]);
          split_f16x2_packed(p[2], p[3], ph1[nt], pl1[nt]);
          if constexpr (PACK) {
            const uint32_t o0 = __shfl_xor_sync(0xffffffffu, pl0[nt], 2);
            const uint32_t o1 = __shfl_xor_sync(0xffffffffu, pl1[nt], 2);
            if (r >= 2) {
              ph0[nt] = o0;
              ph1[nt] = o1;
            }
          }
          ph0[nt] = transpose8x8(ph0[nt]);
          ph1[nt] = transpose8x8(ph1[nt]);
          if constexpr (!PACK) {
            pl0[nt] = transpose8x8(pl0[nt]);
            pl1[nt] = transpose8x8(pl1[nt]);
          }
        }
        // V: tokens 4r .. 4r + 3, values 16g .. 16g + 15 (one block a token). Scales of slots
        // past the context may be anything: zero there (a finite code times zero is 0).
        uint2 vq[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) vq[e] = lds64(va + u * C::PT + e * fp4::kCodeRow);
        const uint32_t z = lds32(vsa + u * C::PT);
        uint32_t s01 = fp4::scale_pair(z), s23 = fp4::scale_pair(z, 0x3424u);
        if constexpr (!FULL) {
          const int vd = u ? valid1 : valid0;
          s01 &= ((4 * r < vd) ? 0x0000ffffu : 0u) | ((4 * r + 1 < vd) ? 0xffff0000u : 0u);
          s23 &= ((4 * r + 2 < vd) ? 0x0000ffffu : 0u) | ((4 * r + 3 < vd) ? 0xffff0000u : 0u);
        }
        // O^T += V^T P^T. The MMA pairs tokens: the even and the odd head_dim codes of two
        // tokens share a byte before they convert. Rows g and g + 8 of m-tile 4h + jj are
        // head_dim 16g + 8h + 2jj and the next.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w0 = h ? vq[0].y : vq[0].x, w1 = h ? vq[1].y : vq[1].x;
          const uint32_t w2 = h ? vq[2].y : vq[2].x, w3 = h ? vq[3].y : vq[3].x;
          constexpr uint32_t kLow = 0x0f0f0f0fu;
          uint32_t A0[4], A1[4], A2[4], A3[4];
          fp4::codes_to_f16x2((w0 & kLow) | ((w1 << 4) & ~kLow), A0[0], A0[1], A0[2], A0[3]);
          fp4::codes_to_f16x2(((w0 >> 4) & kLow) | (w1 & ~kLow), A1[0], A1[1], A1[2], A1[3]);
          fp4::codes_to_f16x2((w2 & kLow) | ((w3 << 4) & ~kLow), A2[0], A2[1], A2[2], A2[3]);
          fp4::codes_to_f16x2(((w2 >> 4) & kLow) | (w3 & ~kLow), A3[0], A3[1], A3[2], A3[3]);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            const int i = 4 * h + jj;
            const uint32_t a0 = fp4::hmul2(A0[jj], s01), a1 = fp4::hmul2(A1[jj], s01);
            const uint32_t a2 = fp4::hmul2(A2[jj], s23), a3 = fp4::hmul2(A3[jj], s23);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816(oacc[i][nt], a0, a1, a2, a3, ph0[nt], ph1[nt]);
              if constexpr (!PACK)
                mma_16816(oacc[i][nt], a0, a1, a2, a3, pl0[nt], pl1[nt]);
            }
          }
        }
      }
      return true;
    };
    for (int k = 0; k < len;) {
      const int first = j & 1;
      // Steps with nothing to check: full pages whose refill lies inside the range and inside the
      // present batch of block ids.
      if (first == 0 && !step_write && !far) {
        const int jr = j + 2 * DEPTH;  // the next refill's first page
        int m = min(len - k, (cctx - (csp + k) * kSubTokens) / kSubTokens) / 2;
        m = min(min(m, (n - jr) / 2), (-jr & 31) / 2);
        for (int i = 0; i < m; ++i) {
          cp_async_wait_groups<DEPTH - 1>();
          __syncwarp();
          if (!step(std::true_type{}, s, kSubTokens, kSubTokens)) break;
          __syncwarp();
          const int e = (j + 2 * DEPTH) & 31;
          copy_pair(__shfl_sync(0xffffffffu, cur, e), __shfl_sync(0xffffffffu, cur, e + 1), s);
          cp_async_commit();
          if (++s == DEPTH) s = 0;
          k += 2;
          j += 2;
        }
        if (k >= len) break;
      }
      const int cnt = min(2 - first, len - k);
      if (first == 0) {  // the stage's copies: this lane's, then every lane's
        cp_async_wait_groups<DEPTH - 1>();
        __syncwarp();
      }
      const int left = cctx - (csp + k) * kSubTokens;  // tokens from the step's first page on
      step(std::false_type{}, s, first ? 0 : min(kSubTokens, left),
           first ? min(kSubTokens, left) : (cnt == 2 ? min(kSubTokens, left - kSubTokens) : 0));
      k += cnt;
      j += cnt;
      if ((j & 1) == 0) {  // both pages of the stage are done with: refill it
        __syncwarp();
        issue_pair(j + 2 * DEPTH - 2, s);
        if (++s == DEPTH) s = 0;
      }
    }
    csp += len;

    {
      // ---- piece epilogue ---------------------------------------------------------------------
      if constexpr (PACK) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            oacc[i][0][e] += __shfl_xor_sync(0xffffffffu, oacc[i][0][e], 2);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
            fl[nt][e] += __shfl_xor_sync(0xffffffffu, fl[nt][e], o);
      const int segid = cb * SEGS + cseg;
      const int kvh = cseg / a.HT;
      const int ht = cseg - kvh * a.HT;
      const int hbase = kvh * a.G + ht * GT;
      const int hcnt = min(GT, a.G - ht * GT);

      // Partial slots hold O and l without the 2^kPExp weight factor (an exact rescale).
      auto write_slot = [&](float* slot, int pad) {  // pad: floats after every sixteen rows
        constexpr float kUnscale = 1.f / (float)(1 << (int)kPExp);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            *reinterpret_cast<float2*>(slot + (16 * GT + pad) * g + 2 * i * GT + nt * 8 + 2 * r) =
                make_float2(oacc[i][nt][0] * kUnscale, oacc[i][nt][1] * kUnscale);
            *reinterpret_cast<float2*>(slot + (16 * GT + pad) * g + (2 * i + 1) * GT + nt * 8 +
                                       2 * r) =
                make_float2(oacc[i][nt][2] * kUnscale, oacc[i][nt][3] * kUnscale);
          }
        }
        slot += pad * (D / 16);
        if (g == 0) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            *reinterpret_cast<float2*>(slot + D * GT + nt * 8 + 2 * r) =
                make_float2(kPExp - fmb[nt][0], kPExp - fmb[nt][1]);
            *reinterpret_cast<float2*>(slot + D * GT + GT + nt * 8 + 2 * r) =
                make_float2(fl[nt][0] * kUnscale, fl[nt][1] * kUnscale);
          }
        }
      };

      if (piece_sp0 == 0 && csp == cpg) {
        // The whole segment was this warp's: normalise and store directly.
        if (a.mode == kModeStream) {
          // A lane holds values 16g .. 16g + 15 of its heads: 32 contiguous bytes each.
          __half* ob = a.out + ((size_t)cb * a.H + hbase) * D;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int h = nt * 8 + 2 * r + e;
              const float f = 1.f / fl[nt][e];
              uint32_t w[MT];
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                const float lo = oacc[i][nt][e] * f, hi = oacc[i][nt][2 + e] * f;
                if (a.act_bf16) {
                  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
                  w[i] = *reinterpret_cast<const uint32_t*>(&v);
                } else {
                  w[i] = pack_f16x2(lo, hi);
                }
              }
              if (h < hcnt) {
                uint4* o = reinterpret_cast<uint4*>(ob + (size_t)h * D + 16 * g);
                o[0] = make_uint4(w[0], w[1], w[2], w[3]);
                o[1] = make_uint4(w[4], w[5], w[6], w[7]);
              }
            }
        } else {
          write_slot(a.part_out + (size_t)segid * SLOT, 0);
        }
      } else {
        // A piece of a segment shared with neighbouring warps: at most two, the one that ends
        // the segment the range begins in and the one the range ends with. The latter goes into
        // the warp's ring, which is done with.
        const int early = j < n ? 1 : 0;
        const int off = early ? (int)(C::RING / sizeof(float)) + warp * C::PIECE
                              : warp * (DEPTH * C::STAGE / (int)sizeof(float));
        __syncwarp();
        write_slot(reinterpret_cast<float*>(ring) + off, 4);
        if (lane == 0 && nrec < 2) {
          const long long s_start = (long long)s_pre[cb] + (long long)cseg * cpg;
          const long long s_end = s_start + cpg;
          int* pe = s_pend[warp][nrec];
          pe[0] = segid;
          pe[1] = off;
          pe[2] = cb;
          pe[3] = (hbase << 5) | hcnt;
          pe[4] = (int)(((s_start + 1) * Wt - 1) / T) / WARPS;  // the segment's first CTA
          pe[5] = (int)((s_end * Wt - 1) / T) / WARPS;          // and its last
        }
        ++nrec;
      }
    }

    // ---- next segment
    if (csp == cpg) {
      csp = 0;
      if (++cseg == SEGS) {
        cseg = 0;
        if (j < n) {
          do { ++cb; } while (pages_of(cb) == 0);
          cctx = s_ctx[cb];
        }
      }
      if (j < n) cpg = pages_of(cb);
    }
  }

  cp_async_wait_all();
  }  // n > 0

  // ---- 5. Merges. A CTA's warps hold neighbouring ranges, so the partials of a segment lie side
  // by side: first the CTA's own are merged in shared memory. A segment that it holds alone is
  // done; of others (at most two, the first and the last) the CTA leaves one partial in the
  // workspace, and the CTA that arrives last merges those. (With a partial of every warp in the
  // workspace one segment of 8192 tokens was up to 512 of them: 1 x 8192 tokens took 58 us.)
  if (lane == 0) s_npend[warp] = min(nrec, 2);
  __syncthreads();
  // Entry i = 2 * warp + e in lane i; groups of entries of one segment.
  static_assert(2 * WARPS <= 32, "a lane for each partial");
  const bool have = lane < 2 * WARPS && (lane & 1) < s_npend[min(lane >> 1, WARPS - 1)];
  const int* pe = s_pend[min(lane >> 1, WARPS - 1)][lane & 1];
  const int e_seg = have ? pe[0] : -1, e_off = have ? pe[1] : 0, e_b = have ? pe[2] : 0;
  const int e_heads = have ? pe[3] : 0, e_c0 = have ? pe[4] : 0, e_c1 = have ? pe[5] : 0;
  const unsigned entries = __ballot_sync(0xffffffffu, have);
  const unsigned below = entries & ((1u << lane) - 1u);
  int* const s_off = s_nblk[warp];  // (done with) the entries' places, packed
  if (have) s_off[__popc(below)] = e_off;
  __syncwarp();
  const int prev_seg = __shfl_sync(0xffffffffu, e_seg, below ? 31 - __clz(below) : 0);
  const unsigned heads = __ballot_sync(0xffffffffu, have && (below == 0u || prev_seg != e_seg));
  const unsigned cross = heads & __ballot_sync(0xffffffffu, have && e_c0 != e_c1);
  const bool stream = (a.mode == kModeStream);
  const bool bf = a.act_bf16 != 0;
  const int cta = blockIdx.x;
  float* const smem = reinterpret_cast<float*>(ring);
  // Slots of the workspace: two a CTA, the second for a segment that starts in it.
  auto global_slot = [&](int c, int first) {
    return a.part + ((size_t)c * 2 + (c == first ? 1 : 0)) * SLOT;
  };
  struct Group {
    int segid, c0, c1, hcnt;
    __half* rows;  // where the segment's output goes
    float* slot;
  };
  auto group_at = [&](int i0) {
    Group x;
    x.segid = __shfl_sync(0xffffffffu, e_seg, i0);
    x.c0 = __shfl_sync(0xffffffffu, e_c0, i0);
    x.c1 = __shfl_sync(0xffffffffu, e_c1, i0);
    const int b = __shfl_sync(0xffffffffu, e_b, i0), hh = __shfl_sync(0xffffffffu, e_heads, i0);
    x.hcnt = hh & 31;
    x.rows = stream ? a.out + ((size_t)b * a.H + (hh >> 5)) * D : nullptr;
    x.slot = stream ? nullptr : a.part_out + (size_t)x.segid * SLOT;
    return x;
  };
  // Merges the entries of the group that begins with entry i0.
  auto merge_own = [&](int i0, int slice, int hcnt, __half* rows, float* slot) {
    const unsigned from = ~((1u << i0) - 1u);
    const unsigned later = heads & from & (heads - (1u << i0));  // heads of later groups
    const unsigned own = entries & from & (later ? (later & (0u - later)) - 1u : ~0u);
    const int* offs = s_off + __popc(entries & ~from);
    merge_rows<D, GT, true>([&](int k) -> const float* { return smem + offs[k]; }, __popc(own),
                            slice, lane, hcnt, rows, bf, slot, a.status);
  };
  // The shared segments' partials first; while their arrivals are on the way, the others.
  static_assert(2 * kSlices <= WARPS, "one item a warp");
  if (warp < __popc(cross) * kSlices) {
    const int i0 = warp < kSlices ? __ffs(cross) - 1 : 31 - __clz(cross);
    const Group x = group_at(i0);
    merge_own(i0, warp % kSlices, x.hcnt, nullptr, global_slot(cta, x.c0));
  }
  int last = 0;
  if (cross != 0u) {
    // Release the CTA's partials; the arrival that completes a segment's count acquires the
    // others'.
    __syncthreads();
    if (warp == 0 && ((cross >> lane) & 1u))
      last = atom_add_acq_rel_gpu(a.counters + e_seg, 1) == e_c1 - e_c0 ? 1 : 0;
  }
  unsigned todo = heads & ~cross;
  for (int item = WARPS - 1 - warp, n_items = __popc(todo) * kSlices, at = 0; item < n_items;
       item += WARPS) {
    for (; at < item / kSlices; ++at) todo &= todo - 1u;
    const int i0 = __ffs(todo) - 1;
    const Group x = group_at(i0);
    merge_own(i0, item % kSlices, x.hcnt, x.rows, x.slot);
  }
  if (cross == 0u) return;
  if (warp == 0 && ((cross >> lane) & 1u)) s_last[below & cross ? 1 : 0] = last;
  __syncthreads();
  todo = cross;
  for (int x = 0; todo != 0u; ++x, todo &= todo - 1u) {
    if (!s_last[x]) continue;
    const Group gr = group_at(__ffs(todo) - 1);
    const int np = gr.c1 - gr.c0 + 1;
    auto piece = [&](int k) -> const float* { return global_slot(gr.c0 + k, gr.c0); };
    if (np <= 8) {  // two rounds of loads
      const int w = warp - x * kSlices;
      if (w >= 0 && w < kSlices)
        merge_rows<D, GT, false>(piece, np, w, lane, gr.hcnt, gr.rows, bf, gr.slot, a.status);
    } else {
      static_assert(Coop<D, GT, NTHR, 16>::floats(1024) * sizeof(float) <= C::RING, "scratch");
      coop_combine<D, GT, NTHR, 16>(piece, np, gr.hcnt, gr.rows, bf, gr.slot, a.status, smem);
    }
    if (threadIdx.x == 0) a.counters[gr.segid] = 0;
  }
}

// Warps per CTA and ring stages per warp, by head tile (16 heads keep twice the accumulators).
// 64 x 8192 / ragged 256 / 8 x 64-128 K tokens (12/2, 28/4 and 64/8 heads): 41.4 / 108.8 / 169.5 us
// with sixteen warps of two stages (128 registers), 43.2 / 110.1 / 170.9 with twelve of two, 43.3 /
// 110.7 / 171.6 with twelve of three, 43.2 / 119.7 / 184.2 with eight of four. The chosen one spills
// 12 bytes of 5-8 heads, none of fewer. Sixteen heads, 32/2, 64 x 8192: 58.3 with eight warps (250
// registers), 7 more with twelve (spills).
template <int GT> struct Shape;
template <> struct Shape<8> { static constexpr int W = 16, DP = 2; };
template <> struct Shape<16> { static constexpr int W = 8, DP = 4; };

template <int GT, bool PACK>
cudaError_t launch_one(const DecodeFp4Args& a, int grid, cudaStream_t stream) {
  constexpr int W = Shape<GT>::W;
  constexpr int DP = Shape<GT>::DP;
  using C = Tile<128, GT, DP, W>;
  static_assert(C::SMEM + 15 * 1024 + 512 <= 227 * 1024, "shared memory of a launch");
  auto kern = decode_fp4_kernel<128, GT, PACK, DP, W>;
  // The shared-memory opt-in is a per-device function attribute: set it once per device.
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit, std::memory_order_acq_rel);
  }
  kern<<<grid, W * 32, C::SMEM, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

int decode_fp4_warps_per_cta(int gt) { return gt == 8 ? Shape<8>::W : Shape<16>::W; }

cudaError_t launch_decode_fp4(int gt, const DecodeFp4Args& a, int grid, cudaStream_t stream) {
  if (gt != 8) return launch_one<16, false>(a, grid, stream);
  // PACK: the PV of at most four heads leaves half of the MMA's columns empty, which then hold the
  // weights' second parts: 8 MMAs a page instead of 16. 32/8 heads, 64 x 4096 tokens: 69.9 us
  // without, 65.1 with; 8 x 65536: 123.0 and 111.1.
  return a.G <= 4 ? launch_one<8, true>(a, grid, stream) : launch_one<8, false>(a, grid, stream);
}

}  // namespace pa
