// Block tables, slot maps and positions of a serving step, built on the GPU from the requests'
// lengths, so that a step (or a captured graph of steps) needs no lengths on the host.
//
// The free blocks are a stack, free_blocks[0 .. free_count). Releasing pushes the blocks of
// finished sequences, in sequence order and by block index; extending pops one block for every
// block a sequence grows by, in sequence order, so the result does not depend on timing.
//
// A sequence's place (its first token in the packed batch, its first popped or pushed block) is
// an exclusive prefix sum over the sequences before it. Every CTA runs the same scan over the
// lengths, a chunk of sequences (one a thread) at a time in shared memory, and searches it for
// its own items; the lengths are a few KB and stay in L2, so the repeated scan costs less than a
// second launch would. Nothing is changed unless the whole call fits: the totals of a first scan
// decide that, in every CTA alike (with one chunk, its scan is kept). The lengths and the count
// may be updated in place: the CTAs are one cluster, and its first one writes them after a
// cluster barrier, when all have read. (A counter in the workspace would allow more CTAs, but two
// captured graphs that share a workspace would share the counter.)
//
// Both are bound by latency, a launch and a chain of dependent loads and barriers. Graph replay of
// the pair: 10.4 us for 256 requests of one new token each, 15.8 us for 64 requests that grow by
// up to 65536 tokens in all; their bytes would take under 0.1 us. So small calls run in small
// CTAs, and a thread takes four neighbouring tokens, which nearly always share their sequence and
// block.

#include "pa_common.cuh"
#include "pa_internal.h"

namespace pa {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kTokens = 4;  // neighbouring tokens of a thread

// Two counts per sequence, saturating at 2^31 - 1 (which every caller's limit refuses).
struct Pair {
  unsigned a, b;
};
constexpr unsigned kSaturated = 0x7fffffffu;
__device__ __forceinline__ unsigned sat_add(unsigned x, unsigned y) {
  return min(x + y, kSaturated);  // both at most 2^31 - 1: no wrap
}
__device__ __forceinline__ Pair sat_add(Pair x, Pair y) {
  return Pair{sat_add(x.a, y.a), sat_add(x.b, y.b)};
}

// Inclusive sums over the block; the block's totals in tot. s_warp: 32 entries.
__device__ __forceinline__ Pair block_scan(Pair v, Pair* s_warp, Pair& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  auto warp_scan = [&](Pair x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Pair u{__shfl_up_sync(0xffffffffu, x.a, o), __shfl_up_sync(0xffffffffu, x.b, o)};
      if (lane >= o) x = sat_add(x, u);
    }
    return x;
  };
  v = warp_scan(v);
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  // Every warp scans the warps' totals for itself: one barrier less.
  const Pair w = warp_scan(lane < warps ? s_warp[lane] : Pair{0u, 0u});
  tot = Pair{__shfl_sync(0xffffffffu, w.a, 31), __shfl_sync(0xffffffffu, w.b, 31)};
  const Pair before{__shfl_sync(0xffffffffu, w.a, max(warp - 1, 0)),
                    __shfl_sync(0xffffffffu, w.b, max(warp - 1, 0))};
  if (warp > 0) v = sat_add(v, before);
  __syncthreads();  // s_warp may be used again
  return v;
}

__device__ __forceinline__ int ceil_div(int a, int b) {
  return (int)(((unsigned)a + (unsigned)b - 1u) / (unsigned)b);
}

// Largest i in [0, n) with s[i] <= x (s ascending, s[0] <= x).
__device__ __forceinline__ int find(const unsigned* s, int n, unsigned x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// All CTAs of the launch (one cluster) wait for each other.
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}

__global__ void __launch_bounds__(kMaxThreads) release_kernel(const TableArgs a) {
  __shared__ unsigned s_off[kMaxThreads];
  __shared__ Pair s_warp[32];
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int cap = a.max_blocks * a.bs;
  const int top = *a.free_count;
  const bool single = a.S <= nthr;

  int err = 0;
  unsigned total = 0;
  int kept = 0, was = 0;  // one chunk: this thread's sequence's new and old length
  bool ok = false;
  for (int pass = single ? 1 : 0; pass < 2; ++pass) {
    unsigned carry = 0;
    for (int base = 0; base < a.S || base == 0; base += nthr) {
      const int i = base + tid;
      int n = 0;
      if (i < a.S) {
        const int f = a.flags[i], c = a.lens[i];
        kept = f != 0 ? 0 : c;
        was = c;
        if (f != 0) {
          if (c < 0 || c > cap) {
            err |= PA_ERR_CONTEXT_RANGE;
          } else {
            n = ceil_div(c, a.bs);
          }
        }
      }
      Pair tot;
      const Pair v = block_scan(Pair{(unsigned)n, 0u}, s_warp, tot);
      if (single) total = tot.a;
      if (pass == 1) {
        if (base == 0) {  // the totals are known: does the call fit?
          if (top < 0 || (long long)top + total > a.pool || total == kSaturated)
            err |= PA_ERR_FREE_BLOCKS;
          ok = __syncthreads_or(err) == 0;
          if (!ok) break;
        }
        if (tot.a > 0) {
          s_off[tid] = carry + v.a - n;
          __syncthreads();
          const int cnt = min(nthr, a.S - base);
          // Pushed block r of the chunk: CTAs take them in turn, a thread each.
          for (unsigned r = carry + blockIdx.x * nthr + tid; r < carry + tot.a;
               r += gridDim.x * nthr) {
            const int q = find(s_off, cnt, r);
            const int j = (int)(r - s_off[q]);
            a.free_blocks[top + (int)r] =
                __ldg(a.table + (size_t)(base + q) * a.max_blocks + j);
          }
          __syncthreads();
        }
      }
      carry = sat_add(carry, tot.a);
    }
    if (pass == 0) total = carry;
  }
  if (!ok && blockIdx.x == 0 && err != 0) flag_error(a.status, err);
  cluster_barrier();
  if (blockIdx.x != 0) return;
  if (single) {
    if (tid < a.S) a.lens_out[tid] = ok ? kept : was;
  } else {
    for (int i = tid; i < a.S; i += nthr) {
      const int c = a.lens[i];
      a.lens_out[i] = ok && a.flags[i] != 0 ? 0 : c;
    }
  }
  if (tid == 0) *a.count_out = ok ? top + (int)total : top;
}

__global__ void __launch_bounds__(kMaxThreads) extend_kernel(const TableArgs a) {
  __shared__ unsigned s_tok[kMaxThreads], s_blk[kMaxThreads];
  __shared__ int s_len[kMaxThreads];
  __shared__ Pair s_warp[32];
  const int tid = threadIdx.x, nthr = blockDim.x;
  const long long cap = (long long)a.max_blocks * a.bs;
  const int top = *a.free_count;
  const unsigned stride = gridDim.x * nthr * kTokens;
  const unsigned me = (blockIdx.x * nthr + tid) * kTokens;
  const bool single = a.S <= nthr;

  int err = 0;
  Pair total{0u, 0u};
  int kept = 0, was = 0;  // one chunk: this thread's sequence's new and old length
  bool ok = false;
  for (int pass = single ? 1 : 0; pass < 2; ++pass) {
    Pair carry{0u, 0u};
    for (int base = 0; base < a.S || base == 0; base += nthr) {
      const int i = base + tid;
      int c = 0, add = 0, need = 0;
      if (i < a.S) {
        c = a.lens[i];
        add = a.flags[i];
        was = c;
        kept = (int)((unsigned)c + (unsigned)add);
        if (c < 0 || add < 0 || (long long)c + add > cap) {
          err |= PA_ERR_CONTEXT_RANGE;
          c = add = 0;
        }
        need = ceil_div(c + add, a.bs) - ceil_div(c, a.bs);
      }
      Pair tot;
      const Pair v = block_scan(Pair{(unsigned)add, (unsigned)need}, s_warp, tot);
      if (single) total = tot;
      if (pass == 1) {
        if (base == 0) {
          if (total.a == kSaturated || total.a > (unsigned)a.max_tokens) err |= PA_ERR_TOKENS;
          if (top < 0 || top > a.pool || total.b > (unsigned)max(top, 0))
            err |= PA_ERR_FREE_BLOCKS;
          ok = __syncthreads_or(err) == 0;
          if (!ok) break;
        }
        s_tok[tid] = carry.a + v.a - add;
        s_blk[tid] = carry.b + v.b - need;
        s_len[tid] = c;
        if (blockIdx.x == 0 && i < a.S) a.starts[i] = (int)(carry.a + v.a - add);
        __syncthreads();
        const int cnt = min(nthr, a.S - base);
        const unsigned end = carry.a + tot.a;
        // This thread's runs of four tokens that reach into the chunk.
        unsigned t0 = me;
        if (t0 + kTokens <= carry.a)
          t0 += (carry.a - t0 - kTokens) / stride * stride + stride;
        for (; t0 < end; t0 += stride) {
          int q = -1, last_col = -1, blk = 0;
#pragma unroll
          for (int e = 0; e < kTokens; ++e) {
            const unsigned t = t0 + e;
            if (t < carry.a || t >= end) continue;
            if (q < 0 || (q + 1 < cnt && s_tok[q + 1] <= t)) {
              q = find(s_tok, cnt, t);
              last_col = -1;
            }
            const int len = s_len[q];
            const int pos = len + (int)(t - s_tok[q]);
            const int col = (int)((unsigned)pos / (unsigned)a.bs);
            const int off = pos - col * a.bs;
            if (col != last_col) {
              last_col = col;
              const int had = ceil_div(len, a.bs);
              int* cell = a.table + (size_t)(base + q) * a.max_blocks + col;
              if (col >= had) {
                blk = __ldg(a.free_blocks + (top - 1 - ((int)s_blk[q] + col - had)));
                if (off == 0) *cell = blk;  // each new block's first token is new
              } else {
                blk = *cell;
              }
            }
            const bool good = blk >= 0 && blk < a.NB;
            if (!good) flag_error(a.status, PA_ERR_BLOCK_ID);
            a.slots[t] = good ? blk * a.bs + off : -1;
            a.positions[t] = pos;
          }
        }
        __syncthreads();
      }
      carry = sat_add(carry, tot);
    }
    if (pass == 0) total = carry;
  }
  if (!ok && blockIdx.x == 0 && err != 0) flag_error(a.status, err);
  // Padding: everything past the last token, or all of a refused call.
  const unsigned tokens = ok ? total.a : 0u;
  for (unsigned t = tokens + blockIdx.x * nthr + tid; t < (unsigned)a.max_tokens;
       t += gridDim.x * nthr) {
    a.slots[t] = -1;
    a.positions[t] = -1;
  }
  if (blockIdx.x == 0) {
    if (!ok)
      for (int i = tid; i < a.S; i += nthr) a.starts[i] = 0;
    if (tid == 0) a.starts[a.S] = (int)tokens;
  }
  cluster_barrier();
  if (blockIdx.x != 0) return;
  if (single) {
    if (tid < a.S) a.lens_out[tid] = ok ? kept : was;
  } else {
    for (int i = tid; i < a.S; i += nthr) {
      const int c = a.lens[i];
      a.lens_out[i] = ok ? c + a.flags[i] : c;
    }
  }
  if (tid == 0) *a.count_out = ok ? top - (int)total.b : top;
}

// One cluster of up to eight CTAs (the portable limit) for at most `items` items of `per` to a
// thread; a CTA has as many threads as the sequences or its items can use.
template <typename K>
cudaError_t launch_cluster(K kern, const TableArgs& a, long long items, int per,
                           cudaStream_t st) {
  const long long want = (items + per - 1) / per > a.S ? (items + per - 1) / per : a.S;
  int threads = 128;
  while (threads < kMaxThreads && threads < want) threads *= 2;
  unsigned n = 1;
  while (n < 8 && (long long)n * threads * per < items) n *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

cudaError_t launch_release(const TableArgs& a, cudaStream_t st) {
  // The pushed blocks are not known on the host: at most max_blocks a sequence, rarely
  // more than an eighth of that.
  return launch_cluster(release_kernel, a, (long long)a.S * a.max_blocks, 8, st);
}

cudaError_t launch_extend(const TableArgs& a, cudaStream_t st) {
  return launch_cluster(extend_kernel, a, a.max_tokens, kTokens, st);
}

}  // namespace pa
