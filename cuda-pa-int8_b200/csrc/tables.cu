// Block tables, slot maps and positions of a serving step, built on the GPU from the requests'
// lengths, so that a step (or a captured graph of steps) needs no lengths on the host.
//
// The free blocks are a stack, free_blocks[0 .. free_count). Releasing pushes the blocks of
// finished sequences, in sequence order and by block index; extending pops one block for every
// block a sequence grows by, in sequence order, so the result does not depend on timing.
//
// A sequence's place (its first token in the packed batch, its first popped or pushed block) is
// an exclusive prefix sum over the sequences before it. Every CTA takes a range of tokens (or
// of pushed blocks) and runs the same scan over the lengths, 1024 sequences at a time in shared
// memory, searching each chunk for its own items; the lengths are a few KB and stay in L2, so
// the repeated scan costs less than a second launch would. Nothing is changed unless the whole
// call fits: a first scan of the totals decides that, in every CTA alike. The lengths and the
// count may be updated in place: the CTAs are one cluster, and its first one writes them after a
// cluster barrier, when all have read. (A counter in the workspace would allow more CTAs, but
// two captured graphs that share a workspace would share the counter; eight SMs write the maps
// of 64 K tokens as fast as the launch itself.)

#include "pa_common.cuh"
#include "pa_internal.h"

namespace pa {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Inclusive sums over the block of two counts per thread; returns the block's totals in tot.
struct Pair {
  long long a, b;
};

__device__ __forceinline__ Pair shfl_up(Pair v, int o) {
  return Pair{__shfl_up_sync(0xffffffffu, v.a, o), __shfl_up_sync(0xffffffffu, v.b, o)};
}

__device__ __forceinline__ Pair block_scan(Pair v, Pair* s_warp, Pair& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Pair u = shfl_up(v, o);
    if (lane >= o) {
      v.a += u.a;
      v.b += u.b;
    }
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    Pair w = s_warp[lane];  // kWarps == 32
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Pair u = shfl_up(w, o);
      if (lane >= o) {
        w.a += u.a;
        w.b += u.b;
      }
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  if (warp > 0) {
    v.a += s_warp[warp - 1].a;
    v.b += s_warp[warp - 1].b;
  }
  tot = s_warp[kWarps - 1];
  __syncthreads();
  return v;
}

__device__ __forceinline__ int ceil_div(int a, int b) { return (int)(((unsigned)a + b - 1) / (unsigned)b); }

// Largest i in [0, n) with s[i] <= x (s ascending, s[0] <= x).
__device__ __forceinline__ int find(const long long* s, int n, long long x) {
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

__global__ void __launch_bounds__(kThreads) release_kernel(const TableArgs a) {
  __shared__ long long s_off[kThreads];
  __shared__ Pair s_warp[kWarps];
  const int tid = threadIdx.x;
  const int cap = a.max_blocks * a.bs;
  const int top = __ldg(a.free_count);

  int err = 0;
  long long total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) {
      if (top < 0 || top + total > a.pool) err |= PA_ERR_FREE_BLOCKS;
      if (__syncthreads_or(err) != 0) break;
    }
    long long carry = 0;
    for (int base = 0; base < a.S; base += kThreads) {
      const int i = base + tid;
      int n = 0;
      if (i < a.S && __ldg(a.flags + i) != 0) {
        const int c = __ldg(a.lens + i);
        if (c < 0 || c > cap) {
          err |= PA_ERR_CONTEXT_RANGE;
        } else {
          n = ceil_div(c, a.bs);
        }
      }
      Pair tot;
      const Pair v = block_scan(Pair{n, 0}, s_warp, tot);
      if (pass == 1 && tot.a > 0) {
        s_off[tid] = carry + v.a - n;
        __syncthreads();
        const int cnt = min(kThreads, a.S - base);
        // Pushed block r of the chunk: CTAs take them in turn, a thread each.
        for (long long r = carry + (long long)blockIdx.x * kThreads + tid; r < carry + tot.a;
             r += (long long)gridDim.x * kThreads) {
          const int q = find(s_off, cnt, r);
          const int j = (int)(r - s_off[q]);
          a.free_blocks[top + r] = __ldg(a.table + (size_t)(base + q) * a.max_blocks + j);
        }
        __syncthreads();
      }
      carry += tot.a;
    }
    total = carry;
  }
  const bool ok = __syncthreads_or(err) == 0;
  if (!ok && blockIdx.x == 0 && err != 0) flag_error(a.status, err);
  cluster_barrier();
  if (blockIdx.x != 0) return;
  for (int i = tid; i < a.S; i += kThreads) {
    const int c = a.lens[i];
    a.lens_out[i] = ok && a.flags[i] != 0 ? 0 : c;
  }
  if (tid == 0) *a.count_out = ok ? (int)(top + total) : top;
}

__global__ void __launch_bounds__(kThreads) extend_kernel(const TableArgs a) {
  __shared__ long long s_tok[kThreads], s_blk[kThreads];
  __shared__ int s_len[kThreads];
  __shared__ Pair s_warp[kWarps];
  const int tid = threadIdx.x;
  const long long cap = (long long)a.max_blocks * a.bs;
  const int top = __ldg(a.free_count);
  const long long stride = (long long)gridDim.x * kThreads;
  const long long me = (long long)blockIdx.x * kThreads + tid;

  int err = 0;
  long long tokens = 0, blocks = 0;
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1) {
      if (tokens > a.max_tokens) err |= PA_ERR_TOKENS;
      if (top < 0 || top > a.pool || blocks > top) err |= PA_ERR_FREE_BLOCKS;
      if (__syncthreads_or(err) != 0) break;
    }
    Pair carry{0, 0};
    for (int base = 0; base < a.S; base += kThreads) {
      const int i = base + tid;
      int c = 0, add = 0, need = 0;
      if (i < a.S) {
        c = __ldg(a.lens + i);
        add = __ldg(a.flags + i);
        if (c < 0 || add < 0 || (long long)c + add > cap) {
          err |= PA_ERR_CONTEXT_RANGE;
          c = add = 0;
        }
        need = ceil_div(c + add, a.bs) - ceil_div(c, a.bs);
      }
      Pair tot;
      const Pair v = block_scan(Pair{add, need}, s_warp, tot);
      if (pass == 1) {
        s_tok[tid] = carry.a + v.a - add;
        s_blk[tid] = carry.b + v.b - need;
        s_len[tid] = c;
        if (blockIdx.x == 0 && i < a.S) a.starts[i] = (int)(carry.a + v.a - add);
        __syncthreads();
        const int cnt = min(kThreads, a.S - base);
        // The CTA's tokens (every gridDim-th run of kThreads) that lie in this chunk.
        long long t = me;
        if (t < carry.a) t += (carry.a - t + stride - 1) / stride * stride;
        for (; t < carry.a + tot.a; t += stride) {
          const int q = find(s_tok, cnt, t);
          const int len = s_len[q];
          const int pos = len + (int)(t - s_tok[q]);
          const int col = (int)((unsigned)pos / (unsigned)a.bs);
          const int off = pos - col * a.bs;
          const int had = ceil_div(len, a.bs);
          int* cell = a.table + (size_t)(base + q) * a.max_blocks + col;
          int blk;
          if (col >= had) {
            blk = __ldg(a.free_blocks + (top - 1 - (s_blk[q] + col - had)));
            if (off == 0) *cell = blk;  // each new block's first token is new
          } else {
            blk = *cell;
          }
          const bool good = blk >= 0 && blk < a.NB;
          if (!good) flag_error(a.status, PA_ERR_BLOCK_ID);
          a.slots[t] = good ? blk * a.bs + off : -1;
          a.positions[t] = pos;
        }
        __syncthreads();
      }
      carry.a += tot.a;
      carry.b += tot.b;
    }
    tokens = carry.a;
    blocks = carry.b;
  }
  const bool ok = __syncthreads_or(err) == 0;
  if (!ok && blockIdx.x == 0 && err != 0) flag_error(a.status, err);
  for (long long t = me; t < a.max_tokens; t += stride) {
    if (ok && t < tokens) continue;
    a.slots[t] = -1;
    a.positions[t] = -1;
  }
  if (blockIdx.x == 0) {
    if (!ok)
      for (int i = tid; i < a.S; i += kThreads) a.starts[i] = 0;
    if (tid == 0) a.starts[a.S] = ok ? (int)tokens : 0;
  }
  cluster_barrier();
  if (blockIdx.x != 0) return;
  for (int i = tid; i < a.S; i += kThreads) {
    const int c = a.lens[i];
    a.lens_out[i] = ok ? c + a.flags[i] : c;
  }
  if (tid == 0) *a.count_out = ok ? (int)(top - blocks) : top;
}

}  // namespace

namespace {
// One cluster of up to eight CTAs (the portable limit), for at most `items` items.
template <typename K>
cudaError_t launch_cluster(K kern, const TableArgs& a, long long items, cudaStream_t st) {
  unsigned n = 1;
  while (n < 8 && (long long)n * kThreads < items) n *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n);
  cfg.blockDim = dim3(kThreads);
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
  // The pushed blocks are not known on the host: at most max_blocks a sequence.
  return launch_cluster(release_kernel, a, (long long)a.S * a.max_blocks, st);
}

cudaError_t launch_extend(const TableArgs& a, cudaStream_t st) {
  return launch_cluster(extend_kernel, a, a.max_tokens, st);
}

}  // namespace pa
