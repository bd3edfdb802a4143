// cache_ops.cuh - helpers shared by the long-cache kernels (block_bounds.cu,
// append_batched.cu, block_select.cu, row_attend.cu, evict.cu): thread-block
// clusters, the launch with programmatic dependent launch, 16-byte vectors of
// cache elements, and the radix selection of the k largest keys.
#pragma once

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <string>

#include "gla_common.cuh"
#include "gla_internal.h"

namespace gla {

// One sequence's rows: *n_pos clamped to [0, cap]; a value outside latches
// GLA_ERR_INVALID_ARG in the status word (the call then covers the clamped rows).
__device__ __forceinline__ int32_t clamped_rows(const int32_t* __restrict__ n_pos, int b,
                                                int32_t cap, int32_t* status) {
  const int32_t n = n_pos[b];
  if (n >= 0 && n <= cap) return n;
  if (threadIdx.x == 0) atomicCAS(status, 0, GLA_ERR_INVALID_ARG);
  return n < 0 ? 0 : cap;
}

// True if every pointer starts on a 16-byte boundary and none is null;
// otherwise latches GLA_ERR_ALIGNMENT (or GLA_ERR_INVALID_ARG for a null).
__device__ __forceinline__ bool usable_ptrs(const void* a, const void* b, int32_t* status) {
  if (a == nullptr || b == nullptr) {
    if (threadIdx.x == 0) atomicCAS(status, 0, GLA_ERR_INVALID_ARG);
    return false;
  }
  if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) != 0) {
    if (threadIdx.x == 0) atomicCAS(status, 0, GLA_ERR_ALIGNMENT);
    return false;
  }
  return true;
}

// The same for running weights: floats, so 4-byte alignment is enough.
__device__ __forceinline__ bool usable_weights(const float* a, int32_t* status) {
  if (a != nullptr && (reinterpret_cast<uintptr_t>(a) & 3u) == 0) return true;
  if (threadIdx.x == 0)
    atomicCAS(status, 0, a == nullptr ? GLA_ERR_INVALID_ARG : GLA_ERR_ALIGNMENT);
  return false;
}

// Barrier over the CTAs of a cluster (a plain block barrier for a cluster of
// one).  Every thread of every CTA of the cluster takes part.
__device__ __forceinline__ void cluster_barrier(int S) {
  if (S > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
  } else {
    __syncthreads();
  }
}

// Address, in CTA `rank` of the cluster, of the shared memory object `p` of this CTA.
template <class T>
__device__ __forceinline__ const T* cluster_peer(const T* p, int rank) {
  uint64_t out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<const T*>(out);
}

// Launches `kern` in clusters of S CTAs (grid a multiple of S) behind the
// preceding kernel of the stream (programmatic dependent launch: the kernel
// itself waits for it).  Clusters above 8 CTAs need the opt-in attribute.
template <class... Params, class... Args>
int launch_clusters(void (*kern)(Params...), unsigned grid, int threads, size_t smem, int S,
                    std::atomic<uint64_t>& attr_done, cudaStream_t stream, const char* what,
                    std::string* err, Args... args) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? (1ull << dev) : 0;
  if (!bit || !(attr_done.load(std::memory_order_acquire) & bit)) {
    int optin = 0;
    cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               optin - (int)fa.sharedSizeBytes);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) {
      cudaGetLastError();
      *err = std::string(what) + " attributes: " + cudaGetErrorString(e);
      return GLA_ERR_CUDA;
    }
    if (bit) attr_done.fetch_or(bit, std::memory_order_acq_rel);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)S;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = S > 1 ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    *err = std::string(what) + " launch failed: " + cudaGetErrorString(e);
    return GLA_ERR_CUDA;
  }
  return GLA_OK;
}

// Order-preserving maps of a score to an unsigned key: a larger score has the
// larger key, -0 equals +0, and a NaN has the lowest key, 0.
__device__ __forceinline__ uint64_t order_key(double x) {
  if (x != x) return 0;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0;
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.0f));
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// ---------------------------------------------------------------------------
// The k largest of the keys that the CTAs of a cluster hold together, ties to
// the lowest index.  CTA r holds the n_local keys key(0..n_local-1) of a
// contiguous index range, ranges ascending with the rank; 0 < k < all keys.
//
// Radix selection, 8 bits a pass from the top: every CTA counts the digits of
// its keys that match the prefix found so far, one cluster barrier publishes
// the counts, and every CTA adds all ranks' counts itself (so the ranks agree
// without a second barrier; two count buffers keep a fast rank from clearing
// what a slow one still reads).  A pass whose bin is taken whole ends the
// search.  A second walk writes the chosen indices in ascending order:
// emit(local index, position in the list of all chosen).
// ---------------------------------------------------------------------------
struct SelectScratch {
  uint32_t hist[2][256];
  uint32_t warp_sum[32];
  uint32_t warp_sum2[32];
  uint32_t found[3];       // digit, keys above it, keys in it
  uint32_t counts[2];      // this CTA's keys above / at the threshold
};

template <int THREADS, class Key, class KeyFn, class Emit>
__device__ __forceinline__ void cluster_select(SelectScratch& sh, int S, int rank, int32_t n_local,
                                               uint32_t k, KeyFn key, Emit emit) {
  static_assert(THREADS >= 256 && THREADS % 32 == 0, "one thread per histogram bin");
  constexpr int kBits = sizeof(Key) * 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Key prefix = 0, mask = 0;
  uint32_t need = k;  // of the keys that match the prefix
  bool whole = false;
  int buf = 0;
  for (int shift = kBits - 8; shift >= 0 && !whole; shift -= 8, buf ^= 1) {
    for (int i = tid; i < 256; i += THREADS) sh.hist[buf][i] = 0;
    __syncthreads();
    for (int32_t i0 = 0; i0 < n_local; i0 += THREADS) {
      const int32_t i = i0 + tid;
      Key kv = 0;
      bool in = i < n_local;
      if (in) {
        kv = key(i);
        in = (kv & mask) == prefix;
      }
      const unsigned live = __ballot_sync(0xffffffffu, in);
      if (in) {
        // the top digits of scores are nearly all the same: one add a warp and digit
        const uint32_t d = (uint32_t)(kv >> shift) & 255u;
        const unsigned same = __match_any_sync(live, d);
        if (lane == __ffs(same) - 1) atomicAdd(&sh.hist[buf][d], (uint32_t)__popc(same));
      }
    }
    cluster_barrier(S);
    uint32_t mine = 0;
    if (tid < 256) {
      if (S == 1) {
        mine = sh.hist[buf][255 - tid];
      } else {
        for (int r = 0; r < S; ++r) mine += *cluster_peer(&sh.hist[buf][255 - tid], r);
      }
    }
    // thread t holds bin 255 - t: the inclusive scan counts the keys at or above it
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) sh.warp_sum[warp] = inc;
    __syncthreads();
    if (tid < 256) {
      for (int w = 0; w < warp; ++w) inc += sh.warp_sum[w];
      if (inc - mine < need && need <= inc) {
        sh.found[0] = 255 - tid;
        sh.found[1] = inc - mine;
        sh.found[2] = mine;
      }
    }
    __syncthreads();
    need -= sh.found[1];
    whole = sh.found[2] == need;
    prefix |= (Key)sh.found[0] << shift;
    mask |= (Key)255 << shift;
  }
  // chosen: above the prefix, or at it (all of those if `whole`, else the first `need`)
  uint32_t above = 0, at = 0;
  for (int32_t i = tid; i < n_local; i += THREADS) {
    const Key kv = key(i) & mask;
    above += kv > prefix;
    at += kv == prefix;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    above += __shfl_xor_sync(0xffffffffu, above, o);
    at += __shfl_xor_sync(0xffffffffu, at, o);
  }
  if (lane == 0) {
    sh.warp_sum[warp] = above;
    sh.warp_sum2[warp] = at;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t a = 0, e = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      a += sh.warp_sum[w];
      e += sh.warp_sum2[w];
    }
    sh.counts[0] = a;
    sh.counts[1] = e;
  }
  cluster_barrier(S);
  uint32_t out = 0, at_before = 0;
  for (int r = 0; r < rank; ++r) {
    const uint32_t* c = S == 1 ? sh.counts : cluster_peer(sh.counts, r);
    const uint32_t a = c[0], e = c[1];
    const uint32_t room = need > at_before ? need - at_before : 0;
    out += a + (e < room ? e : room);
    at_before += e;
  }
  for (int32_t i0 = 0; i0 < n_local; i0 += THREADS) {
    const int32_t i = i0 + tid;
    Key kv = 0;
    if (i < n_local) kv = key(i) & mask;
    const bool gt = i < n_local && kv > prefix, eq = i < n_local && kv == prefix;
    const unsigned beq = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) sh.warp_sum2[warp] = __popc(beq);
    __syncthreads();
    uint32_t eq_pos = at_before + __popc(beq & ((1u << lane) - 1)), eq_all = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      const uint32_t x = sh.warp_sum2[w];
      if (w < warp) eq_pos += x;
      eq_all += x;
    }
    const bool take = gt || (eq && eq_pos < need);
    const unsigned bt = __ballot_sync(0xffffffffu, take);
    if (lane == 0) sh.warp_sum[warp] = __popc(bt);
    __syncthreads();
    uint32_t pos = out + __popc(bt & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      const uint32_t x = sh.warp_sum[w];
      if (w < warp) pos += x;
      all += x;
    }
    if (take) emit(i, pos);
    out += all;
    at_before += eq_all;
  }
  cluster_barrier(S);  // no CTA leaves while another still reads its counts
}

// Contiguous share [lo, hi) of n items for CTA `rank` of S.
GLA_HD void share_of(int32_t n, int S, int rank, int32_t* lo, int32_t* hi) {
  const int32_t per = (n + S - 1) / S;
  const int64_t a = (int64_t)per * rank;
  *lo = a < n ? (int32_t)a : n;
  *hi = a + per < n ? (int32_t)(a + per) : n;
}

}  // namespace gla
