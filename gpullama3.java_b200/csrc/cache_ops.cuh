// cache_ops.cuh - helpers shared by the long-cache kernels (block_bounds.cu,
// append_batched.cu, block_select.cu, row_attend.cu, evict.cu): thread-block
// clusters, the launch with programmatic dependent launch, 16-byte vectors of
// cache elements, and the radix selection of the k largest keys.
#pragma once

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
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

// The same barrier in two halves, for work between them; a cluster of one passes.
__device__ __forceinline__ void cluster_arrive(int S) {
  if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait(int S) {
  if (S > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address, in CTA `rank` of the cluster, of the shared memory object `p` of this CTA.
template <class T>
__device__ __forceinline__ const T* cluster_peer(const T* p, int rank) {
  uint64_t out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<const T*>(out);
}

// What a kernel's cluster launches need once a device: raised limits (shared
// memory, clusters above 8 CTAs), and how many clusters of 1, 2, 4, 8 and 16 CTAs
// the device holds at once (a cluster lies in one GPC, so fewer than its SMs
// suggest: 7 of 16 CTAs at one CTA an SM of 148).
struct ClusterKernel {
  std::atomic<uint64_t> attr_done{0};  // bit d: device d
  std::atomic<int> held[5] = {};       // 0: not asked yet (all devices are alike)
};

template <class... Params>
int prepare_clusters(void (*kern)(Params...), ClusterKernel& ck, const char* what,
                     std::string* err) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? (1ull << dev) : 0;
  if (bit && (ck.attr_done.load(std::memory_order_acquire) & bit)) return GLA_OK;
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
  if (bit) ck.attr_done.fetch_or(bit, std::memory_order_acq_rel);
  return GLA_OK;
}

inline void cluster_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute (&attr)[2], unsigned grid,
                           int threads, size_t smem, int S, cudaStream_t stream) {
  cfg->gridDim = dim3(grid);
  cfg->blockDim = dim3((unsigned)threads);
  cfg->dynamicSmemBytes = smem;
  cfg->stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)S;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg->attrs = attr;
  cfg->numAttrs = S > 1 ? 2 : 1;
}

// Clusters of S CTAs that the device holds at once (a guess if it cannot say).
template <class... Params>
int clusters_held(void (*kern)(Params...), ClusterKernel& ck, int threads, size_t smem, int S,
                  const DeviceInfo& dev) {
  int slot = 0;
  while ((1 << slot) < S) ++slot;
  int n = ck.held[slot].load(std::memory_order_relaxed);
  if (n > 0) return n;
  std::string err;
  if (prepare_clusters(kern, ck, "cluster", &err) != GLA_OK) return std::max(1, dev.sms / S);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cluster_config(&cfg, attr, (unsigned)S, threads, smem, S, nullptr);
  cfg.attrs = attr + 1;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = std::max(1, dev.sms / S);
  }
  ck.held[slot].store(n, std::memory_order_relaxed);
  return n;
}

// Launches `kern` in clusters of S CTAs (grid a multiple of S) behind the
// preceding kernel of the stream (programmatic dependent launch: the kernel
// itself waits for it).
template <class... Params, class... Args>
int launch_clusters(void (*kern)(Params...), unsigned grid, int threads, size_t smem, int S,
                    ClusterKernel& ck, cudaStream_t stream, const char* what, std::string* err,
                    Args... args) {
  const int rc = prepare_clusters(kern, ck, what, err);
  if (rc != GLA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cluster_config(&cfg, attr, grid, threads, smem, S, stream);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    *err = std::string(what) + " launch failed: " + cudaGetErrorString(e);
    return GLA_ERR_CUDA;
  }
  return GLA_OK;
}

// Bulk copy global -> shared (bulk_g2s without its evict-first hint: data that is
// read again, by the other queries of a chunk or at the next token).
__device__ __forceinline__ void bulk_g2s_keep(void* dst, const void* src, uint32_t bytes,
                                              uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
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
// The score of an FP32 key; keys that are no score's are the infinities.
__device__ __forceinline__ float key_score(uint32_t key) {
  if (key == 0) return -INFINITY;
  if (key == ~0u) return INFINITY;
  return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key);
}

// ---------------------------------------------------------------------------
// The k largest of the keys that the CTAs of a cluster hold together, ties to
// the lowest index.  CTA r holds the n_local keys key(0..n_local-1) of a
// contiguous index range, ranges ascending with the rank; 0 < k < all keys.
// The keys are walked once a pass, and the walks are bound by instructions: 32-bit
// keys in shared memory (SharedKeys) are taken four at a time.
//
// find_threshold: radix selection, 8 bits a pass over the range [kmin, kmax] of the
// keys (key_range finds it: full-width digits would put nearly all scores into a few
// bins first and take more passes).  Every CTA counts the digits of its keys in the range found so far, one cluster
// barrier publishes the counts, and every CTA adds all ranks' counts itself (so the
// ranks agree without a second barrier; two count buffers keep a fast rank from
// clearing what a slow one still reads).  A pass whose bin is taken whole ends the
// search.
// emit_chosen: each warp, which owns a contiguous share of the CTA's keys, counts
// what it holds above and at the threshold, and after one more barrier writes its
// chosen indices, so the list ascends with no barrier inside:
// emit(local index, position in the list of all chosen).
// ---------------------------------------------------------------------------
// 32-bit keys in shared memory, 16-byte aligned and filled up with keys of 0 to a
// multiple of 4.  (A filling key ranks behind every real one: 0 is the lowest and it
// has the highest index of its CTA; walks that break ties by index leave it out.)
struct SharedKeys {
  static constexpr bool kQuads = true;
  const uint32_t* p;
  __device__ __forceinline__ uint32_t operator()(int32_t i) const { return p[i]; }
  __device__ __forceinline__ uint4 quad(int32_t q) const {
    return reinterpret_cast<const uint4*>(p)[q];
  }
};
__device__ __forceinline__ void fill_up_keys(uint32_t* p, int32_t n) {
  if (threadIdx.x < 4 && (n & 3) + (int)threadIdx.x < 4 && (n & 3)) p[n + threadIdx.x] = 0;
}
// Any other keys: one at a time.
template <class F>
struct KeysBy {
  static constexpr bool kQuads = false;
  F f;
  __device__ __forceinline__ auto operator()(int32_t i) const { return f(i); }
};
template <class F>
__device__ __forceinline__ KeysBy<F> keys_by(F f) {
  return KeysBy<F>{f};
}

constexpr int kSelectWarps = 32;  // at most
struct SelectScratch {
  uint32_t hist[2][256];
  uint32_t warp_sum[8];
  uint32_t found[3];                 // digit, keys above it, keys in it
  uint32_t above[kSelectWarps];      // of each warp's share: keys above the threshold
  uint32_t at[kSelectWarps];         // and at it
  uint32_t counts[2];                // of the CTA's share
  uint32_t low[kSelectWarps], high[kSelectWarps];  // each warp's smallest and largest key
};

__device__ __forceinline__ int bit_count(uint32_t x) { return 32 - __clz((int)x); }
__device__ __forceinline__ int bit_count(uint64_t x) { return 64 - __clzll((long long)x); }

template <class Key>
struct Threshold {
  Key lo, span;      // chosen: keys above lo + span, and of those in [lo, lo + span] ...
  uint32_t need;     // ... the first `need`
  bool whole;        // which are all of them
  __device__ __forceinline__ bool at(Key k) const { return k >= lo && k - lo <= span; }
  __device__ __forceinline__ bool above(Key k) const { return k >= lo && k - lo > span; }
};

// The smallest and the largest of the cluster's keys from those of each thread.
template <int THREADS>
__device__ __forceinline__ void key_range(SelectScratch& sh, int S, uint32_t* kmin, uint32_t* kmax) {
  constexpr int W = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t lo = __reduce_min_sync(0xffffffffu, *kmin), hi = __reduce_max_sync(0xffffffffu, *kmax);
  if (lane == 0) {
    sh.low[warp] = lo;
    sh.high[warp] = hi;
  }
  cluster_barrier(S);
  lo = ~0u;
  hi = 0;
  if (lane < W) {
#pragma unroll 4
    for (int r = 0; r < S; ++r) {
      lo = min(lo, S == 1 ? sh.low[lane] : *cluster_peer(&sh.low[lane], r));
      hi = max(hi, S == 1 ? sh.high[lane] : *cluster_peer(&sh.high[lane], r));
    }
  }
  *kmin = __reduce_min_sync(0xffffffffu, lo);
  *kmax = __reduce_max_sync(0xffffffffu, hi);
}

template <int THREADS, class Key, class KeyFn>
__device__ __forceinline__ Threshold<Key> find_threshold(SelectScratch& sh, int S, int32_t n_local,
                                                         uint32_t k, Key kmin, Key kmax,
                                                         KeyFn key) {
  static_assert(THREADS >= 256 && THREADS % 32 == 0, "one thread per histogram bin");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t need = k;  // of the keys in the range
  bool whole = false;
  int buf = 0;
  for (int i = tid; i < 512; i += THREADS) (&sh.hist[0][0])[i] = 0;
  __syncthreads();
  Key base = kmin, span = kmax - kmin;  // the range is [base, base + span]
  int shift = bit_count(span) > 8 ? bit_count(span) - 8 : 0;
  for (;; buf ^= 1) {
    // (a key below base wraps to a distance beyond span)
    auto count = [&](Key kv) {
      const Key d = kv - base;
      if (d <= span) atomicAdd(&sh.hist[buf][(uint32_t)(d >> shift)], 1u);
    };
    if constexpr (KeyFn::kQuads) {
#pragma unroll 2
      for (int32_t q = tid; q < (n_local + 3) / 4; q += THREADS) {
        const uint4 kv = key.quad(q);
        count(kv.x);
        count(kv.y);
        count(kv.z);
        count(kv.w);
      }
    } else {
#pragma unroll 4
      for (int32_t i = tid; i < n_local; i += THREADS) count(key(i));
    }
    cluster_barrier(S);
    uint32_t mine = 0;
    if (tid < 256) {
      if (S == 1) {
        mine = sh.hist[buf][255 - tid];
      } else {
#pragma unroll 4
        for (int r = 0; r < S; ++r) mine += *cluster_peer(&sh.hist[buf][255 - tid], r);
      }
      sh.hist[buf ^ 1][tid] = 0;  // every rank has read it: it did so before the barrier
    }
    // thread t holds bin 255 - t: the inclusive scan counts the keys at or above it
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (tid < 256 && lane == 31) sh.warp_sum[warp] = inc;
    __syncthreads();
    if (tid < 256) {
#pragma unroll
      for (int w = 0; w < 7; ++w) inc += w < warp ? sh.warp_sum[w] : 0;
      if (inc - mine < need && need <= inc) {
        sh.found[0] = 255 - tid;
        sh.found[1] = inc - mine;
        sh.found[2] = mine;
      }
    }
    __syncthreads();
    need -= sh.found[1];
    whole = sh.found[2] == need;
    base += (Key)sh.found[0] << shift;
    // the last digit's range ends at kmax: past the type's end it would hold the lowest
    // keys too, the filling ones among them
    span = ((Key)1 << shift) - 1;
    span = span < kmax - base ? span : kmax - base;
    if (whole || shift == 0) break;
    shift = shift > 8 ? shift - 8 : 0;
  }
  return Threshold<Key>{base, span, need, whole};
}

template <int THREADS, class Key, class KeyFn, class Emit>
__device__ __forceinline__ void emit_chosen(SelectScratch& sh, int S, int rank, int32_t n_local,
                                            const Threshold<Key>& th, KeyFn key, Emit emit) {
  constexpr int W = THREADS / 32;
  static_assert(W <= kSelectWarps, "per-warp counts");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t need = th.need;
  // this warp's share of the CTA's keys: whole warps of (four) keys, contiguous
  constexpr int kStep = KeyFn::kQuads ? 128 : 32;
  const int32_t share = ((n_local + W * kStep - 1) / (W * kStep)) * kStep;
  const int32_t w_lo = min(warp * share, n_local), w_hi = min(w_lo + share, n_local);
  const bool fast = KeyFn::kQuads && th.whole;
  uint32_t above = 0, at = 0;
  if constexpr (KeyFn::kQuads) {
    if (fast && w_lo < w_hi) {  // (an empty share starts at n_local, inside a quad)
#pragma unroll 4
      for (int32_t q = w_lo / 4 + lane; q < (w_hi + 3) / 4; q += 32) {
        const uint4 kv = key.quad(q);
        above += (kv.x >= th.lo) + (kv.y >= th.lo) + (kv.z >= th.lo) + (kv.w >= th.lo);
      }
    }
  }
  if (!fast) {
#pragma unroll 4
    for (int32_t i = w_lo + lane; i < w_hi; i += 32) {
      const Key kv = key(i);
      above += th.above(kv);
      at += th.at(kv);
    }
  }
  above = __reduce_add_sync(0xffffffffu, above);
  at = __reduce_add_sync(0xffffffffu, at);
  if (lane == 0) {
    sh.above[warp] = above;
    sh.at[warp] = at;
  }
  __syncthreads();
  if (S > 1) {
    if (tid == 0) {
      uint32_t a = 0, e = 0;
      for (int w = 0; w < W; ++w) {
        a += sh.above[w];
        e += sh.at[w];
      }
      sh.counts[0] = a;
      sh.counts[1] = e;
    }
    cluster_barrier(S);
  }
  // keys above, and at the threshold, before this warp's share
  uint32_t before = lane < warp ? sh.above[lane % W] : 0;
  uint32_t at_before = lane < warp ? sh.at[lane % W] : 0;
  if (S > 1 && lane < rank) {  // a cluster has at most 16 CTAs
    const uint32_t* c = cluster_peer(sh.counts, lane);
    before += c[0];
    at_before += c[1];
  }
  before = __reduce_add_sync(0xffffffffu, before);
  at_before = __reduce_add_sync(0xffffffffu, at_before);
  uint32_t out = before + (at_before < need ? at_before : need);
  const unsigned below = (1u << lane) - 1;
  if constexpr (KeyFn::kQuads) {
    if (fast) {
#pragma unroll 2
      for (int32_t i0 = w_lo; i0 < w_hi; i0 += 128) {
        const int32_t i = i0 + lane * 4;
        uint4 kv = make_uint4(0, 0, 0, 0);
        if (i < w_hi) kv = key.quad(i / 4);
        const bool a = kv.x >= th.lo, b = kv.y >= th.lo, c = kv.z >= th.lo, d = kv.w >= th.lo;
        // prefix sums of the lanes' counts, 0 to 4, by their binary digits
        const uint32_t mine = (uint32_t)a + b + c + d;
        const unsigned b0 = __ballot_sync(0xffffffffu, mine & 1);
        const unsigned b1 = __ballot_sync(0xffffffffu, mine & 2);
        const unsigned b2 = __ballot_sync(0xffffffffu, mine & 4);
        uint32_t pos = out + __popc(b0 & below) + 2 * __popc(b1 & below) + 4 * __popc(b2 & below);
        if (a) emit(i, pos++);
        if (b) emit(i + 1, pos++);
        if (c) emit(i + 2, pos++);
        if (d) emit(i + 3, pos);
        out += __popc(b0) + 2 * __popc(b1) + 4 * __popc(b2);
      }
    }
  }
  if (!fast) {
    for (int32_t i0 = w_lo; i0 < w_hi; i0 += 32) {
      const int32_t i = i0 + lane;
      const bool in = i < w_hi;
      const Key kv = key(in ? i : w_lo);
      const bool eq = in && th.at(kv);
      const unsigned beq = __ballot_sync(0xffffffffu, eq);
      const bool take = (in && th.above(kv)) || (eq && at_before + __popc(beq & below) < need);
      const unsigned bt = __ballot_sync(0xffffffffu, take);
      if (take) emit(i, out + __popc(bt & below));
      out += __popc(bt);
      at_before += __popc(beq);
    }
  }
  if (S > 1) cluster_barrier(S);  // no CTA leaves while another still reads its counts
}

// Contiguous share [lo, hi) of n items for CTA `rank` of S.
GLA_HD void share_of(int32_t n, int S, int rank, int32_t* lo, int32_t* hi) {
  const int32_t per = (n + S - 1) / S;
  const int64_t a = (int64_t)per * rank;
  *lo = a < n ? (int32_t)a : n;
  *hi = a + per < n ? (int32_t)(a + per) : n;
}

}  // namespace gla
