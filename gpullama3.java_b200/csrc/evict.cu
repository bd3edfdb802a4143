// evict.cu - eviction from a KV cache by accumulated attention weight.
//
// Of a sequence's n rows each kv head keeps n_keep: the n_recent newest, and
// of the older ones those with the largest accumulated weight
// (gla_decode_weights_*), ties to the oldest.  Kept rows stay in order and
// move to rows 0..n_keep-1, each kv head by itself (its columns of a cache
// row), and their weights with them.  Rows carry their RoPE'd keys, so
// attention over the kept rows needs no positions.
//
// Which rows: one CTA a (sequence, kv head), past 32,768 rows a cluster, selects over
// the weights with the radix selection of cache_ops.cuh, its keys in shared memory,
// and writes the ascending list.  The rows then move in a second kernel (HBM-bound,
// each kept row read and written once): to another cache, every (row, 16-byte chunk)
// by itself; in place, a cluster a (sequence, kv head), in rounds (evict_compact_kernel).
//
// Calls of few kv heads do both in one launch (evict_small_kernel).
//
// Measured on one B200: 4096 rows of 8 kv heads to 1024, FP32, 8.4 us (a chain of loads
// and passes); 16 sequences of up to 32,768 FP16 rows to 4096 111 us, 21
// the selection (the longest sequence's walks) and 87 the copy (6.2 TB/s read and
// written); the same in place 149 us (16 of exactly 32,768 rows; one CTA a head and
// 64 columns of K or V: 209).
#include <algorithm>

#include "cache_ops.cuh"

namespace gla {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256;

// Selects the `pick` largest of the CTA's weights mine[0 .. count) (of a cluster's,
// if S > 1) and hands their indices to emit(index, position), ascending.  Keys are
// staged in s_key if they fit, else the weights are read again a pass.
template <class Emit>
__device__ __forceinline__ void select_weights(SelectScratch& sh, uint32_t* s_key, int S, int rank,
                                               const float* mine, int32_t count, int32_t pick,
                                               bool fits, Emit emit) {
  uint32_t kmin = ~0u, kmax = 0;
#pragma unroll 8
  for (int32_t i = threadIdx.x; i < count; i += kSelThreads) {
    const uint32_t k = order_key(__ldcg(mine + i));
    if (fits) s_key[i] = k;
    kmin = min(kmin, k);
    kmax = max(kmax, k);
  }
  if (fits) fill_up_keys(s_key, count);
  key_range<kSelThreads>(sh, S, &kmin, &kmax);  // (a barrier: the keys are staged)
  auto select = [&](auto key) {
    const Threshold<uint32_t> th = find_threshold<kSelThreads, uint32_t>(
        sh, S, count, (uint32_t)pick, kmin, kmax, key);
    emit_chosen<kSelThreads, uint32_t>(sh, S, rank, count, th, key, emit);
  };
  if (fits)
    select(SharedKeys{s_key});
  else
    select(keys_by([&](int32_t i) { return order_key(__ldcg(mine + i)); }));
}

__global__ void __launch_bounds__(kSelThreads)
    evict_select_kernel(const float* const* __restrict__ weight_ptrs, int64_t weight_stride,
                        const int32_t* __restrict__ n_pos, int32_t max_n_pos, int32_t n_keep,
                        int32_t n_recent, int32_t* __restrict__ kept, int32_t n_kv, int S,
                        int32_t key_cap, int32_t* __restrict__ status) {
  extern __shared__ __align__(16) uint32_t s_key[];
  __shared__ SelectScratch sh;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int rank = S > 1 ? (int)(blockIdx.x % (unsigned)S) : 0;
  const int item = (int)(blockIdx.x / (unsigned)S);
  const int b = item / n_kv, g = item - b * n_kv;
  int32_t n = clamped_rows(n_pos, b, max_n_pos, status);
  const float* w = weight_ptrs[b];
  if (!usable_weights(w, status)) n = 0;
  int32_t* out = kept + (int64_t)item * n_keep;
  if (n <= n_keep) {  // nothing to evict
    for (int32_t i = rank * kSelThreads + tid; i < n_keep; i += S * kSelThreads)
      out[i] = i < n ? i : -1;
    return;  // every CTA of the cluster takes this way
  }
  const int32_t older = n - n_recent, pick = n_keep - n_recent;
  for (int32_t i = rank * kSelThreads + tid; i < n_recent; i += S * kSelThreads)
    out[pick + i] = older + i;
  if (pick == 0) return;
  int32_t lo, hi;
  share_of(older, S, rank, &lo, &hi);
  // the ranks' shares differ by rounding alone, and every rank takes the same way
  const bool fits = (older + S - 1) / S <= key_cap;  // (not so past 16 CTAs' shared memory)
  select_weights(sh, s_key, S, rank, w + (int64_t)g * weight_stride + lo, hi - lo, pick, fits,
                 [&](int32_t i, uint32_t at) { out[at] = lo + i; });
}

// Selection and copy to another cache in one launch, for calls of few kv heads:
// `parts` CTAs of an item each select all of it (the weights are read from L2) and
// copy a share of the kept rows, which saves the second launch and its first loads
// (4096 FP32 rows of 8 kv heads to 1024: 8.4 us, in two launches 10.3).
template <int kChunks, int kPer, class T>
__global__ void __launch_bounds__(kSelThreads)
    evict_small_kernel(T* const* __restrict__ k_ptrs, T* const* __restrict__ v_ptrs,
                       float* const* __restrict__ weight_ptrs, int64_t weight_stride,
                       T* const* __restrict__ k_out_ptrs, T* const* __restrict__ v_out_ptrs,
                       float* const* __restrict__ weight_out_ptrs, int64_t weight_out_stride,
                       const int32_t* __restrict__ n_pos, int32_t max_n_pos, int32_t n_keep,
                       int32_t n_recent, int32_t* __restrict__ kept, int32_t n_kv,
                       int64_t kv_stride, int32_t parts, int32_t key_words,
                       int32_t* __restrict__ status) {
  extern __shared__ __align__(16) uint32_t s_key[];  // keys, then the list of kept rows
  __shared__ SelectScratch sh;
  pdl_wait();
  const int tid = threadIdx.x;
  const int item = (int)(blockIdx.x / (unsigned)parts), part = (int)(blockIdx.x % (unsigned)parts);
  const int b = item / n_kv, g = item - b * n_kv;
  const T* k = k_ptrs[b];
  const T* v = v_ptrs[b];
  const float* w = weight_ptrs[b];
  T* ko = k_out_ptrs[b];
  T* vo = v_out_ptrs[b];
  float* wo = weight_out_ptrs[b];
  int32_t n = clamped_rows(n_pos, b, max_n_pos, status);
  bool move = true;
  if (!usable_weights(w, status)) {
    n = 0;
  } else if (!usable_ptrs(k, v, status) || !usable_ptrs(ko, vo, status) ||
             !usable_weights(wo, status)) {
    move = false;
  } else if (k == ko || v == vo || w == wo) {  // another order of moves is needed in place
    if (tid == 0) atomicCAS(status, 0, GLA_ERR_INVALID_ARG);
    move = false;
  }
  int32_t* list = reinterpret_cast<int32_t*>(s_key) + key_words;
  const int32_t m = min(n, n_keep);
  w += (int64_t)g * weight_stride;
  if (n > n_keep) {
    const int32_t older = n - n_recent, pick = n_keep - n_recent;
    for (int32_t i = tid; i < n_recent; i += kSelThreads) list[pick + i] = older + i;
    if (pick > 0)
      select_weights(sh, s_key, 1, 0, w, older, pick, true,
                     [&](int32_t i, uint32_t at) { list[at] = i; });
  } else {
    for (int32_t i = tid; i < m; i += kSelThreads) list[i] = i;
  }
  __syncthreads();
  if (part == 0)
    for (int32_t i = tid; i < n_keep; i += kSelThreads)
      kept[(int64_t)item * n_keep + i] = i < m ? list[i] : -1;
  if (!move) return;
  const int32_t r0 = (int32_t)((int64_t)m * part / parts);
  const int32_t r1 = (int32_t)((int64_t)m * (part + 1) / parts);
  const int64_t col = (int64_t)g * kChunks * kPer;
#pragma unroll 2
  for (int32_t i = tid; i < (r1 - r0) * kChunks; i += kSelThreads) {
    const int32_t r = r0 + i / kChunks, c = i % kChunks;
    const int64_t src = (int64_t)list[r] * kv_stride + col + c * kPer;
    const int64_t dst = (int64_t)r * kv_stride + col + c * kPer;
    const float4 xk = __ldcg(reinterpret_cast<const float4*>(k + src));
    const float4 xv = __ldcg(reinterpret_cast<const float4*>(v + src));
    *reinterpret_cast<float4*>(ko + dst) = xk;
    *reinterpret_cast<float4*>(vo + dst) = xv;
  }
  for (int32_t r = r0 + tid; r < r1; r += kSelThreads)
    wo[(int64_t)g * weight_out_stride + r] = w[list[r]];
}

// Kept rows of one kv head to another cache: thread = (row, 16-byte chunk).
template <int kChunks, int kPer, class T>
__global__ void __launch_bounds__(kMoveThreads)
    evict_copy_kernel(T* const* __restrict__ k_ptrs, T* const* __restrict__ v_ptrs,
                      float* const* __restrict__ weight_ptrs, int64_t weight_stride,
                      T* const* __restrict__ k_out_ptrs, T* const* __restrict__ v_out_ptrs,
                      float* const* __restrict__ weight_out_ptrs, int64_t weight_out_stride,
                      const int32_t* __restrict__ n_pos, int32_t max_n_pos, int32_t n_keep,
                      const int32_t* __restrict__ kept, int32_t n_kv, int64_t kv_stride,
                      int32_t parts, int32_t* __restrict__ status) {
  constexpr int kUnroll = 4;
  constexpr int kRows = kMoveThreads * kUnroll / kChunks;  // rows of a CTA
  pdl_wait();
  const int tid = threadIdx.x;
  const int item = (int)(blockIdx.x / (unsigned)parts), part = (int)(blockIdx.x % (unsigned)parts);
  const int b = item / n_kv, g = item - b * n_kv;
  const int32_t n = clamped_rows(n_pos, b, max_n_pos, status);
  const T* k = k_ptrs[b];
  const T* v = v_ptrs[b];
  const float* w = weight_ptrs[b];
  T* ko = k_out_ptrs[b];
  T* vo = v_out_ptrs[b];
  float* wo = weight_out_ptrs[b];
  if (!usable_ptrs(k, v, status) || !usable_ptrs(ko, vo, status) || !usable_weights(w, status) ||
      !usable_weights(wo, status))
    return;
  if (k == ko || v == vo || w == wo) {  // another order of moves is needed in place
    if (tid == 0) atomicCAS(status, 0, GLA_ERR_INVALID_ARG);
    return;
  }
  const int32_t m = min(n, n_keep);
  const int32_t row0 = part * kRows;
  if (row0 >= m) return;
  const int32_t* list = kept + (int64_t)item * n_keep;
  float4 xk[kUnroll], xv[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = u * kMoveThreads + tid;
    const int r = i / kChunks, c = i - r * kChunks;
    if (r < kRows && row0 + r < m) {
      const int64_t src =
          (int64_t)list[row0 + r] * kv_stride + (int64_t)g * kChunks * kPer + c * kPer;
      xk[u] = __ldcg(reinterpret_cast<const float4*>(k + src));
      xv[u] = __ldcg(reinterpret_cast<const float4*>(v + src));
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int i = u * kMoveThreads + tid;
    const int r = i / kChunks, c = i - r * kChunks;
    if (r < kRows && row0 + r < m) {
      const int64_t dst = (int64_t)(row0 + r) * kv_stride + (int64_t)g * kChunks * kPer + c * kPer;
      *reinterpret_cast<float4*>(ko + dst) = xk[u];
      *reinterpret_cast<float4*>(vo + dst) = xv[u];
    }
  }
  for (int r = tid; r < kRows && row0 + r < m; r += kMoveThreads)
    wo[(int64_t)g * weight_out_stride + row0 + r] = w[(int64_t)g * weight_stride + list[row0 + r]];
}

// In place.  A cluster of S CTAs moves the rows of K and V of one (sequence, kv
// head), and its weights, in rounds of as many (row, 16-byte chunk) pairs as its
// threads take kUnroll each: all loads of a round, a cluster barrier, its stores.
// A kept row's source is never below its destination (list[i] >= i, ascending), so
// the stores of round r, to rows below the next round's first, can only hit sources
// of rounds <= r, which are all loaded; the loads of round r + 1 may therefore be in
// flight meanwhile, and the list entries of round r + 2 (which hides both their
// latency: 16 x 32,768 FP16 rows to 4096, 178 us with the entries read at their load).
template <int kChunks, int kPer, class T>
__global__ void __launch_bounds__(kMoveThreads, 2)
    evict_compact_kernel(T* const* __restrict__ k_ptrs, T* const* __restrict__ v_ptrs,
                         float* const* __restrict__ weight_ptrs, int64_t weight_stride,
                         const int32_t* __restrict__ n_pos, int32_t max_n_pos, int32_t n_keep,
                         const int32_t* __restrict__ kept, int32_t n_kv, int64_t kv_stride, int S,
                         int32_t* __restrict__ status) {
  constexpr int kUnroll = 8;
  constexpr int kRow = 2 * kChunks;  // chunks of a row: K's, then V's
  pdl_wait();
  const int rank = S > 1 ? (int)(blockIdx.x % (unsigned)S) : 0;
  const int item = (int)(blockIdx.x / (unsigned)S);
  const int b = item / n_kv, g = item - b * n_kv;
  const int32_t n = clamped_rows(n_pos, b, max_n_pos, status);
  if (n <= n_keep) return;  // every CTA of the cluster takes these ways
  T* k = k_ptrs[b];
  T* v = v_ptrs[b];
  float* w = weight_ptrs[b];
  if (!usable_ptrs(k, v, status) || !usable_weights(w, status)) return;
  const int32_t* list = kept + (int64_t)item * n_keep;
  const int me = rank * kMoveThreads + (int)threadIdx.x, all = S * kMoveThreads;
  k += (int64_t)g * kChunks * kPer;
  v += (int64_t)g * kChunks * kPer;
  w += (int64_t)g * weight_stride;

  const int32_t round = all * kUnroll / kRow;  // rows
  float4 cur[kUnroll], nxt[kUnroll];
  // sources of the round at work, of the next (its rows under way), of the one after
  int32_t from[kUnroll], from_next[kUnroll], from_then[kUnroll];
  // chunk u of this thread: row i0 + e / kRow of the round, chunk e % kRow
  auto at = [&](int32_t row, int c) {
    return (c < kChunks ? k : v) + (int64_t)row * kv_stride + (c % kChunks) * kPer;
  };
  auto sources = [&](int32_t i0, int32_t (&src)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = (u * all + me) / kRow;
      const int32_t i = i0 + r;
      src[u] = r < round && i < n_keep ? list[i] : i;  // (nothing to move)
    }
  };
  auto load = [&](int32_t i0, float4 (&x)[kUnroll], const int32_t (&src)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = u * all + me;
      // a row that stays needs no move
      if (src[u] != i0 + e / kRow) x[u] = __ldcg(reinterpret_cast<const float4*>(at(src[u], e % kRow)));
    }
  };
  sources(0, from);
  sources(round, from_next);
  load(0, cur, from);
  for (int32_t i0 = 0; i0 < n_keep; i0 += round) {
    cluster_barrier(S);  // every load of this round is done
    load(i0 + round, nxt, from_next);
    sources(i0 + 2 * round, from_then);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = u * all + me;
      const int32_t i = i0 + e / kRow;
      if (from[u] != i) *reinterpret_cast<float4*>(at(i, e % kRow)) = cur[u];
      cur[u] = nxt[u];
      from[u] = from_next[u];
      from_next[u] = from_then[u];
    }
  }
  for (int32_t i0 = 0; i0 < n_keep; i0 += all * kUnroll) {
    float x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int32_t i = i0 + u * all + me;
      if (i < n_keep) x[u] = __ldcg(w + list[i]);
    }
    cluster_barrier(S);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int32_t i = i0 + u * all + me;
      if (i < n_keep) w[i] = x[u];
    }
  }
  // the rows behind have no weight yet: a token appended there starts at zero (every
  // source is loaded: the last round's barrier)
  for (int32_t i = n_keep + me; i < n; i += all) w[i] = 0.f;
}

template <class... Params, class... Args>
int launch_pdl(void (*kern)(Params...), unsigned grid, int threads, cudaStream_t stream,
               const char* what, std::string* err, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    *err = std::string(what) + " launch failed: " + cudaGetErrorString(e);
    return GLA_ERR_CUDA;
  }
  return GLA_OK;
}

// CTAs of an item when one launch does it all, 0 when two do: the CTAs have to
// hold all keys and the list, must not make a second wave, and where they leave half
// of the device idle, the copy must be short (measured, one launch against two: 64 kv
// heads of 1000 to 8192 FP16 rows to 2048 31 and 33 us; 4 kv heads of 32,768 FP32
// rows to 16,384 on 64 CTAs 51 and 46).
int small_parts(const EvictRequest& r, const DeviceInfo& dev, int32_t* key_words) {
  const int64_t items = (int64_t)r.batch * r.n_kv;
  const int64_t keys = ((int64_t)r.max_n_pos + 3) / 4 * 4;
  const int64_t most = std::min(r.n_keep, r.max_n_pos);
  if (!r.k_out_ptrs || items * 2 > dev.sms || r.max_n_pos > 32768 ||
      (keys + most) * 4 > dev.smem_optin - 12 * 1024)
    return 0;
  *key_words = (int32_t)keys;
  const int64_t parts = std::max<int64_t>(1, std::min({(int64_t)16, dev.sms / items, (most + 31) / 32}));
  const int64_t bytes = most * 2 * r.head_dim * (r.dtype == GLA_DTYPE_F16 ? 2 : 4);
  return 2 * items * parts < dev.sms && bytes > parts * 128 * 1024 ? 0 : (int)parts;
}

template <class T, int HD>
int launch_small(const EvictRequest& r, int parts, int32_t key_words, cudaStream_t stream,
                 std::string* err) {
  static ClusterKernel ck;
  constexpr int kPer = 16 / sizeof(T);
  const int64_t items = (int64_t)r.batch * r.n_kv;
  const size_t smem = ((size_t)key_words + std::min(r.n_keep, r.max_n_pos)) * 4;
  return launch_clusters(evict_small_kernel<HD / kPer, kPer, T>, (unsigned)(items * parts),
                         kSelThreads, smem, 1, ck, stream, "evict",
                         err, reinterpret_cast<T* const*>(r.k_ptrs),
                         reinterpret_cast<T* const*>(r.v_ptrs), r.weight_ptrs, r.weight_stride,
                         reinterpret_cast<T* const*>(r.k_out_ptrs),
                         reinterpret_cast<T* const*>(r.v_out_ptrs), r.weight_out_ptrs,
                         r.weight_out_stride, r.n_pos, r.max_n_pos, r.n_keep, r.n_recent, r.kept,
                         r.n_kv, r.kv_stride, (int32_t)parts, key_words, r.status);
}

template <class T>
int small_dim(const EvictRequest& r, int parts, int32_t key_words, cudaStream_t stream,
              std::string* err) {
  switch (r.head_dim) {
    case 64: return launch_small<T, 64>(r, parts, key_words, stream, err);
    case 96: return launch_small<T, 96>(r, parts, key_words, stream, err);
    default: return launch_small<T, 128>(r, parts, key_words, stream, err);
  }
}

template <class T, int HD>
int launch_move(const EvictRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                std::string* err) {
  constexpr int kPer = 16 / sizeof(T);
  constexpr int kChunks = HD / kPer;
  const int64_t items = (int64_t)r.batch * r.n_kv;
  if (r.k_out_ptrs) {
    constexpr int kRows = kMoveThreads * 4 / kChunks;
    const int32_t most = std::min(r.n_keep, r.max_n_pos);
    const int64_t parts = std::max(1, (most + kRows - 1) / kRows);
    if (items * parts > INT32_MAX) {
      *err = "too many rows to move in one call";
      return GLA_ERR_NOT_SUPPORTED;
    }
    return launch_pdl(evict_copy_kernel<kChunks, kPer, T>, (unsigned)(items * parts), kMoveThreads,
                      stream, "evict copy", err, reinterpret_cast<T* const*>(r.k_ptrs),
                      reinterpret_cast<T* const*>(r.v_ptrs), r.weight_ptrs, r.weight_stride,
                      reinterpret_cast<T* const*>(r.k_out_ptrs),
                      reinterpret_cast<T* const*>(r.v_out_ptrs), r.weight_out_ptrs,
                      r.weight_out_stride, r.n_pos, r.max_n_pos, r.n_keep,
                      (const int32_t*)r.kept, r.n_kv, r.kv_stride, (int32_t)parts, r.status);
  }
  // CTAs of an item's cluster: as many as the device holds at once (two an SM), while
  // a round is not more than half of the rows
  static ClusterKernel ck;
  auto kern = evict_compact_kernel<kChunks, kPer, T>;
  int S = 1;
  while (S < 16 && items * S * 2 <= 2 * dev.sms &&
         (int64_t)2 * S * kMoveThreads * 8 / (2 * kChunks) * 2 <= r.n_keep &&
         items <= clusters_held(kern, ck, kMoveThreads, 0, 2 * S, dev))
    S *= 2;
  if (items * S > INT32_MAX) {
    *err = "batch * n_kv_heads too large";
    return GLA_ERR_NOT_SUPPORTED;
  }
  return launch_clusters(kern, (unsigned)(items * S), kMoveThreads, 0, S, ck, stream,
                         "evict compaction", err, reinterpret_cast<T* const*>(r.k_ptrs),
                         reinterpret_cast<T* const*>(r.v_ptrs), r.weight_ptrs, r.weight_stride,
                         r.n_pos, r.max_n_pos, r.n_keep, (const int32_t*)r.kept, r.n_kv,
                         r.kv_stride, S, r.status);
}

template <class T>
int move_dim(const EvictRequest& r, const DeviceInfo& dev, cudaStream_t stream,
             std::string* err) {
  switch (r.head_dim) {
    case 64: return launch_move<T, 64>(r, dev, stream, err);
    case 96: return launch_move<T, 96>(r, dev, stream, err);
    default: return launch_move<T, 128>(r, dev, stream, err);
  }
}

}  // namespace

int launch_evict(const EvictRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                 std::string* err) {
  int32_t key_words = 0;
  if (const int parts = small_parts(r, dev, &key_words))
    return r.dtype == GLA_DTYPE_F16 ? small_dim<__half>(r, parts, key_words, stream, err)
                                    : small_dim<float>(r, parts, key_words, stream, err);
  static ClusterKernel ck;
  const int64_t items = (int64_t)r.batch * r.n_kv;
  // One CTA a kv head up to 32,768 weights: each of the passes of a cluster costs it
  // about 1.5 us in barriers and remote counts, more than walking that many keys in
  // shared memory (16 sequences of up to 32,768 rows: 28 us with clusters of 4).
  // Past 16 CTAs' shared memory the weights are read again a pass.
  const int64_t most_keys = (dev.smem_optin - 12 * 1024) / 4;
  int S = 1;
  while (S < 16 && r.max_n_pos > (int64_t)32768 * S) S *= 2;
  const int32_t key_cap =
      (int32_t)std::min<int64_t>(most_keys, ((int64_t)r.max_n_pos + S - 1) / S);
  if (items * S > INT32_MAX) {
    *err = "batch * n_kv_heads too large";
    return GLA_ERR_NOT_SUPPORTED;
  }
  int rc = launch_clusters(evict_select_kernel, (unsigned)(items * S), kSelThreads,
                           ((size_t)key_cap + 3) / 4 * 16, S, ck,
                           stream, "evict selection", err,
                           (const float* const*)r.weight_ptrs, r.weight_stride, r.n_pos,
                           r.max_n_pos, r.n_keep, r.n_recent, r.kept, r.n_kv, S, key_cap, r.status);
  if (rc != GLA_OK) return rc;
  return r.dtype == GLA_DTYPE_F16 ? move_dim<__half>(r, dev, stream, err)
                                  : move_dim<float>(r, dev, stream, err);
}

}  // namespace gla
