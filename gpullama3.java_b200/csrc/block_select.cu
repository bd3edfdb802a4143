// block_select.cu - the blocks of cached rows that one query's kv heads read.
//
// score(j, g) = max over the q heads h of kv head g of
//               sum_d max(q_hd lo_jgd, q_hd hi_jgd)
//             = max_h sum_d (min(q_hd, 0) lo_jgd + max(q_hd, 0) hi_jgd),
// an upper bound of q_h . k_t for every row t of block j.  The first n_first
// and the last n_last blocks are always chosen; of the others the highest
// scores, ties to the lowest block.
//
// Scores are summed in FP64: which of two blocks is chosen is a comparison of
// two sums of up to 256 products, and with FP32 sums it would depend on the
// order of the additions (on the kernel's shape) about once in a hundred
// selections.  An FP32 query times an FP16 or FP32 bound is exact in FP64 (48
// bits), so what is left is 2^-53 of the sum.
//
// A cluster of S CTAs works on one (sequence, kv head): CTA r scores a
// contiguous range of blocks into its shared memory, then the cluster finds
// the n_sel-th largest key together (cache_ops.cuh) and writes the ids in
// ascending order.  One launch, no global workspace.
#include "cache_ops.cuh"

namespace gla {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Sums N values (N a power of two <= 32) over LANES lanes: each halving step
// exchanges half of the values, so the whole costs N - 1 exchanges instead of
// N log2(LANES).  Afterwards lane l of the group holds the sum of value
// l >> (log2 LANES - log2 N) (lanes that share a value all hold it).
template <int N, int LANES>
__device__ __forceinline__ double reduce_scatter(double (&v)[N], int lane) {
  int n = N;
#pragma unroll
  for (int m = LANES / 2; m > 0; m >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = (lane & m) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const double keep = up ? v[i + n] : v[i];
          const double send = up ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
    }
  }
  return v[0];
}

constexpr int ilog2(int x) { return x <= 1 ? 0 : 1 + ilog2(x >> 1); }

// GP: heads of a group, padded to a power of two.
template <class T, int HD, int GP>
__global__ void __launch_bounds__(kThreads)
    block_select_kernel(const float* __restrict__ q, const T* const* __restrict__ bounds_ptrs,
                        const int32_t* __restrict__ n_pos, int32_t max_n_pos,
                        int32_t* __restrict__ block_ids, int32_t n_heads, int32_t n_kv,
                        int32_t br_shift, int32_t n_sel, int32_t n_first, int32_t n_last, int S,
                        int32_t* __restrict__ status) {
  constexpr int kPer = 16 / sizeof(T);                  // elements of a 16-byte chunk
  constexpr int kChunks = 2 * HD / kPer;                // of one (block, head): lo then hi
  constexpr int kLanes = kChunks >= 32 ? 32 : (kChunks > 16 ? 32 : 16);
  constexpr int kCpl = (kChunks + kLanes - 1) / kLanes; // chunks a lane
  constexpr int kSub = 32 / kLanes;                     // blocks side by side in a warp
  // blocks a lane group scores at once: as many as one exchange of 32 values joins
  constexpr int kNB = 32 / GP > 8 ? 8 : 32 / GP;
  constexpr int kVals = kNB * GP > kLanes ? kLanes : kNB * GP;
  constexpr int kBlk = kVals / GP;
  extern __shared__ uint64_t s_key[];
  __shared__ SelectScratch sh;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = S > 1 ? (int)(blockIdx.x % (unsigned)S) : 0;
  const int item = (int)(blockIdx.x / (unsigned)S);
  const int b = item / n_kv, g = item - b * n_kv;
  const int G = n_heads / n_kv;
  const int32_t n = clamped_rows(n_pos, b, max_n_pos, status);
  const T* bounds = bounds_ptrs[b];
  const bool ok = usable_ptrs(bounds, bounds, status);
  const int32_t nb = ok ? (int32_t)(((int64_t)n + (1 << br_shift) - 1) >> br_shift) : 0;
  int32_t* ids = block_ids + (int64_t)item * n_sel;
  if (nb <= n_sel) {  // every block is chosen, whatever its score
    for (int i = rank * kThreads + tid; i < n_sel; i += S * kThreads) ids[i] = i < nb ? i : -1;
    return;  // every CTA of the cluster takes this way
  }
  int32_t lo, hi;
  share_of(nb, S, rank, &lo, &hi);

  // this lane's coefficients: element e of its chunks, all heads
  const int sub = lane / kLanes, sl = lane % kLanes;
  double co[kCpl * kPer][GP];
#pragma unroll
  for (int c = 0; c < kCpl; ++c) {
    const int chunk = sl + c * kLanes;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int el = chunk * kPer + e;  // [0, HD) lo, [HD, 2 HD) hi
      const int d = el < HD ? el : el - HD;
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        float x = 0.f;
        if (chunk < kChunks && h < G)
          x = q[((int64_t)b * n_heads + (int64_t)g * G + h) * HD + d];
        // a NaN query element stays NaN: its block ranks lowest
        co[c * kPer + e][h] = (double)(el < HD ? (x > 0.f ? 0.f : x) : (x < 0.f ? 0.f : x));
      }
    }
  }
  const int64_t row = (int64_t)n_kv * 2 * HD;
  for (int32_t j0 = lo + (warp * kSub + sub) * kBlk; j0 - sub * kBlk < hi;
       j0 += kWarps * kSub * kBlk) {
    float4 x[kBlk][kCpl];
#pragma unroll
    for (int i = 0; i < kBlk; ++i) {
      const T* src = bounds + (int64_t)min(j0 + i, hi - 1) * row + (int64_t)g * 2 * HD;
#pragma unroll
      for (int c = 0; c < kCpl; ++c) {
        const int chunk = sl + c * kLanes;
        x[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (chunk < kChunks) x[i][c] = __ldg(reinterpret_cast<const float4*>(src) + chunk);
      }
    }
    double acc[kVals];
#pragma unroll
    for (int i = 0; i < kBlk; ++i) {
#pragma unroll
      for (int h = 0; h < GP; ++h) acc[i * GP + h] = 0.0;
#pragma unroll
      for (int c = 0; c < kCpl; ++c) {
        const T* e = reinterpret_cast<const T*>(&x[i][c]);
#pragma unroll
        for (int p = 0; p < kPer; ++p) {
          const double y = (double)(float)e[p];
#pragma unroll
          for (int h = 0; h < GP; ++h)
            acc[i * GP + h] = fma(co[c * kPer + p][h], y, acc[i * GP + h]);
        }
      }
    }
    double s = reduce_scatter<kVals, kLanes>(acc, sl);
    // lane sl holds value sl >> kRep: block value / GP, head value % GP
    constexpr int kRep = ilog2(kLanes) - ilog2(kVals);
    const int val = sl >> kRep;
    const int h = val % GP;
    uint64_t key = h < G ? order_key(s) : 0;
#pragma unroll
    for (int m = (GP << kRep) >> 1; m >= (1 << kRep) && m > 0; m >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, key, m);
      key = o > key ? o : key;
    }
    const int32_t j = j0 + val / GP;
    if (h == 0 && (sl & ((1 << kRep) - 1)) == 0 && j < hi)
      s_key[j - lo] = (j < n_first || j >= nb - n_last) ? ~0ull : key;
  }
  __syncthreads();
  cluster_select<kThreads, uint64_t>(
      sh, S, rank, hi - lo, (uint32_t)n_sel, [&](int32_t i) { return s_key[i]; },
      [&](int32_t i, uint32_t at) { ids[at] = lo + i; });
}

template <class T, int HD, int GP>
int launch_select(const SelectRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                  std::string* err) {
  static std::atomic<uint64_t> attr_done{0};
  int32_t br_shift = 0;
  while ((1 << br_shift) < r.block_rows) ++br_shift;
  const int64_t items = (int64_t)r.batch * r.n_kv;
  const int64_t max_nb = ((int64_t)r.max_n_pos + r.block_rows - 1) / r.block_rows;
  // as many CTAs a (sequence, kv head) as fill the device once, while each
  // still has 64 blocks to score; and enough for the keys to fit shared memory
  const int64_t key_cap = (dev.smem_optin - 8 * 1024) / 8;
  int S = 1;
  while (S < 16 && ((items * S < dev.sms && max_nb > 64 * S) || (max_nb + S - 1) / S > key_cap))
    S *= 2;
  const int64_t per = (max_nb + S - 1) / S;
  if (per > key_cap) {
    *err = "too many blocks for one selection";
    return GLA_ERR_NOT_SUPPORTED;
  }
  if (items * S > INT32_MAX) {
    *err = "batch * n_kv_heads too large";
    return GLA_ERR_NOT_SUPPORTED;
  }
  return launch_clusters(block_select_kernel<T, HD, GP>, (unsigned)(items * S), kThreads,
                         (size_t)per * 8, S, attr_done, stream, "block selection", err, r.q,
                         reinterpret_cast<const T* const*>(r.bounds_ptrs), r.n_pos, r.max_n_pos,
                         r.block_ids, r.n_heads, r.n_kv, br_shift, r.n_sel, r.n_first, r.n_last, S,
                         r.status);
}

template <class T, int HD>
int select_group(const SelectRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                 std::string* err) {
  const int G = r.n_heads / r.n_kv;
  if (G == 1) return launch_select<T, HD, 1>(r, dev, stream, err);
  if (G == 2) return launch_select<T, HD, 2>(r, dev, stream, err);
  if (G <= 4) return launch_select<T, HD, 4>(r, dev, stream, err);
  return launch_select<T, HD, 8>(r, dev, stream, err);
}

template <class T>
int select_dim(const SelectRequest& r, const DeviceInfo& dev, cudaStream_t stream,
               std::string* err) {
  switch (r.head_dim) {
    case 64: return select_group<T, 64>(r, dev, stream, err);
    case 96: return select_group<T, 96>(r, dev, stream, err);
    default: return select_group<T, 128>(r, dev, stream, err);
  }
}

}  // namespace

int launch_block_select(const SelectRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                        std::string* err) {
  return r.dtype == GLA_DTYPE_F16 ? select_dim<__half>(r, dev, stream, err)
                                  : select_dim<float>(r, dev, stream, err);
}

}  // namespace gla
