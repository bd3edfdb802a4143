// block_select.cu - the blocks of cached rows that one query's kv heads read.
//
// score(j, g) = max over the q heads h of kv head g of
//               sum_d max(q_hd lo_jgd, q_hd hi_jgd)
//             = max_h sum_d (min(q_hd, 0) lo_jgd + max(q_hd, 0) hi_jgd),
// an upper bound of q_h . k_t for every row t of block j.  The first n_first
// and the last n_last blocks are always chosen; of the others the highest
// scores, ties to the lowest block.
//
// The order is that of the sums in FP64: which of two blocks is chosen must
// not depend on the order of additions, so on the kernel's shape.  But FP64
// sums of everything would cost more than reading the bounds (a conversion
// and an FMA at 1/8 and 1/2 of the FP32 rate), and few comparisons need them:
//  1. scores in FP32.  A sum of at most 8 FMAs and 5 tree additions is within
//     E = 2^-20 M of the exact one (13 roundings of 2^-24 of the sum of
//     magnitudes at most); M bounds that sum for all blocks: over the lanes, a
//     lane's largest |bound| times its sum of |coefficients|.
//  2. the n_sel highest FP32 scores, lowest vmin, against the others, highest
//     vmax.  If vmin - vmax > 2E the order is settled.
//  3. otherwise scores above vmax + 2E are surely chosen (they exceed every one
//     that was not), those below vmin - 2E surely not, and the few between are
//     summed again in FP64 (an FP32 query times an FP16 or FP32 bound is exact
//     there up to 2^-53) and ranked by that.
// M = 0 (a zero query, zero bounds, no channel with both) means that the FP32 scores
// are exact; where a product of M falls below FP32's normal range its smallest normal
// number stands for it, and 2E has room for what the scores' own products lose there.
// A bound or query too large for E to be finite leaves everything to step 3.
//
// A cluster of S CTAs works on one (sequence, kv head): each scores a
// contiguous range of blocks and stores the keys into rank 0's shared memory,
// where rank 0 selects alone with block barriers (a radix pass that every CTA
// of the cluster took part in cost a cluster barrier of about 0.5 us each).
// One launch, no global workspace.
//
// HBM-bound for a batch, latency-bound for a token.  Measured on one B200: 2048
// blocks of 4 kv heads, FP16, 11.1 us, of which 3 until the first bounds are here, 3
// scoring, 1 the cluster's barrier and 4 the selection; 16 sequences of up to 1024
// blocks, 8 kv heads, FP32 21.5 us (FP64 scores throughout: 40; copies of 16 bytes a
// lane instead of bulk ones: 24).
#include <algorithm>
#include <cfloat>

#include "cache_ops.cuh"

namespace gla {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kErr = 9.5367431640625e-07f;  // 2^-20
constexpr int kNear = 64;  // scores near the border that are ranked by comparing all pairs

// Sums N values (N a power of two <= 32) over LANES lanes: each halving step
// exchanges half of the values, so the whole costs N - 1 exchanges instead of
// N log2(LANES).  Afterwards lane l of the group holds the sum of value
// l >> (log2 LANES - log2 N) (lanes that share a value all hold it).
template <int N, int LANES>
__device__ __forceinline__ float reduce_scatter(float (&v)[N], int lane) {
  int n = N;
#pragma unroll
  for (int m = LANES / 2; m > 0; m >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = (lane & m) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const float keep = up ? v[i + n] : v[i];
          const float send = up ? v[i] : v[i + n];
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

// The coefficient of a bound: min(q, 0) of lo, max(q, 0) of hi, written so
// that a NaN stays NaN.
__device__ __forceinline__ float coefficient(float q, bool is_lo) {
  return is_lo ? (q > 0.f ? 0.f : q) : (q < 0.f ? 0.f : q);
}

// How a (head size, type, padded group GP) is scored.  A (block, kv head) is
// kChunks 16-byte chunks, lo then hi, over kLanes lanes; a lane holds the
// coefficients of its chunks in registers (at most 8 elements of GP heads) and
// a lane group scores kBlk blocks at once, so that one reduce_scatter joins
// them.  The blocks come through a ring of each warp's own in shared memory, kStages
// steps deep, by one bulk copy a block: its 256 to 1024 bytes lie together, and
// copies by 16 bytes a lane compete with the lanes' own shared memory traffic.
template <class T, int HD, int GP>
struct Shape {
  static constexpr int kPer = 16 / sizeof(T);
  static constexpr int kChunks = 2 * HD / kPer;
  static constexpr int kLanes = kChunks > 16 ? 32 : 16;
  static constexpr int kCpl = (kChunks + kLanes - 1) / kLanes;
  static constexpr int kSub = 32 / kLanes;  // lane groups of a warp
  static constexpr int kWant = GP <= 2 ? 8 / kCpl : 4;
  static constexpr int kBlk = kWant * GP > kLanes ? kLanes / GP : kWant;  // a value a lane
  static constexpr int kVals = kBlk * GP;
  static constexpr int kSlot = kSub * kBlk * kChunks * 16;  // bytes of a step
  static constexpr int kStages = std::min(6, 96 * 1024 / (kWarps * kSlot));
  static constexpr int kRing = kWarps * kStages * kSlot;
  static_assert(kCpl * kPer <= 8, "the error bound counts 8 terms a lane");
  static_assert(kStages >= 2, "a step in flight beside the one at work");
};

// The ring and the 64-bit keys' upper words share their bytes.
template <class T, int HD, int GP>
size_t select_smem(int64_t max_nb) {  // max_nb: a multiple of 4
  using Sh = Shape<T, HD, GP>;
  return (size_t)std::max<int64_t>(Sh::kRing, max_nb * 4) + (size_t)max_nb * 4;
}

// The FP64 score of one (block, kv head), by one warp: the larger product of
// each channel, so that an infinite bound on the other side does not count
// (the FP32 scores' min(q, 0) lo + max(q, 0) hi would make it a NaN, but an
// infinity among the bounds leaves no finite E, and all scores come here).
template <class T, int HD>
__device__ __forceinline__ uint64_t exact_key(const T* src, const float* s_q, int G, int lane) {
  uint64_t key = 0;
  for (int h = 0; h < G; ++h) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int d = i * 32 + lane;
      const double qd = (double)s_q[h * HD + d];
      const double a = qd * (double)(float)src[d], c = qd * (double)(float)src[HD + d];
      s += (a > c || a != a) ? a : c;  // a NaN of either stays
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    const uint64_t k = order_key(s);
    key = k > key ? k : key;
  }
  return key;
}

// GP: heads of a group, padded to a power of two.
template <class T, int HD, int GP>
__global__ void __launch_bounds__(kThreads, 2)
    block_select_kernel(const float* __restrict__ q, const T* const* __restrict__ bounds_ptrs,
                        const int32_t* __restrict__ n_pos, int32_t max_n_pos,
                        int32_t* __restrict__ block_ids, int32_t n_heads, int32_t n_kv,
                        int32_t br_shift, int32_t n_sel, int32_t n_first, int32_t n_last, int S,
                        int32_t max_nb, int32_t* __restrict__ status) {
  using Sh = Shape<T, HD, GP>;
  constexpr int kPer = Sh::kPer, kLanes = Sh::kLanes, kCpl = Sh::kCpl, kBlk = Sh::kBlk;
  constexpr int kStages = Sh::kStages;
  constexpr int kVals = Sh::kVals, kStep = kWarps * Sh::kSub * kBlk;
  // the warps' rings, in rank 0 later the upper words of 64-bit keys; then rank 0's
  // FP32 keys, later the lower words
  extern __shared__ __align__(16) char s_dyn[];
  __shared__ SelectScratch sh;
  // rank 0's, of every warp of the cluster: M, the smallest and the largest key
  __shared__ float s_mag[16 * kWarps];
  __shared__ uint32_t s_min[16 * kWarps], s_max[16 * kWarps];
  __shared__ __align__(16) float s_q[GP * HD];
  __shared__ uint32_t s_least[kWarps], s_most[kWarps];
  __shared__ int32_t s_near[kNear];
  __shared__ uint64_t s_near_key[kNear];
  __shared__ int32_t s_near_n, s_sure_n;
  __shared__ uint64_t s_bar[kWarps * Sh::kStages];
  __shared__ int s_abort, s_late;  // a bounded wait gave up; so did one for what it left
  __shared__ int32_t s_lost[kWarps];  // of a warp whose wait gave up: that step
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = S > 1 ? (int)(blockIdx.x % (unsigned)S) : 0;
  const int item = (int)(blockIdx.x / (unsigned)S);
  const int b = item / n_kv, g = item - b * n_kv;
  const int G = n_heads / n_kv;
  if (tid == 0) s_abort = s_late = 0;
  pdl_wait();
  pdl_launch_dependents();
  // q, the length and the pointer are loaded side by side
  constexpr int kQ = (GP * HD + kThreads - 1) / kThreads;
  float qr[kQ];
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    const int at = i * kThreads + tid;
    qr[i] = at < G * HD ? __ldg(q + ((int64_t)b * n_heads + (int64_t)g * G) * HD + at) : 0.f;
  }
  const int32_t n = clamped_rows(n_pos, b, max_n_pos, status);
  const T* bounds = bounds_ptrs[b];
  const bool ok = usable_ptrs(bounds, bounds, status);
  const int32_t nb = ok ? (int32_t)(((int64_t)n + (1 << br_shift) - 1) >> br_shift) : 0;
  int32_t* ids = block_ids + (int64_t)item * n_sel;
  // the blocks between those that are always chosen: `pick` of them
  const int32_t pick = n_sel - n_first - n_last, nc = nb - n_first - n_last;
  if (nb <= n_sel || pick == 0) {
    for (int i = rank * kThreads + tid; i < n_sel; i += S * kThreads)
      ids[i] = nb <= n_sel ? (i < nb ? i : -1) : (i < n_first ? i : nb - n_sel + i);
    return;  // every CTA of the cluster takes this way
  }
  int32_t lo, hi;  // this CTA's candidates, counted from block n_first
  share_of(nc, S, rank, &lo, &hi);

  const int sub = lane / kLanes, sl = lane % kLanes;
  const int64_t row = (int64_t)n_kv * 2 * HD;
  const T* base = bounds + (int64_t)n_first * row + (int64_t)g * 2 * HD;
  uint32_t* s_upper = reinterpret_cast<uint32_t*>(s_dyn);
  uint32_t* s_lower = reinterpret_cast<uint32_t*>(s_dyn + max(Sh::kRing, max_nb * 4));
  char* ring = s_dyn + warp * (kStages * Sh::kSlot);
  uint64_t* bars = s_bar + warp * kStages;  // a slot's copies have landed
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) mbar_init(bars + s, 1);
    fence_mbarrier_init();
  }
  __syncwarp();
  constexpr int kBytes = Sh::kChunks * 16;  // of a block
  auto fetch = [&](int s, int32_t jw) {  // blocks jw + 0 .. kSub * kBlk - 1, a lane each
    if (jw >= hi) return;
    if (lane == 0) mbar_arrive_expect_tx(bars + s, Sh::kSlot);
    __syncwarp();
    if (lane < Sh::kSub * kBlk)  // (the last block again past the end)
      bulk_g2s_keep(ring + s * Sh::kSlot + lane * kBytes,
                    base + (int64_t)min(jw + lane, hi - 1) * row, kBytes, bars + s);
  };
  const int32_t w0 = lo + warp * Sh::kSub * kBlk;  // the warp's first block
  // in flight while the coefficients are set up
#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(s, w0 + s * kStep);
  cluster_arrive(S);
#pragma unroll
  for (int i = 0; i < kQ; ++i)
    if (i * kThreads + tid < GP * HD) s_q[i * kThreads + tid] = qr[i];
  __syncthreads();
  // (products of two heads at once: packed FMAs)
  constexpr int kPairs = GP >= 2 ? GP / 2 : 1;
  uint64_t co[kCpl * kPer][kPairs];
#pragma unroll
  for (int c = 0; c < kCpl; ++c) {
    const int el = (sl + c * kLanes) * kPer;  // [0, HD) lo, [HD, 2 HD) hi
    const int d = el < HD ? el : el - HD;
#pragma unroll
    for (int h = 0; h < kPairs; ++h)
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        auto of = [&](int head) {
          return el < 2 * HD && head < GP ? coefficient(s_q[head * HD + d + p], el < HD) : 0.f;
        };
        co[c * kPer + p][h] = pk2(of(2 * h), of(2 * h + 1));
      }
  }

  // keys, M and the keys' range go to rank 0's shared memory
  uint32_t* key0 = S > 1 ? const_cast<uint32_t*>(cluster_peer(s_lower, 0)) : s_lower;
  cluster_wait(S);  // rank 0 is running: its shared memory may be written
  float big = 0.f;
  bool strange = false;  // a NaN bound (its scores are NaN; a maximum would drop it)
  uint32_t kmin = ~0u, kmax = 0;
  uint32_t phase = 0;  // parity of the ring's round
  // A wait that gave up (the status word says so) ends the warp's copies: what it scores
  // from then on is arbitrary, but every block gets a key.
  bool alive = true;
  for (int32_t jw0 = w0; jw0 < hi; jw0 += kStages * kStep, phase ^= 1) {
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      const int32_t jw = jw0 + st * kStep, j0 = jw + sub * kBlk;
      if (jw >= hi) break;
      const bool here = mbar_wait(bars + st, phase, &s_abort, status);
      float acc[kVals];
#pragma unroll
      for (int i = 0; i < kBlk; ++i) {
        uint64_t sum[kPairs];
#pragma unroll
        for (int h = 0; h < kPairs; ++h) sum[h] = 0;
#pragma unroll
        for (int c = 0; c < kCpl; ++c) {
          const int chunk = sl + c * kLanes;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (chunk < Sh::kChunks)
            x = reinterpret_cast<const float4*>(ring + st * Sh::kSlot +
                                                (sub * kBlk + i) * kBytes)[chunk];
#pragma unroll
          for (int p = 0; p < kPer; ++p) {
            const float y = (float)reinterpret_cast<const T*>(&x)[p];
            big = fmaxf(big, fabsf(y));
            const uint64_t yy = pk2(y, y);
#pragma unroll
            for (int h = 0; h < kPairs; ++h) sum[h] = fma2(co[c * kPer + p][h], yy, sum[h]);
          }
        }
#pragma unroll
        for (int h = 0; h < kPairs; ++h) {
          float a, b2;
          upk2(sum[h], a, b2);
          acc[i * GP + 2 * h] = a;
          if (GP > 1) acc[i * GP + (2 * h + 1) % GP] = b2;
        }
      }
      if (alive) {
        alive = __all_sync(0xffffffffu, here);  // and read out by every lane
        if (alive)
          fetch(st, jw + kStages * kStep);
        else
          s_lost[warp] = (jw - w0) / kStep;
      }
      const float s = reduce_scatter<kVals, kLanes>(acc, sl);
      // lane sl holds value sl >> kRep: block value / GP, head value % GP
      constexpr int kRep = ilog2(kLanes) - ilog2(kVals);
      const int val = sl >> kRep;
      const int h = val % GP;
      strange |= s != s;
      uint32_t key = h < G ? order_key(s) : 0;
#pragma unroll
      for (int m = (GP << kRep) >> 1; m >= (1 << kRep) && m > 0; m >>= 1)
        key = max(key, __shfl_xor_sync(0xffffffffu, key, m));
      const int32_t j = j0 + val / GP;
      if (j < hi) {
        kmin = min(kmin, key);
        kmax = max(kmax, key);
        if (h == 0 && (sl & ((1 << kRep) - 1)) == 0) key0[j] = key;
      }
    }
  }
  if (!alive) {  // no copy may land after the CTA has left
    __syncwarp();
    for (int32_t i = s_lost[warp], e = i + kStages; i < e && w0 + i * kStep < hi; ++i)
      mbar_wait(bars + i % kStages, (i / kStages) & 1, &s_late, status);
  }
  // M of this warp's blocks (its lane groups see different blocks: their maximum counts)
  if (strange) big = INFINITY;
#pragma unroll
  for (int m = kLanes; m < 32; m <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, m));
  float mag = 0.f;
  bool nan_q = false;
#pragma unroll
  for (int h = 0; h < GP; ++h) {
    float cs = 0.f;
#pragma unroll
    for (int e = 0; e < kCpl * kPer; ++e) {
      float a, b2;
      upk2(co[e][h / 2], a, b2);
      cs += fabsf(h % 2 ? b2 : a);
    }
    const bool none = cs == 0.f;  // an infinite bound that no coefficient meets
    cs = none ? 0.f : cs * big;
    if (!none && big != 0.f) cs = cs < FLT_MIN ? FLT_MIN : cs;  // 0 only if all products are
#pragma unroll
    for (int m = kLanes / 2; m > 0; m >>= 1) cs += __shfl_xor_sync(0xffffffffu, cs, m);
    nan_q |= cs != cs;
    mag = fmaxf(mag, cs);
  }
  if (nan_q || __any_sync(0xffffffffu, big == INFINITY)) mag = INFINITY;
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if (lane == 0) {
    float* mag0 = S > 1 ? const_cast<float*>(cluster_peer(s_mag, 0)) : s_mag;
    uint32_t* min0 = S > 1 ? const_cast<uint32_t*>(cluster_peer(s_min, 0)) : s_min;
    uint32_t* max0 = S > 1 ? const_cast<uint32_t*>(cluster_peer(s_max, 0)) : s_max;
    mag0[rank * kWarps + warp] = mag;
    min0[rank * kWarps + warp] = kmin;
    max0[rank * kWarps + warp] = kmax;
  }
  if (tid == 0) s_near_n = s_sure_n = 0;
  if (rank == 0) fill_up_keys(s_lower, nc);
  cluster_barrier(S);
  if (rank != 0) return;

  // rank 0: all keys are here
  for (int i = tid; i < n_first + n_last; i += kThreads)
    ids[i < n_first ? i : pick + i] = i < n_first ? i : nc + i;
  ids += n_first;
  const SharedKeys key_of{s_lower};
  auto emit = [&](int32_t i, uint32_t at) { ids[at] = n_first + i; };
  mag = 0.f;
  kmin = ~0u;
  kmax = 0;
  for (int i = lane; i < S * kWarps; i += 32) {
    mag = fmaxf(mag, s_mag[i]);
    kmin = min(kmin, s_min[i]);
    kmax = max(kmax, s_max[i]);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, m));
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  const Threshold<uint32_t> th = find_threshold<kThreads, uint32_t>(
      sh, 1, nc, (uint32_t)pick, kmin, kmax, key_of);
  // the lowest chosen and the highest other key
  uint32_t least = ~0u, most = 0;
#pragma unroll 4
  for (int32_t i = tid; i < nc; i += kThreads) {
    const uint32_t key = key_of(i);
    if (key >= th.lo) least = min(least, key);
    if (key < th.lo || (!th.whole && th.at(key))) most = max(most, key);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) {
    s_least[warp] = least;
    s_most[warp] = most;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    least = min(least, s_least[w]);
    most = max(most, s_most[w]);
  }
  // 2E, rounded up (products below FP32's normal range lose at most 2^-149 each);
  // no bound where a sum could have overflowed
  float two_e = mag == 0.f ? 0.f : 2.01f * kErr * mag + 1e-41f;
  if (!(mag < 1e37f)) two_e = INFINITY;
  const float vmin = key_score(least), vmax = key_score(most);
  if (two_e == 0.f || vmin - vmax > two_e) {
    emit_chosen<kThreads, uint32_t>(sh, 1, 0, nc, th, key_of, emit);
    return;
  }
  // Scores too near the border for FP32.  Few: rank them among themselves.
  for (int32_t i = tid; i < nc; i += kThreads) {
    const float s = key_score(key_of(i));
    if (s - vmax > two_e) {
      atomicAdd(&s_sure_n, 1);
    } else if (!(vmin - s > two_e)) {
      const int32_t at = atomicAdd(&s_near_n, 1);
      if (at < kNear) s_near[at] = i;
    }
  }
  __syncthreads();
  const int32_t near_n = s_near_n, wanted = pick - s_sure_n;
  if (near_n <= kNear) {
    for (int32_t i = warp; i < near_n; i += kWarps) {
      const uint64_t k = exact_key<T, HD>(base + (int64_t)s_near[i] * row, s_q, G, lane);
      if (lane == 0) s_near_key[i] = k;
    }
    __syncthreads();
    if (tid < near_n) {
      const uint64_t k = s_near_key[tid];
      const int32_t me = s_near[tid];
      int32_t before = 0;
      for (int32_t i = 0; i < near_n; ++i)
        before += s_near_key[i] > k || (s_near_key[i] == k && s_near[i] < me);
      s_lower[me] = before < wanted ? ~0u : 0u;
    }
    __syncthreads();
    // sure ones exceed `most`; the near ones no longer do unless they are wanted
    const Threshold<uint32_t> past{most, 0u, 0u, false};
    emit_chosen<kThreads, uint32_t>(sh, 1, 0, nc, past, key_of, emit);
    return;
  }
  // Many (equal scores, infinities): 64-bit keys for all.
  for (int32_t i = warp; i < nc; i += kWarps) {
    const float s = key_score(key_of(i));
    uint64_t key64;
    if (s - vmax > two_e) {
      key64 = ~0ull;
    } else if (vmin - s > two_e) {
      key64 = 0;
    } else {
      key64 = exact_key<T, HD>(base + (int64_t)i * row, s_q, G, lane);
    }
    __syncwarp();
    if (lane == 0) {
      s_lower[i] = (uint32_t)key64;
      s_upper[i] = (uint32_t)(key64 >> 32);
    }
  }
  __syncthreads();
  auto slot_of = keys_by([&](int32_t i) { return (uint64_t)s_upper[i] << 32 | s_lower[i]; });
  const Threshold<uint64_t> th64 = find_threshold<kThreads, uint64_t>(
      sh, 1, nc, (uint32_t)pick, (uint64_t)0, ~(uint64_t)0, slot_of);
  emit_chosen<kThreads, uint64_t>(sh, 1, 0, nc, th64, slot_of, emit);
}

template <class T, int HD, int GP>
int launch_select(const SelectRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                  std::string* err) {
  static ClusterKernel ck;
  int32_t br_shift = 0;
  while ((1 << br_shift) < r.block_rows) ++br_shift;
  const int64_t items = (int64_t)r.batch * r.n_kv;
  const int64_t max_nb = (((int64_t)r.max_n_pos + r.block_rows - 1) / r.block_rows + 3) / 4 * 4;
  if (max_nb > kMaxSelectBlocks) {
    *err = "too many blocks for one selection: use larger blocks";
    return GLA_ERR_NOT_SUPPORTED;
  }
  // as many CTAs a (sequence, kv head) as the device holds at once (a second wave would
  // start over with its queries' loads), while each still has 64 blocks
  const size_t smem = select_smem<T, HD, GP>(max_nb);
  int S = 1;
  while (S < 16 && max_nb > 64 * S && items * S * 2 <= 2 * dev.sms &&
         items <= clusters_held(block_select_kernel<T, HD, GP>, ck, kThreads,
                                select_smem<T, HD, GP>(4), 2 * S, dev))
    S *= 2;
  if (items * S > INT32_MAX) {
    *err = "batch * n_kv_heads too large";
    return GLA_ERR_NOT_SUPPORTED;
  }
  return launch_clusters(block_select_kernel<T, HD, GP>, (unsigned)(items * S), kThreads,
                         smem, S, ck, stream, "block selection", err, r.q,
                         reinterpret_cast<const T* const*>(r.bounds_ptrs), r.n_pos, r.max_n_pos,
                         r.block_ids, r.n_heads, r.n_kv, br_shift, r.n_sel, r.n_first, r.n_last, S,
                         (int32_t)max_nb, r.status);
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
