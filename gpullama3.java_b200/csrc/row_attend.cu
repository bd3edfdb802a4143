// row_attend.cu - decode attention over listed blocks of rows
// (gla_decode_blocks_*), and over all rows with each row's weight added to a
// running sum (gla_decode_weights_*).
//
//   xb_h = sum_t p_ht v_t,  p_ht = exp(scale q_h.k_t - m_h) / l_h,
//   w[g][t] += sum over the q heads h of kv head g of p_ht.
//
// HBM-bound: every listed row of K and V is read once for all G <= 8 q heads
// of its kv head.  One cluster of S CTAs works on one (sequence, kv head); the
// rows are dealt in units of 16 (FP16) or 8 (FP32) to the cluster's warps,
// round robin.  A block is a multiple of 16 rows, so a unit lies in one block,
// and a listed block costs one id lookup a unit.  Each warp streams its units
// through a ring of its own in shared memory (cp.async, 16 bytes a lane, rows
// past the last one zero-filled and never read) and keeps its own running
// maximum, sum and output: no block barrier inside the stream.  The warps join
// in shared memory and the CTAs through the cluster's shared memory, in a
// fixed order, so results do not depend on timing, and there is no workspace,
// counter or second launch.  Rows in shared memory are padded by 16 bytes: a
// row's pitch is an odd number of 16-byte chunks, which keeps ldmatrix and the
// vector loads free of bank conflicts.
//
// FP16 cache: mma.sync.m16n8k16.  The 16 rows of A hold the high halves of the
// (up to 8) q heads and their low halves, x - float(hi(x)): the two products
// add to about 22 bits of x, and the cache's FP16 values are exact, so the
// result has FP32 accuracy.  q is first scaled by a power of two to [1, 2) at
// its largest (so the low halves do not fall under FP16's range), p by 2^15
// (p <= 1; a weight of 2^-17 still has all 22 bits).  tcgen05 has no place
// here: 8 rows of a 128-row tile, and the stream is HBM-bound.
// FP32 cache: FP32 pairs on the CUDA cores.
//
// Weights: the normalisation is known only when all rows were seen, so the
// scores (log2 units) go to a workspace, G floats a row against 2 head_dim
// elements of K and V, and each CTA reads its own rows' scores again (from L2)
// after the cluster has joined its maxima and sums.
#include <cmath>

#include "cache_ops.cuh"

namespace gla {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPScale = 32768.0f;  // FP16 path: p enters the product times 2^15

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16-byte cp.async that reads `bytes` (16 or 0) and zero-fills the rest.
__device__ __forceinline__ void cp_async_16_zfill(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_half2(__half a, __half b) {
  const __half2 v = __halves2half2(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct AttendParams {
  const float* q;
  const void* const* k_ptrs;
  const void* const* v_ptrs;
  const int32_t* n_pos;
  int32_t max_n_pos;
  float* xb;
  int32_t n_heads, n_kv, S;
  int64_t kv_stride;
  float scale_log2;  // scale * log2(e)
  const int32_t* block_ids;
  int32_t n_sel, br_shift;
  float* const* weight_ptrs;
  int64_t weight_stride;
  float* scores;  // [batch][n_kv][max_n_pos][G]
  int32_t* status;
};

// Where unit u's rows start, or -1 if it has none.  kUnitShift: log2 of the
// rows of a unit.
template <bool BLOCKS, int kUnitShift>
__device__ __forceinline__ int32_t unit_row(const AttendParams& p, const int32_t* ids, int32_t u,
                                            int32_t n) {
  int64_t row;
  if constexpr (BLOCKS) {
    const int shift = p.br_shift - kUnitShift;  // units of a block, log2
    const int32_t id = __ldg(ids + (u >> shift));
    if (id < 0) return -1;
    row = ((int64_t)id << p.br_shift) + ((int64_t)(u & ((1 << shift) - 1)) << kUnitShift);
  } else {
    row = (int64_t)u << kUnitShift;
  }
  return row < n ? (int32_t)row : -1;
}

// Copies unit rows [row0, row0 + U) of K and V into a ring slot (K then V).
template <class T, int HD, int U>
__device__ __forceinline__ void load_unit(uint32_t slot, const T* k, const T* v, int64_t kv_stride,
                                          int32_t row0, int32_t n, int lane) {
  constexpr int kChunks = HD * (int)sizeof(T) / 16;
  constexpr int kPitch = HD * (int)sizeof(T) + 16;
  constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < U * kChunks / 32; ++i) {
    const int c = i * 32 + lane;
    const int r = c / kChunks, ch = c - r * kChunks;
    const int32_t row = row0 + r;
    const int bytes = row < n ? 16 : 0;
    const int64_t off = (int64_t)(row < n ? row : row0) * kv_stride + ch * kPer;
    const uint32_t dst = slot + r * kPitch + ch * 16;
    cp_async_16_zfill(dst, k + off, bytes);
    cp_async_16_zfill(dst + U * kPitch, v + off, bytes);
  }
}

template <class T, int HD>
constexpr int unit_rows() {
  return sizeof(T) == 2 ? 16 : 8;
}
template <class T, int HD>
constexpr int slot_bytes() {
  return 2 * unit_rows<T, HD>() * (HD * (int)sizeof(T) + 16);
}
// As deep a ring as one CTA an SM allows.
template <class T, int HD>
constexpr int ring_stages() {
  return 212 * 1024 / (kWarps * slot_bytes<T, HD>());
}

// ---------------------------------------------------------------------------
// One warp's state over its units: FP16 cache.
// ---------------------------------------------------------------------------
template <int HD, int GP>
struct WarpF16 {
  static constexpr int kUnit = 16;
  static constexpr int kPitch = HD * 2 + 16;
  uint32_t qa[HD / 16][4];  // A fragments: rows 0-7 the high, 8-15 the low halves of q
  float o[HD / 8][4];       // rows as qa, times kPScale; the two halves are added at the end
  float m, l;               // head lane / 4; l: this lane's share of the sum
  float factor;             // score = product * factor (log2 units)

  // q of the group's heads, scaled and split into shared memory, then to registers.
  __device__ __forceinline__ void init(const float* q, int G, float scale_log2, char* scratch,
                                       int warp, int lane) {
    __half* s_q = reinterpret_cast<__half*>(scratch);                 // [16][HD + 8]
    float* s_f = reinterpret_cast<float*>(scratch + 16 * kPitch);     // [8]
    {
      const int h = warp;  // one head a warp
      float x[HD / 32], big = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        x[i] = h < G ? q[(int64_t)h * HD + i * 32 + lane] : 0.f;
        big = fmaxf(big, fabsf(x[i]));
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
      const int e = (big > 0.f && big < INFINITY) ? ilogbf(big) : 0;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const float y = scalbnf(x[i], -e);
        const __half hi = __float2half_rn(y);
        s_q[h * (HD + 8) + i * 32 + lane] = hi;
        s_q[(h + 8) * (HD + 8) + i * 32 + lane] = __float2half_rn(y - __half2float(hi));
      }
      if (lane == 0) s_f[h] = scalbnf(scale_log2, e);
    }
    __syncthreads();
    // ldmatrix order: rows 0-7 | rows 8-15 of columns 0-7, then of columns 8-15
    const uint32_t base = smem_u32(s_q) + (lane & 15) * kPitch + (lane >> 4) * 16;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) ldmatrix_x4(qa[ks], base + ks * 32);
    factor = s_f[lane >> 2];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  template <bool WEIGHTS>
  __device__ __forceinline__ void step(uint32_t slot, int rows, float* scores, int G, float*,
                                       int lane) {
    float s[2][2];
    const int sub = lane >> 3, in = lane & 7;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
      const uint32_t base = slot + (nt * 8 + in) * kPitch + sub * 16;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ks += 2) {
        uint32_t b[4];
        ldmatrix_x4(b, base + ks * 32);
        mma_f16(c, qa[ks], b[0], b[1]);
        mma_f16(c, qa[ks + 1], b[2], b[3]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = nt * 8 + 2 * (lane & 3) + j;
        s[nt][j] = (c[j] + c[2 + j]) * factor;
        if (r >= rows) {
          s[nt][j] = -INFINITY;
        } else if (WEIGHTS && (lane >> 2) < G) {
          __stcg(scores + (int64_t)r * G + (lane >> 2), s[nt][j]);
        }
      }
    }
    float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float m_new = fmaxf(m, top);
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    if (__any_sync(0xffffffffu, m_new != m)) {
      const float a = m == m_new ? 1.f : exp2_approx(m - ref);
      l *= a;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] *= a;
      m = m_new;
    }
    uint32_t pa[4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      float p0 = exp2_approx(s[nt][0] - ref), p1 = exp2_approx(s[nt][1] - ref);
      l += p0 + p1;
      p0 *= kPScale;
      p1 *= kPScale;
      const __half h0 = __float2half_rn(p0), h1 = __float2half_rn(p1);
      pa[nt * 2] = pack_half2(h0, h1);
      pa[nt * 2 + 1] = pack_half2(__float2half_rn(p0 - __half2float(h0)),
                                  __float2half_rn(p1 - __half2float(h1)));
    }
    const uint32_t vbase = slot + kUnit * kPitch + ((sub & 1) * 8 + in) * kPitch + (sub >> 1) * 16;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
      uint32_t b[4];
      ldmatrix_x4_trans(b, vbase + j * 32);
      mma_f16(o[2 * j], pa, b[0], b[1]);
      mma_f16(o[2 * j + 1], pa, b[2], b[3]);
    }
  }

  // m, l and o of the warp into shared memory: o [8][HD], ml [8][2].
  __device__ __forceinline__ void store(float* so, float* ml, int lane) {
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int h = lane >> 2;
    if (h >= GP) return;
    if ((lane & 3) == 0) {
      ml[h * 2] = m;
      ml[h * 2 + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      const float2 v = make_float2((o[i][0] + o[i][2]) * (1.0f / kPScale),
                                   (o[i][1] + o[i][3]) * (1.0f / kPScale));
      *reinterpret_cast<float2*>(so + h * HD + i * 8 + 2 * (lane & 3)) = v;
    }
  }
};

// Sums N = 4 * GP values over the 16 lanes of a half-warp by halving exchanges;
// lane l then holds the values of row (l >> 2) & 3 and heads starting at
// (l & 3) * GP / 4 (GP < 4: head (l & 3) * GP >> 2), GP / 4 (at least one) of them.
template <int N>
__device__ __forceinline__ void half_warp_scatter(float (&v)[N], int lane) {
  int n = N;
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) {
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
}

// ---------------------------------------------------------------------------
// FP32 cache.  Scores: lane = (row group lane / 16, part lane % 16); a part
// holds HD / 16 channels of all heads of q in registers, a row group the rows
// rg, rg + 2, rg + 4, rg + 6 of a unit.  Outputs: a lane owns HD / 32 channels
// of every head.
// ---------------------------------------------------------------------------
template <int HD, int GP>
struct WarpF32 {
  static constexpr int kUnit = 8;
  static constexpr int kPitch = HD * 4 + 16;
  static constexpr int kPairs = HD / 32;       // channel pairs of a part
  static constexpr int kHpl = GP >= 4 ? GP / 4 : 1;
  static constexpr int kOwn = HD / 32;         // output channels of a lane
  uint64_t qr[GP][kPairs];
  float o[GP][kOwn];
  float m[kHpl], l[kHpl];
  float factor;

  // Channel of pair j of a part: part-major 8-byte chunks, 16 parts side by side.
  __device__ __forceinline__ void init(const float* q, int G, float scale_log2, char*, int,
                                       int lane) {
    const int part = lane & 15;
#pragma unroll
    for (int h = 0; h < GP; ++h) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        float2 x = make_float2(0.f, 0.f);
        if (h < G) x = *reinterpret_cast<const float2*>(q + (int64_t)h * HD + (j * 16 + part) * 2);
        qr[h][j] = pk2(x.x, x.y);
      }
#pragma unroll
      for (int j = 0; j < kOwn; ++j) o[h][j] = 0.f;
    }
    factor = scale_log2;
#pragma unroll
    for (int j = 0; j < kHpl; ++j) {
      m[j] = -INFINITY;
      l[j] = 0.f;
    }
  }

  template <bool WEIGHTS>
  __device__ __forceinline__ void step(uint32_t slot, int rows, float* scores, int G, float* sp,
                                       int lane) {
    const int part = lane & 15, rg = lane >> 4;
    float acc[4 * GP];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t base = slot + (rg + 2 * i) * kPitch + part * 8;
      uint64_t kx[kPairs];
#pragma unroll
      for (int j = 0; j < kPairs; ++j)
        asm volatile("ld.shared.b64 %0, [%1];" : "=l"(kx[j]) : "r"(base + j * 128));
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        uint64_t a = mul2(qr[h][0], kx[0]);
#pragma unroll
        for (int j = 1; j < kPairs; ++j) a = fma2(qr[h][j], kx[j], a);
        float x, y;
        upk2(a, x, y);
        acc[i * GP + h] = x + y;
      }
    }
    half_warp_scatter<4 * GP>(acc, lane);
    const int r = rg + 2 * ((lane >> 2) & 3);
    const int h0 = ((lane & 3) * GP) >> 2;
    // GP < 4: lanes that share a (row, head) hold the same sum; one of them counts
    const bool first = GP >= 4 || (((lane & 3) * GP) & 3) == 0;
    float a[kHpl];
    bool moved = false;
#pragma unroll
    for (int j = 0; j < kHpl; ++j) {
      float s = acc[j] * factor;
      if (r >= rows) {
        s = -INFINITY;
      } else if (WEIGHTS && first && h0 + j < G) {
        __stcg(scores + (int64_t)r * G + h0 + j, s);
      }
      float top = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float m_new = fmaxf(m[j], top);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      a[j] = m[j] == m_new ? 1.f : exp2_approx(m[j] - ref);
      moved |= m[j] != m_new;
      m[j] = m_new;
      const float pr = exp2_approx(s - ref);
      l[j] = l[j] * a[j] + (first ? pr : 0.f);
      // sp: p [8 rows][GP], then the factors of the old output [GP]
      if (first) sp[r * GP + h0 + j] = pr;
      if (first && r == 0) sp[8 * GP + h0 + j] = a[j];
    }
    const bool any = __any_sync(0xffffffffu, moved);
    __syncwarp();
    if (any) {
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const float x = sp[8 * GP + h];
#pragma unroll
        for (int j = 0; j < kOwn; ++j) o[h][j] *= x;
      }
    }
    const uint32_t vbase = slot + kUnit * kPitch;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      float v[kOwn];
      const uint32_t at = vbase + t * kPitch;
      if constexpr (kOwn == 4) {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                     : "r"(at + lane * 16));
      } else if constexpr (kOwn == 2) {
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(at + lane * 8));
      } else {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) v[j] = lds_f32(at + (j * 32 + lane) * 4);
      }
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const float pr = sp[t * GP + h];
#pragma unroll
        for (int j = 0; j < kOwn; ++j) o[h][j] = fmaf(pr, v[j], o[h][j]);
      }
    }
    __syncwarp();
  }

  __device__ __forceinline__ void store(float* so, float* ml, int lane) {
    const int h0 = ((lane & 3) * GP) >> 2;
#pragma unroll
    for (int j = 0; j < kHpl; ++j) {
      float x = l[j];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (GP == 1) {
        // lanes 0-3 hold the one head; only lane 0 of each quad counted
        x = __shfl_sync(0xffffffffu, x, 0);
      } else if (GP == 2) {
        x = __shfl_sync(0xffffffffu, x, lane & ~1);
      }
      if (lane < 4) {
        ml[(h0 + j) * 2] = m[j];
        ml[(h0 + j) * 2 + 1] = x;
      }
    }
#pragma unroll
    for (int h = 0; h < GP; ++h)
#pragma unroll
      for (int j = 0; j < kOwn; ++j)
        so[h * HD + (kOwn == 3 ? j * 32 + lane : lane * kOwn + j)] = o[h][j];
  }
};

template <class T, int HD, int GP>
struct WarpOf;
template <int HD, int GP>
struct WarpOf<__half, HD, GP> {
  using type = WarpF16<HD, GP>;
};
template <int HD, int GP>
struct WarpOf<float, HD, GP> {
  using type = WarpF32<HD, GP>;
};

// Shared memory: the warps' rings; after the stream the same bytes hold the
// warps' outputs [kWarps][GP][HD], then (m, l) [kWarps][GP][2].  Static: the
// CTA's joined output and (m, l), read by the other CTAs of the cluster.
template <class T, int HD, int GP, bool BLOCKS, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, 1) attend_kernel(const __grid_constant__ AttendParams p) {
  using Warp = typename WarpOf<T, HD, GP>::type;
  constexpr int U = Warp::kUnit;
  constexpr int kShift = U == 16 ? 4 : 3;
  constexpr int kStages = ring_stages<T, HD>();
  constexpr int kSlot = slot_bytes<T, HD>();
  extern __shared__ __align__(16) char s_ring[];
  __shared__ __align__(16) float s_o[GP * HD];
  __shared__ float s_ml[GP * 2];
  __shared__ float s_p[sizeof(T) == 4 ? kWarps * 9 * GP : 1];
  __shared__ float s_norm[GP * 2];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int S = p.S;
  const int rank = S > 1 ? (int)(blockIdx.x % (unsigned)S) : 0;
  const int item = (int)(blockIdx.x / (unsigned)S);
  const int b = item / p.n_kv, g = item - b * p.n_kv;
  const int G = p.n_heads / p.n_kv;
  int32_t n = clamped_rows(p.n_pos, b, p.max_n_pos, p.status);
  const T* k = static_cast<const T*>(p.k_ptrs[b]);
  const T* v = static_cast<const T*>(p.v_ptrs[b]);
  if (!usable_ptrs(k, v, p.status)) n = 0;
  float* wts = WEIGHTS ? p.weight_ptrs[b] : nullptr;
  if (WEIGHTS && !usable_weights(wts, p.status)) n = 0;
  k += (int64_t)g * HD;
  v += (int64_t)g * HD;
  const int32_t* ids = BLOCKS ? p.block_ids + (int64_t)item * p.n_sel : nullptr;
  const int32_t units = BLOCKS ? (n > 0 ? p.n_sel << (p.br_shift - kShift) : 0)
                               : (int32_t)(((int64_t)n + U - 1) / U);
  const int32_t first = rank * kWarps + warp, stride = S * kWarps;
  float* scores = WEIGHTS ? p.scores + (int64_t)item * p.max_n_pos * G : nullptr;

  const uint32_t ring = smem_u32(s_ring) + warp * (kStages * kSlot);
  Warp w;
  w.init(p.q + ((int64_t)b * p.n_heads + (int64_t)g * G) * HD, G, p.scale_log2, s_ring, warp, lane);

  // unit i of this warp is first + i * stride; its ring slot i % kStages
  const int32_t mine = units > first ? (units - first - 1) / stride + 1 : 0;
  int32_t row_of[kStages];
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    row_of[i] = -1;
    if (i < mine) {
      row_of[i] = unit_row<BLOCKS, kShift>(p, ids, first + i * stride, n);
      if (row_of[i] >= 0) load_unit<T, HD, U>(ring + i * kSlot, k, v, p.kv_stride, row_of[i], n, lane);
    }
    cp_async_commit();
  }
  for (int32_t i0 = 0; i0 < mine; i0 += kStages) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      const int32_t i = i0 + s;
      if (i < mine) {
        constexpr int kAhead = kStages - 1;
        const int ahead = (s + kAhead) % kStages;
        cp_async_wait<kStages - 2>();
        __syncwarp();  // unit i is here for every lane, and slot `ahead` is read out
        row_of[ahead] = -1;
        if (i + kAhead < mine) {
          row_of[ahead] = unit_row<BLOCKS, kShift>(p, ids, first + (i + kAhead) * stride, n);
          if (row_of[ahead] >= 0)
            load_unit<T, HD, U>(ring + ahead * kSlot, k, v, p.kv_stride, row_of[ahead], n, lane);
        }
        cp_async_commit();
        const int32_t row0 = row_of[s];
        if (row0 >= 0)
          w.template step<WEIGHTS>(ring + s * kSlot, n - row0, scores + (int64_t)row0 * G, G,
                                   s_p + warp * 9 * GP, lane);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // rings drained

  // warps -> CTA
  float* so = reinterpret_cast<float*>(s_ring);
  float* sml = so + kWarps * GP * HD;
  w.store(so + warp * GP * HD, sml + warp * GP * 2, lane);
  __syncthreads();
  for (int i = tid; i < GP * HD; i += kThreads) {
    const int h = i / HD;
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) top = fmaxf(top, sml[(x * GP + h) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float e = exp2_approx(sml[(x * GP + h) * 2] - ref);
      acc = fmaf(so[x * GP * HD + i], e, acc);
      sum = fmaf(sml[(x * GP + h) * 2 + 1], e, sum);
    }
    s_o[i] = acc;
    if (i == h * HD) {
      s_ml[h * 2] = top;
      s_ml[h * 2 + 1] = sum;
    }
  }
  cluster_barrier(S);

  // CTAs -> result: each rank joins its share of the G x HD outputs
  float* out = p.xb + ((int64_t)b * p.n_heads + (int64_t)g * G) * HD;
  for (int i = rank * kThreads + tid; i < G * HD; i += S * kThreads) {
    const int h = i / HD;
    float top = -INFINITY;
    for (int x = 0; x < S; ++x) top = fmaxf(top, S == 1 ? s_ml[h * 2] : *cluster_peer(&s_ml[h * 2], x));
    const float ref = top == -INFINITY ? 0.f : top;
    float acc = 0.f, sum = 0.f;
    for (int x = 0; x < S; ++x) {
      const float* ml = S == 1 ? &s_ml[h * 2] : cluster_peer(&s_ml[h * 2], x);
      const float* ox = S == 1 ? &s_o[i] : cluster_peer(&s_o[i], x);
      const float e = exp2_approx(ml[0] - ref);
      acc = fmaf(*ox, e, acc);
      sum = fmaf(ml[1], e, sum);
    }
    // no row at all: zeros (sum is 0 only then: the largest weight is 1, or NaN)
    out[i] = sum == 0.f ? 0.f : acc / sum;
  }
  if constexpr (WEIGHTS) {
    if (tid < GP) {
      float top = -INFINITY, sum = 0.f;
      for (int x = 0; x < S; ++x)
        top = fmaxf(top, S == 1 ? s_ml[tid * 2] : *cluster_peer(&s_ml[tid * 2], x));
      const float ref = top == -INFINITY ? 0.f : top;
      for (int x = 0; x < S; ++x) {
        const float* ml = S == 1 ? &s_ml[tid * 2] : cluster_peer(&s_ml[tid * 2], x);
        sum = fmaf(ml[1], exp2_approx(ml[0] - ref), sum);
      }
      s_norm[tid * 2] = ref;  // p = 2^(s - ref) / sum
      s_norm[tid * 2 + 1] = 1.0f / sum;
    }
  }
  cluster_barrier(S);  // no CTA leaves while another reads its shared memory
  if constexpr (WEIGHTS) {
    // this CTA's own rows, in the order their units were dealt
    float* wrow = wts + (int64_t)g * p.weight_stride;
    const int32_t cta_units = units > rank * kWarps ? (units - rank * kWarps - 1) / stride + 1 : 0;
    const int64_t all = (int64_t)cta_units * kWarps * U;
    for (int64_t i = tid; i < all; i += kThreads) {
      const int32_t round = (int32_t)(i / (kWarps * U)), in = (int32_t)(i - (int64_t)round * kWarps * U);
      const int64_t row = ((int64_t)rank * kWarps + (int64_t)round * stride) * U + in;
      if (row >= n) continue;
      const float* sc = scores + row * G;
      float x = 0.f;
      for (int h = 0; h < G; ++h)
        x = fmaf(exp2_approx(__ldcg(sc + h) - s_norm[h * 2]), s_norm[h * 2 + 1], x);
      wrow[row] += x;
    }
  }
}

template <class T, int HD, int GP, bool BLOCKS>
int launch_one(const AttendRequest& r, const DeviceInfo& dev, cudaStream_t stream,
               std::string* err) {
  static std::atomic<uint64_t> attr_done{0};
  constexpr bool WEIGHTS = !BLOCKS;
  constexpr int U = unit_rows<T, HD>();
  constexpr size_t ring = (size_t)kWarps * ring_stages<T, HD>() * slot_bytes<T, HD>();
  static_assert(ring >= (size_t)kWarps * GP * (HD + 2) * 4, "the outputs reuse the rings");
  static_assert(ring >= 16 * (HD * 2 + 16) + 32, "q is split in the rings");
  AttendParams p{};
  p.q = r.q;
  p.k_ptrs = r.k_ptrs;
  p.v_ptrs = r.v_ptrs;
  p.n_pos = r.n_pos;
  p.max_n_pos = r.max_n_pos;
  p.xb = r.xb;
  p.n_heads = r.n_heads;
  p.n_kv = r.n_kv;
  p.kv_stride = r.kv_stride;
  p.scale_log2 = r.scale * kLog2e;
  p.block_ids = r.block_ids;
  p.n_sel = r.n_sel;
  while (BLOCKS && (1 << p.br_shift) < r.block_rows) ++p.br_shift;
  p.weight_ptrs = r.weight_ptrs;
  p.weight_stride = r.weight_stride;
  p.scores = r.scores;
  p.status = r.status;
  const int64_t rows = BLOCKS ? std::min<int64_t>((int64_t)r.n_sel * r.block_rows, INT32_MAX)
                              : (int64_t)r.max_n_pos;
  const int64_t units = (rows + U - 1) / U;
  const int64_t items = (int64_t)r.batch * r.n_kv;
  // CTAs a (sequence, kv head): as many as fill the device once, while every
  // warp still has a unit
  int S = 1;
  while (S < 16 && items * S < dev.sms && units > (int64_t)kWarps * S) S *= 2;
  p.S = S;
  if (items * S > INT32_MAX) {
    *err = "batch * n_kv_heads too large";
    return GLA_ERR_NOT_SUPPORTED;
  }
  return launch_clusters(attend_kernel<T, HD, GP, BLOCKS, WEIGHTS>, (unsigned)(items * S), kThreads,
                         ring, S, attr_done, stream, "attention", err, p);
}

template <class T, int HD, int GP>
int by_mode(const AttendRequest& r, const DeviceInfo& dev, cudaStream_t stream, std::string* err) {
  return r.block_ids ? launch_one<T, HD, GP, true>(r, dev, stream, err)
                     : launch_one<T, HD, GP, false>(r, dev, stream, err);
}

template <int HD>
int by_group(const AttendRequest& r, const DeviceInfo& dev, cudaStream_t stream,
             std::string* err) {
  // FP16: the matrix instruction takes 8 heads whatever the group
  if (r.dtype == GLA_DTYPE_F16) return by_mode<__half, HD, 8>(r, dev, stream, err);
  const int G = r.n_heads / r.n_kv;
  if (G == 1) return by_mode<float, HD, 1>(r, dev, stream, err);
  if (G == 2) return by_mode<float, HD, 2>(r, dev, stream, err);
  if (G <= 4) return by_mode<float, HD, 4>(r, dev, stream, err);
  return by_mode<float, HD, 8>(r, dev, stream, err);
}

}  // namespace

size_t attend_score_floats(const AttendRequest& r) {
  return (size_t)r.batch * r.n_heads * (size_t)r.max_n_pos;
}

int launch_attend(const AttendRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                  std::string* err) {
  switch (r.head_dim) {
    case 64: return by_group<64>(r, dev, stream, err);
    case 96: return by_group<96>(r, dev, stream, err);
    default: return by_group<128>(r, dev, stream, err);
  }
}

}  // namespace gla
