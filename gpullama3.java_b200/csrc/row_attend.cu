// row_attend.cu - decode attention over listed blocks of rows
// (gla_decode_blocks_*), and over all rows with each row's weight added to a
// running sum (gla_decode_weights_*).
//
//   xb_h = sum_t p_ht v_t,  p_ht = exp(scale q_h.k_t - m_h) / l_h,
//   w[g][t] += sum over the q heads h of kv head g of p_ht.
//
// HBM-bound: every listed row of K and V is read once for all G <= 8 q heads of
// its kv head.  One cluster of S CTAs works on one (sequence, kv head); the rows
// are dealt in units of 16 (FP16) or 8 (FP32) to the cluster's warps, round robin.
// A block is a multiple of 16 rows, so a unit lies in one block, and a listed block
// costs one id lookup a unit.  Each warp streams its units through a ring of its own
// in shared memory (cp.async, 16 bytes a lane, rows past the last one zero-filled
// and never read) and keeps its own running maximum, sum and output: no block
// barrier inside the stream.  The warps join in shared memory and the CTAs through
// the cluster's shared memory, in a fixed order, so results do not depend on timing.
// Long lists of few kv heads are cut into parts, one CTA each, that a second kernel
// joins (list_part_rows_for).  Rows in shared
// memory are padded by 16 bytes: a row's pitch is an odd number of 16-byte chunks,
// which keeps ldmatrix and the vector loads free of bank conflicts.  (One bulk copy
// a row instead of 16 cp.async a lane: 320 us against 244 for 256 queries over
// listed blocks; the copy engine takes short pieces more slowly.)
//
// FP16 cache: mma.sync.m16n8k16.  The 16 rows of A hold the high halves of the
// (up to 8) q heads and their low halves, x - float(hi(x)): the two products
// add to about 22 bits of x, and the cache's FP16 values are exact, so the
// result has FP32 accuracy.  q is first scaled by a power of two to [1, 2) at
// its largest (so the low halves do not fall under FP16's range), p by 2^15
// (p <= 1; a weight of 2^-17 still has all 22 bits).  tcgen05 has no place
// here: 8 rows of a 128-row tile, and the stream is HBM-bound.
// FP32 cache: the same with mma.sync.m16n8k8 on TF32 halves (split_tf32) of q and p
// (the two row halves of A) and of K and V (two products).  On the CUDA cores a unit
// of 8 rows and 8 heads took about 600 instructions, this way about 330, whatever the
// group (16 sequences of 77 to 8191 rows, groups of 8: 47 us and 36).
// Rows are taken to be finite: an infinite key or value makes a half a NaN.
//
// Weights: the normalisation is known only when all rows were seen, so the scores
// (log2 units) go to a workspace, G floats a row against 2 head_dim elements of K
// and V (read with an evict-first hint, so the scores stay in L2), and are read again
// to add the weights.  Long sequences: the rows are cut into parts of equal size, one
// CTA each, so that a ragged batch still fills the device evenly, and a second kernel
// joins the parts and adds the weights (part_rows_for).
//
// Measured on one B200: listed blocks, 64 of 64 FP16 rows for 4 kv heads of 128
// 8.6 us (latency: 131 KB an SM through 64 bytes a clock, then the joins); 256
// queries over one cache of 32,768 rows, 32 blocks each, 220 us (2.1 GB through L2,
// 9.8 TB/s, as every query and kv head reads its own rows); 64 separate FP16 caches 105 us, 5.1 TB/s.  Weights, 131,072 FP16 rows of
// 4 kv heads 58 us (4.7 TB/s with scores and weights).
#include <cmath>

#include "cache_ops.cuh"

namespace gla {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPScale = 32768.0f;  // FP16 path: p enters the product times 2^15

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16-byte cp.async that reads `bytes` (16 or 0) and zero-fills the rest; ONCE:
// data that is read once, first to leave L2.
template <bool ONCE>
__device__ __forceinline__ void cp_async_16_zfill(uint32_t dst, const void* src, int bytes,
                                                  uint64_t policy) {
  if constexpr (ONCE) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst),
                 "l"(src), "r"(bytes), "l"(policy)
                 : "memory");
  } else {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
  }
}
template <bool ONCE>
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint64_t policy) {
  if constexpr (ONCE) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst),
                 "l"(src), "l"(policy)
                 : "memory");
  } else {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  }
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
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// x = hi + lo, up to what the matrix instruction drops of lo: hi is x rounded to
// TF32's 11 bits, so |lo| is at most 2^12 units of x's last place (2^-23 of its
// power of two), and of its 12 bits 11 count: one unit at most is lost.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
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
  int32_t n_heads, n_kv;
  int32_t S;          // CTAs of an item: a cluster, or (part != null) parts joined later
  uint32_t kv_bytes;  // of a cache row
  float scale_log2;  // scale * log2(e)
  const int32_t* block_ids;
  int32_t n_sel, br_shift;
  float* const* weight_ptrs;
  int64_t weight_stride;
  float* scores;      // [item][G][score_pitch]
  int64_t score_pitch;
  float* part;        // o of the parts: [item][S][G][HD]
  float2* part_ml;    // their (m, l): [item][G][S]
  int32_t part_units;  // of a part
  int32_t* status;
};

// Where unit u's rows start, or -1 if it has none, from the id of its block (all
// rows: no id).  kUnitShift: log2 of the rows of a unit.
template <bool BLOCKS, int kUnitShift>
__device__ __forceinline__ int32_t unit_row(int32_t br_shift, int32_t id, int32_t u, int32_t n) {
  int64_t row;
  if constexpr (BLOCKS) {
    const int shift = br_shift - kUnitShift;  // units of a block, log2
    if (id < 0) return -1;
    row = ((int64_t)id << br_shift) + ((int64_t)(u & ((1 << shift) - 1)) << kUnitShift);
  } else {
    row = (int64_t)u << kUnitShift;
  }
  return row < n ? (int32_t)row : -1;
}

// Copies unit rows [row0, row0 + U) of K and V into a ring slot (K then V);
// rows from n on are zero-filled, not read.
template <class T, int HD, int U, bool ONCE>
__device__ __forceinline__ void load_unit(uint32_t slot, const T* k, const T* v, uint32_t kv_bytes,
                                          int32_t row0, int32_t n, uint64_t policy, int lane) {
  constexpr int kChunks = HD * (int)sizeof(T) / 16;
  constexpr int kPitch = HD * (int)sizeof(T) + 16;
  const char* kr = reinterpret_cast<const char*>(k) + (uint64_t)(uint32_t)row0 * kv_bytes;
  const char* vr = reinterpret_cast<const char*>(v) + (uint64_t)(uint32_t)row0 * kv_bytes;
  if (n - row0 >= U) {
#pragma unroll
    for (int i = 0; i < U * kChunks / 32; ++i) {
      const uint32_t c = i * 32 + lane, r = c / kChunks, ch = c - r * kChunks;
      const uint32_t dst = slot + r * kPitch + ch * 16;
      const uint64_t off = (uint64_t)r * kv_bytes + ch * 16;
      cp_async_16<ONCE>(dst, kr + off, policy);
      cp_async_16<ONCE>(dst + U * kPitch, vr + off, policy);
    }
  } else {
#pragma unroll
    for (int i = 0; i < U * kChunks / 32; ++i) {
      const uint32_t c = i * 32 + lane, r = c / kChunks, ch = c - r * kChunks;
      const int bytes = (int32_t)r < n - row0 ? 16 : 0;
      const uint32_t dst = slot + r * kPitch + ch * 16;
      const uint64_t off = bytes ? (uint64_t)r * kv_bytes + ch * 16 : 0;
      cp_async_16_zfill<ONCE>(dst, kr + off, bytes, policy);
      cp_async_16_zfill<ONCE>(dst + U * kPitch, vr + off, bytes, policy);
    }
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
// Two shapes of CTA.  Wide: 8 warps with a ring as deep as one CTA an SM
// allows, for calls whose clusters do not fill the device; a warp's few units
// are then all in flight at once.  Slim: 4 warps with rings of 72 KB in all,
// three CTAs an SM (168 registers a thread): 12 warps hide the dependent steps
// of a unit (product, maximum, exponential, product), which 8 warps do not, and
// one CTA streams while another starts or joins.
template <class T, int HD, bool WIDE>
struct Cta {
  static constexpr int kWarps = WIDE ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kBudget = (WIDE ? 212 : 70) * 1024;
  static constexpr int kStages = kBudget / (kWarps * slot_bytes<T, HD>());
  static constexpr int kRing = kWarps * kStages * slot_bytes<T, HD>();
  static constexpr int kMinCtas = WIDE ? 1 : 3;
  static_assert(kStages >= 2, "a unit in flight beside the one at work");
};

// ---------------------------------------------------------------------------
// One warp's state over its units: FP16 cache.
// ---------------------------------------------------------------------------
template <int HD>
struct WarpF16 {
  static constexpr int kUnit = 16;
  static constexpr int kPitch = HD * 2 + 16;
  uint32_t qa[HD / 16][4];  // A fragments: rows 0-7 the high, 8-15 the low halves of q
  float o[HD / 8][4];       // rows as qa, times kPScale; the two halves are added at the end
  float m, l;               // head lane / 4; l: this lane's share of the sum
  float factor;             // score = product * factor (log2 units)

  // q of the group's heads, scaled and split into shared memory, then to registers.
  static constexpr int kQBytes = 16 * kPitch + 32;

  // This thread's part of q, loaded ahead of its use: a warp takes every W-th head.
  template <int W>
  struct Query {
    float x[8 / W][HD / 32];
    __device__ __forceinline__ void load(const float* q, int G, int warp, int lane) {
#pragma unroll
      for (int j = 0; j < 8 / W; ++j)
#pragma unroll
        for (int i = 0; i < HD / 32; ++i)
          x[j][i] = warp + j * W < G ? __ldg(q + (warp + j * W) * HD + i * 32 + lane) : 0.f;
    }
  };

  template <int W>
  __device__ __forceinline__ void init(const Query<W>& in, float scale_log2, char* scratch,
                                       int warp, int lane) {
    const auto& x = in.x;
    __half* s_q = reinterpret_cast<__half*>(scratch);                 // [16][HD + 8]
    float* s_f = reinterpret_cast<float*>(scratch + 16 * kPitch);     // [8]
#pragma unroll
    for (int j = 0; j < 8 / W; ++j) {
      const int h = warp + j * W;
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) big = fmaxf(big, fabsf(x[j][i]));
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
      const int e = (big > 0.f && big < INFINITY) ? ilogbf(big) : 0;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const float y = scalbnf(x[j][i], -e);
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
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  template <bool WEIGHTS>
  __device__ __forceinline__ void step(const char* slot_ptr, int rows, float* scores, int64_t pitch,
                                       int G, const char*, int lane) {
    const uint32_t slot = smem_u32(slot_ptr);
    float s[2][2];
    const int sub = lane >> 3, in = lane & 7;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      // accumulators of 32 channels each, added in FP32: the matrix instruction
      // truncates, and a chain over all channels did so on the whole sum
      // (1.5e-6 of the output over 131,072 rows; 0.7e-6 this way), and waited longer
      float c[HD / 32][4];
      const uint32_t base = slot + (nt * 8 + in) * kPitch + sub * 16;
      // (products of one accumulator apart: a product waits 21 clocks for the last)
      uint32_t bk[HD / 32][4];
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {
        c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
        ldmatrix_x4(bk[j], base + j * 64);
      }
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) mma_f16(c[j], qa[2 * j], bk[j][0], bk[j][1]);
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) mma_f16(c[j], qa[2 * j + 1], bk[j][2], bk[j][3]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = nt * 8 + 2 * (lane & 3) + j;
        float hi = c[0][j], lo = c[0][2 + j];
#pragma unroll
        for (int i = 1; i < HD / 32; ++i) {
          hi += c[i][j];
          lo += c[i][2 + j];
        }
        s[nt][j] = r < rows ? (hi + lo) * factor : -INFINITY;
      }
      if (WEIGHTS && (lane >> 2) < G)  // the pitch has room for a whole unit
        __stcg(reinterpret_cast<float2*>(scores + (lane >> 2) * pitch + nt * 8 + 2 * (lane & 3)),
               make_float2(s[nt][0], s[nt][1]));
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

// ---------------------------------------------------------------------------
// FP32 cache.  The fragments of q, both halves, lie in shared memory in the order
// the lanes read them.  A product's row order within a unit is free: C of the
// scores leaves a lane rows 2 (lane & 3) and + 1, which are k indices lane & 3 and
// + 4 of the second product, so p needs no exchange; and a lane's two output
// columns of a pair of tiles are neighbours, read by one 8-byte load.  With
// pitches of HD + 4 floats all these loads are free of bank conflicts.
// ---------------------------------------------------------------------------
template <int HD>
struct WarpF32 {
  static constexpr int kUnit = 8;
  static constexpr int kPitch = HD * 4 + 16;
  float o[HD / 8][4];  // tile pair j: columns 16 j + 2 n (tile 2 j) and + 1 (tile 2 j + 1)
  float m, l;          // head lane / 4; l: this lane's share of the sum
  float factor;

  static constexpr int kQBytes = HD / 8 * 32 * 16;

  // This thread's part of q, loaded ahead of its use.  The fragment of step ks is
  // (hi, lo) of channels 8 ks + (lane & 3) and + 4 of head lane / 4; a warp takes
  // every W-th step.
  template <int W>
  struct Query {
    static constexpr int kSteps = (HD / 8 + W - 1) / W;
    float x[kSteps], y[kSteps];
    __device__ __forceinline__ void load(const float* q, int G, int warp, int lane) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const int h = lane >> 2, ch = (warp + j * W) * 8 + (lane & 3);
        const bool in = h < G && ch < HD;
        x[j] = in ? __ldg(q + h * HD + ch) : 0.f;
        y[j] = in ? __ldg(q + h * HD + ch + 4) : 0.f;
      }
    }
  };

  template <int W>
  __device__ __forceinline__ void init(const Query<W>& in, float scale_log2, char* scratch,
                                       int warp, int lane) {
    uint4* s_q = reinterpret_cast<uint4*>(scratch);
#pragma unroll
    for (int j = 0; j < Query<W>::kSteps; ++j) {
      if (warp + j * W < HD / 8) {
        uint4 f;
        split_tf32(in.x[j], f.x, f.y);
        split_tf32(in.y[j], f.z, f.w);
        s_q[(warp + j * W) * 32 + lane] = f;
      }
    }
    __syncthreads();
    factor = scale_log2;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  template <bool WEIGHTS>
  __device__ __forceinline__ void step(const char* slot, int rows, float* scores, int64_t pitch,
                                       int G, const char* scratch, int lane) {
    const uint4* s_q = reinterpret_cast<const uint4*>(scratch);
    // scores: accumulators of 32 channels each, added in FP32 (see WarpF16)
    float c[HD / 32][4];
    const float* kbase =
        reinterpret_cast<const float*>(slot + (lane >> 2) * kPitch) + (lane & 3);
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 a[HD / 32];
      uint32_t l0[HD / 32], l1[HD / 32];
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {
        const int ks = 4 * j + i;
        uint32_t h0, h1;
        a[j] = s_q[ks * 32 + lane];
        split_tf32(kbase[ks * 8], h0, l0[j]);
        split_tf32(kbase[ks * 8 + 4], h1, l1[j]);
        mma_tf32(c[j], a[j], h0, h1);
      }
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) mma_tf32(c[j], a[j], l0[j], l1[j]);
    }
    float s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float hi = c[0][j], lo = c[0][2 + j];
#pragma unroll
      for (int i = 1; i < HD / 32; ++i) {
        hi += c[i][j];
        lo += c[i][2 + j];
      }
      s[j] = 2 * (lane & 3) + j < rows ? (hi + lo) * factor : -INFINITY;
    }
    if (WEIGHTS && (lane >> 2) < G)
      __stcg(reinterpret_cast<float2*>(scores + (lane >> 2) * pitch + 2 * (lane & 3)),
             make_float2(s[0], s[1]));
    float top = fmaxf(s[0], s[1]);
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
    const float p0 = exp2_approx(s[0] - ref), p1 = exp2_approx(s[1] - ref);
    l += p0 + p1;
    uint4 pa;  // k index lane & 3: row 2 (lane & 3); + 4: the row after it
    split_tf32(p0, pa.x, pa.y);
    split_tf32(p1, pa.z, pa.w);
    const float2* vbase = reinterpret_cast<const float2*>(
                              slot + kUnit * kPitch + 2 * (lane & 3) * kPitch) + (lane >> 2);
#pragma unroll
    for (int j = 0; j < HD / 16; j += 2) {
      uint32_t lo[4][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // this lane's two columns of its two rows
        const float2 v0 = vbase[(j + e) * 8], v1 = vbase[(j + e) * 8 + kPitch / 8];
        uint32_t h0, h1;
        split_tf32(v0.x, h0, lo[2 * e][0]);
        split_tf32(v1.x, h1, lo[2 * e][1]);
        mma_tf32(o[2 * (j + e)], pa, h0, h1);
        split_tf32(v0.y, h0, lo[2 * e + 1][0]);
        split_tf32(v1.y, h1, lo[2 * e + 1][1]);
        mma_tf32(o[2 * (j + e) + 1], pa, h0, h1);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) mma_tf32(o[2 * j + e], pa, lo[e][0], lo[e][1]);
    }
  }

  __device__ __forceinline__ void store(float* so, float* ml, int lane) {
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int h = lane >> 2;
    if ((lane & 3) == 0) {
      ml[h * 2] = m;
      ml[h * 2 + 1] = l;
    }
    // C of a tile: columns n = 2 (lane & 3) and + 1 of head h
#pragma unroll
    for (int j = 0; j < HD / 16; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = 2 * (lane & 3) + e;
        *reinterpret_cast<float2*>(so + h * HD + 16 * j + 2 * n) =
            make_float2(o[2 * j][e] + o[2 * j][2 + e], o[2 * j + 1][e] + o[2 * j + 1][2 + e]);
      }
  }
};

template <class T, int HD>
struct WarpOf;
template <int HD>
struct WarpOf<__half, HD> {
  using type = WarpF16<HD>;
};
template <int HD>
struct WarpOf<float, HD> {
  using type = WarpF32<HD>;
};

constexpr int GP = 8;  // heads of a product's row halves

// The weight of a row, all heads of the group: sc its scores, norm (m, 1 / l) of each head.
__device__ __forceinline__ float row_weight(const float* sc, int64_t pitch, const float* norm,
                                            int G) {
  float s[GP], x = 0.f;
#pragma unroll
  for (int h = 0; h < GP; ++h) s[h] = h < G ? __ldcg(sc + h * pitch) : 0.f;
#pragma unroll
  for (int h = 0; h < GP; ++h)
    if (h < G) x = fmaf(exp2_approx(s[h] - norm[h * 2]), norm[h * 2 + 1], x);
  return x;
}

// Shared memory: the warps' rings; after the stream the same bytes hold the
// warps' outputs [kWarps][GP][HD] and (m, l) [kWarps][GP][2], then the CTA's joined
// output [GP][HD], which the other CTAs of the cluster read as they do s_ml.
template <class T, int HD, bool BLOCKS, bool WIDE>
__global__ void __launch_bounds__(Cta<T, HD, WIDE>::kThreads, Cta<T, HD, WIDE>::kMinCtas)
    attend_kernel(const __grid_constant__ AttendParams p) {
  using Warp = typename WarpOf<T, HD>::type;
  using C = Cta<T, HD, WIDE>;
  constexpr bool WEIGHTS = !BLOCKS;
  constexpr int kWarps = C::kWarps, kThreads = C::kThreads, kStages = C::kStages;
  constexpr int U = Warp::kUnit;
  constexpr int kShift = U == 16 ? 4 : 3;
  constexpr int kSlot = slot_bytes<T, HD>();
  extern __shared__ __align__(16) char s_ring[];
  __shared__ float s_ml[GP * 2];
  __shared__ __align__(16) char s_q[Warp::kQBytes];  // q, split
  // wide CTAs of a cluster: what the others send, this rank's share of their outputs
  // [S][share] and all their (m, l) [S][GP][2]
  __shared__ float s_recv[WIDE ? GP * HD + 16 : 1];
  __shared__ float s_recv_ml[WIDE ? 16 * GP * 2 : 1];
  __shared__ float s_norm[GP * 2];
  __shared__ float s_wt[kWarps][GP];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int S = p.S;
  const int rank = S > 1 ? (int)(blockIdx.x % (unsigned)S) : 0;
  int item = (int)(blockIdx.x / (unsigned)S);
  int b = item / p.n_kv, g = item - b * p.n_kv;
  if (BLOCKS) {
    // Kv head by kv head: queries over one cache (a prompt chunk) then find their
    // head's rows in L2 (256 queries over 32,768 rows of 2 x 2 KB: 211 us against
    // 252 query by query; separate caches: no difference).
    const int batch = (int)(gridDim.x / (unsigned)S) / p.n_kv;
    g = item / batch;
    b = item - g * batch;
    item = b * p.n_kv + g;
  }
  const int G = p.n_heads / p.n_kv;
  pdl_wait();
  // A join that follows is let in only behind the stream: its CTAs would take the
  // first free places of this kernel's SMs and crowd there (109 us against 73 for
  // 131,072 rows).
  if (!p.part) pdl_launch_dependents();
  // q, the first units' ids, the length and the pointers are loaded side by side
  typename Warp::template Query<kWarps> query;
  query.load(p.q + ((int64_t)b * p.n_heads + (int64_t)g * G) * HD, G, warp, lane);
  const int32_t* ids = BLOCKS ? p.block_ids + (int64_t)item * p.n_sel : nullptr;
  const int32_t listed = BLOCKS ? p.n_sel << (p.br_shift - kShift) : 0;
  auto id_of = [&](int32_t u) {
    return BLOCKS && u < listed ? __ldg(ids + (u >> (p.br_shift - kShift))) : -1;
  };
  // units of this CTA's warps: a cluster's deal, or this part's
  const int32_t cta_first = rank * (p.part ? p.part_units : kWarps);
  const int32_t stride = p.part ? kWarps : S * kWarps;
  int32_t id[kStages + 1];
#pragma unroll
  for (int s = 0; s <= kStages; ++s) id[s] = id_of(cta_first + s * stride + warp);
  int32_t n = clamped_rows(p.n_pos, b, p.max_n_pos, p.status);
  if (WEIGHTS && p.part && (int64_t)rank * p.part_units * U >= n) return;
  const T* k = static_cast<const T*>(p.k_ptrs[b]);
  const T* v = static_cast<const T*>(p.v_ptrs[b]);
  if (!usable_ptrs(k, v, p.status)) n = 0;
  float* wts = WEIGHTS ? p.weight_ptrs[b] : nullptr;
  if (WEIGHTS && !usable_weights(wts, p.status)) n = 0;
  k += (int64_t)g * HD;
  v += (int64_t)g * HD;
  int32_t units = BLOCKS ? (n > 0 ? listed : 0) : (int32_t)(((int64_t)n + U - 1) / U);
  if (p.part) units = min(units, cta_first + p.part_units);
  const int32_t first = cta_first + warp;
  float* scores = WEIGHTS ? p.scores + (int64_t)item * G * p.score_pitch : nullptr;

  const uint32_t ring = smem_u32(s_ring) + warp * (kStages * kSlot);
  const uint64_t policy = WEIGHTS ? l2_evict_first_policy() : 0;

  // unit i of this warp is first + i * stride; its ring slot i % kStages.  A slot
  // is filled again as soon as it is read out, so while a warp waits for a unit the
  // ring's other units are under way too.
  int32_t mine = units > first ? (units - first - 1) / stride + 1 : 0;
  int32_t row_of[kStages];
  auto fetch = [&](int s, int32_t i, int32_t id) {
    row_of[s] = -1;
    if (i < mine) {
      row_of[s] = unit_row<BLOCKS, kShift>(p.br_shift, id, first + i * stride, n);
      if (row_of[s] >= 0)
        load_unit<T, HD, U, WEIGHTS>(ring + s * kSlot, k, v, p.kv_bytes, row_of[s], n, policy, lane);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) fetch(s, s, id[s]);
  int32_t next_id = id[kStages];  // ids are loaded a step before the rows they name
  if (WIDE) cluster_arrive(S);
  const int32_t tail_id = BLOCKS && p.n_sel - 32 + lane >= 0 ? __ldg(ids + p.n_sel - 32 + lane) : -1;
  Warp w;  // while the first units are under way
  w.template init<kWarps>(query, p.scale_log2, s_q, warp, lane);
  // A list counts up to its last id that names rows: the short sequences of a batch
  // leave much of theirs empty, and an empty unit too costs a warp a step (960 lists of
  // up to 4 blocks of 64 rows in 64 slots: 45 us, in 4 slots 19).
  if (BLOCKS && mine > kStages) {
    int32_t used = 0;
    for (int32_t end = p.n_sel; end > 0 && used == 0; end -= 32) {
      const int32_t i = end - 32 + lane;
      const int32_t last = end == p.n_sel ? tail_id : i < 0 ? -1 : __ldg(ids + i);
      const unsigned named = __ballot_sync(
          0xffffffffu, last >= 0 && ((int64_t)last << p.br_shift) < n);
      if (named) used = end - __clz((int)named);
    }
    units = min(units, used << (p.br_shift - kShift));
    mine = units > first ? (units - first - 1) / stride + 1 : 0;
  }
  for (int32_t i0 = 0; i0 < mine; i0 += kStages) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      if (i0 + s < mine) {
        cp_async_wait<kStages - 1>();
        __syncwarp();  // the unit is here for every lane
        if (row_of[s] >= 0)
          w.template step<WEIGHTS>(s_ring + (warp * kStages + s) * kSlot, n - row_of[s], scores + row_of[s],
                                   p.score_pitch, G, s_q, lane);
        __syncwarp();  // and read out by every lane
        fetch(s, i0 + s + kStages, next_id);
        next_id = id_of(first + (i0 + s + kStages + 1) * stride);
      }
    }
  }
  cp_async_wait<0>();
  if (p.part) pdl_launch_dependents();
  __syncthreads();  // rings drained

  // warps -> CTA
  float* so = reinterpret_cast<float*>(s_ring);
  float* sml = so + kWarps * GP * HD;
  float* s_o = sml + kWarps * GP * 2;
  w.store(so + warp * GP * HD, sml + warp * GP * 2, lane);
  __syncthreads();
  // each head's largest m, its sum, and the warps' weights relative to it
  if (tid < GP * kWarps) {
    const int x = tid / GP, h = tid % GP;
    float top = -INFINITY;
#pragma unroll
    for (int y = 0; y < kWarps; ++y) top = fmaxf(top, sml[(y * GP + h) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
    s_wt[x][h] = exp2_approx(sml[(x * GP + h) * 2] - ref);
    if (x == 0) {
      float sum = 0.f;
#pragma unroll
      for (int y = 0; y < kWarps; ++y)
        sum = fmaf(sml[(y * GP + h) * 2 + 1], exp2_approx(sml[(y * GP + h) * 2] - ref), sum);
      s_ml[h * 2] = top;
      s_ml[h * 2 + 1] = sum;
    }
  }
  __syncthreads();
  auto cta_o = [&](int i) {
    float acc = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) acc = fmaf(so[x * GP * HD + i], s_wt[x][i / HD], acc);
    return acc;
  };
  // the outputs of a list of (o, m, l): o_of(x) and ml_of(x, h) of rank x
  float* out = p.xb + ((int64_t)b * p.n_heads + (int64_t)g * G) * HD;
  auto joined_ml = [&](int h, auto ml_of) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int x = 0; x < S; ++x) top = fmaxf(top, ml_of(x, h)[0]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
    for (int x = 0; x < S; ++x) sum = fmaf(ml_of(x, h)[1], exp2_approx(ml_of(x, h)[0] - ref), sum);
    return make_float2(ref, sum);
  };
  auto joined_o = [&](int i, auto o_of, auto ml_of) {
    const int h = i / HD;
    const float2 rs = joined_ml(h, ml_of);
    float acc = 0.f;
#pragma unroll 4
    for (int x = 0; x < S; ++x) acc = fmaf(*o_of(x), exp2_approx(ml_of(x, h)[0] - rs.x), acc);
    // no row at all: zeros (the sum is 0 only then: the largest weight is 1, or NaN)
    out[i] = rs.y == 0.f ? 0.f : acc / rs.y;
  };
  auto norm_of = [&](auto ml_of) {  // p = 2^(s - ref) / sum
    if (tid < GP) {
      const float2 rs = joined_ml(tid, ml_of);
      s_norm[tid * 2] = rs.x;
      s_norm[tid * 2 + 1] = 1.0f / rs.y;
    }
    __syncthreads();
  };
  if (p.part) {  // joined by attend_join_kernel
    float* part = p.part + ((int64_t)item * S + rank) * G * HD;
    for (int i = tid; i < G * HD; i += kThreads) part[i] = cta_o(i);
    if (tid < G)
      p.part_ml[((int64_t)item * G + tid) * S + rank] = make_float2(s_ml[tid * 2], s_ml[tid * 2 + 1]);
    return;
  }
  if (WIDE && S > 1) {
    // every rank sends each other one its share: one barrier, and local reads behind it
    const int share = (G * HD + S - 1) / S;
    cluster_wait(S);  // all CTAs run: their shared memory may be written
    for (int i = tid; i < S * G; i += kThreads) {
      const int r = i / G, h = i - r * G;
      float* dst = const_cast<float*>(cluster_peer(s_recv_ml, r)) + (rank * GP + h) * 2;
      dst[0] = s_ml[h * 2];
      dst[1] = s_ml[h * 2 + 1];
    }
    for (int i = tid; i < G * HD; i += kThreads) {
      const int r = i / share;
      const_cast<float*>(cluster_peer(s_recv, r))[rank * share + i - r * share] = cta_o(i);
    }
    cluster_barrier(S);
    auto ml_of = [&](int x, int h) { return s_recv_ml + (x * GP + h) * 2; };
    const int i0 = rank * share;
    for (int i = tid; i < min(share, G * HD - i0); i += kThreads)
      joined_o(i0 + i, [&](int x) { return s_recv + x * share + i; }, ml_of);
    if (WEIGHTS) norm_of(ml_of);
  } else {
    for (int i = tid; i < GP * HD; i += kThreads) s_o[i] = cta_o(i);
    cluster_barrier(S);
    auto ml_of = [&](int x, int h) {
      return S == 1 ? &s_ml[h * 2] : cluster_peer(&s_ml[h * 2], x);
    };
    for (int i = rank * kThreads + tid; i < G * HD; i += S * kThreads)
      joined_o(i, [&](int x) { return S == 1 ? &s_o[i] : cluster_peer(&s_o[i], x); }, ml_of);
    if (WEIGHTS) norm_of(ml_of);
    if (S > 1) cluster_barrier(S);  // no CTA leaves while another reads its shared memory
  }
  if constexpr (WEIGHTS) {
    // this CTA's own rows, in the order their units were dealt
    float* wrow = wts + (int64_t)g * p.weight_stride;
    const int32_t cta_units = units > cta_first ? (units - cta_first - 1) / stride + 1 : 0;
    const int64_t all = (int64_t)cta_units * kWarps * U;
    for (int64_t i = tid; i < all; i += kThreads) {
      const int32_t round = (int32_t)(i / (kWarps * U)), in = (int32_t)(i - (int64_t)round * kWarps * U);
      const int64_t row = ((int64_t)cta_first + (int64_t)round * stride) * U + in;
      if (row < n) wrow[row] += row_weight(scores + row, p.score_pitch, s_norm, G);
    }
  }
}

// Joins the parts of every item.  Of an item's CTAs the first `out_shares` add up
// 32 outputs each, the others normalise kJoinRows rows' scores and add the
// weights (listed blocks have none: outputs only).  Latency-bound: everything that does not need the joined (m, l) is
// loaded before they are known.
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 512;

__global__ void __launch_bounds__(kJoinThreads)
    attend_join_kernel(const __grid_constant__ AttendParams p, int32_t head_dim, int32_t unit,
                       int32_t out_shares, int32_t shares) {
  __shared__ float s_norm[GP * 2];
  __shared__ float s_acc[kJoinThreads / 32][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int item = (int)(blockIdx.x / (unsigned)shares);
  const int share = (int)(blockIdx.x % (unsigned)shares) - out_shares;
  const int b = item / p.n_kv, g = item - b * p.n_kv;
  const int G = p.n_heads / p.n_kv;
  pdl_wait();
  pdl_launch_dependents();
  const bool weights = p.weight_ptrs != nullptr;
  int32_t n = clamped_rows(p.n_pos, b, p.max_n_pos, p.status);
  float* wts = weights ? p.weight_ptrs[b] : nullptr;
  if (weights && !usable_weights(wts, p.status)) n = 0;
  if (!usable_ptrs(p.k_ptrs[b], p.v_ptrs[b], p.status)) n = 0;
  const int64_t row0 = (int64_t)share * kJoinRows;
  if (share < 0 && n == 0) {  // no rows: zeros
    if (tid < 32)
      p.xb[((int64_t)b * p.n_heads + (int64_t)g * G) * head_dim + (share + out_shares) * 32 + tid] = 0.f;
    return;
  }
  if (row0 >= n) return;
  // parts with rows (of a list: all, some perhaps without)
  const int64_t part_rows = (int64_t)p.part_units * unit;
  const int32_t S = weights ? (int32_t)((n + part_rows - 1) / part_rows) : p.S;
  const float2* ml = p.part_ml + (int64_t)item * G * p.S;

  constexpr int kPer = kJoinRows / kJoinThreads;
  float s[kPer][GP], old[kPer];
  float* wrow = wts + (int64_t)g * p.weight_stride + row0;
  const float* scores = p.scores + (int64_t)item * G * p.score_pitch + row0;
  if (share >= 0) {
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int i = r * kJoinThreads + tid;
      if (row0 + i < n) {
        old[r] = wrow[i];
#pragma unroll
        for (int h = 0; h < GP; ++h)
          if (h < G) s[r][h] = __ldcg(scores + h * p.score_pitch + i);
      }
    }
  }
  // one head a warp (an output share needs only its own): its largest m and its sum
  const int out0 = (share + out_shares) * 32, out_head = out0 / head_dim;
  if (warp < G && (share >= 0 || warp == out_head)) {
    float top = -INFINITY;
#pragma unroll 8
    for (int x = lane; x < S; x += 32) top = fmaxf(top, ml[warp * p.S + x].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll 8
    for (int x = lane; x < S; x += 32) {
      const float2 y = ml[warp * p.S + x];
      sum = fmaf(y.y, exp2_approx(y.x - ref), sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      s_norm[warp * 2] = ref;
      s_norm[warp * 2 + 1] = sum == 0.f ? 0.f : 1.0f / sum;  // no row listed: zeros
    }
  }
  __syncthreads();
  if (share >= 0) {
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int i = r * kJoinThreads + tid;
      if (row0 + i < n) {
        float x = 0.f;
#pragma unroll
        for (int h = 0; h < GP; ++h)
          if (h < G) x = fmaf(exp2_approx(s[r][h] - s_norm[h * 2]), s_norm[h * 2 + 1], x);
        wrow[i] = old[r] + x;
      }
    }
    return;
  }
  // outputs: a warp for every eighth part
  const float ref = s_norm[out_head * 2];
  const float* part = p.part + (int64_t)item * p.S * G * head_dim + out0 + lane;
  float acc = 0.f;
#pragma unroll 8
  for (int x = warp; x < S; x += kJoinThreads / 32)
    acc = fmaf(__ldcg(part + (int64_t)x * G * head_dim),
               exp2_approx(ml[out_head * p.S + x].x - ref), acc);
  s_acc[warp][lane] = acc;
  __syncthreads();
  if (warp == 0) {
    acc = 0.f;
#pragma unroll
    for (int x = 0; x < kJoinThreads / 32; ++x) acc += s_acc[x][lane];
    p.xb[((int64_t)b * p.n_heads + (int64_t)g * G) * head_dim + out0 + lane] =
        acc * s_norm[out_head * 2 + 1];
  }
}

// Rows of a part when a second kernel joins the parts, 0 when a cluster does.
// A single sequence is cut into one wave of CTAs (three an SM).  A batch may be
// ragged, and its CTAs are counted for the longest sequence: two waves, so that
// half of them idle still leaves one (131,072 rows of one sequence: 64 us with one
// wave, 68 with two; 16 sequences of 77 to 8191 rows: 41 and 30).  A part takes at
// least 8 units a warp; sequences too short for two such parts are left to a
// cluster (one launch less, about 3 us).
int32_t part_rows_for(int32_t batch, int32_t n_kv, int64_t max_rows, int unit,
                      const DeviceInfo& dev) {
  const int64_t step = 4 * unit, least = 8 * step, items = (int64_t)batch * n_kv;
  const int64_t ctas = (batch == 1 ? 3 : 6) * (int64_t)dev.sms;
  int64_t rows = (max_rows * items + ctas - 1) / ctas;
  rows = std::max(least, (rows + step - 1) / step * step);
  return max_rows > rows ? (int32_t)rows : 0;
}

// The same for listed blocks: a cluster does it, unless so few lists are so long
// that a cluster's warps (of 16 wide CTAs up to 7 lists, else of 16 slim ones) have
// more than 4 units each while most of the device is idle.  One FP16 sequence of 8 kv
// heads: 4096 rows 12.1 us by clusters and 11.8 by parts, 8192 16.4 and 14.4, 12,800
// 21.2 and 16.3; of 4 kv heads: 4160 rows 9.2 and 12.0, 8192 11.3 and 11.8.  FP32, 8 kv
// heads: 6400 rows 25.4 and 17.4.
int64_t list_part_rows_for(int64_t items, int64_t rows, int unit, const DeviceInfo& dev) {
  const int64_t step = 4 * unit, full = 3 * (int64_t)dev.sms;
  if (items * 32 > full || rows <= 4 * (items < 8 ? 128 : 64) * (int64_t)unit) return 0;
  return std::max(2 * step, (rows * items / full + step - 1) / step * step);
}

// Floats between the heads' scores: a last unit stores its rows past the end too.
int64_t score_pitch_for(int64_t max_rows) { return (max_rows + 15) / 16 * 16; }

template <class T, int HD, bool BLOCKS, bool WIDE>
struct Launch {
  using C = Cta<T, HD, WIDE>;
  static_assert(C::kRing >= (C::kWarps * (HD + 2) + HD) * GP * 4, "the outputs reuse the rings");

  static ClusterKernel& state() {
    static ClusterKernel ck;
    return ck;
  }
  // CTAs of an item's cluster: as many as the device holds at once, while every
  // warp still has a unit.
  static int cluster_size(int64_t items, int64_t units, const DeviceInfo& dev) {
    int S = 1;
    while (S < 16 && units > (int64_t)C::kWarps * S &&
           items * S * 2 <= (int64_t)C::kMinCtas * dev.sms &&
           items <= clusters_held(attend_kernel<T, HD, BLOCKS, WIDE>, state(), C::kThreads,
                                  (size_t)C::kRing, 2 * S, dev))
      S *= 2;
    return S;
  }
  // p.part: S parts of an item, else a cluster of S.
  static int run(AttendParams& p, int64_t items, int S, cudaStream_t stream, std::string* err) {
    if (items * S > INT32_MAX) {
      *err = "batch * n_kv_heads too large";
      return GLA_ERR_NOT_SUPPORTED;
    }
    p.S = S;
    return launch_clusters(attend_kernel<T, HD, BLOCKS, WIDE>, (unsigned)(items * S), C::kThreads,
                           (size_t)C::kRing, p.part ? 1 : S, state(), stream, "attention", err, p);
  }
};

template <class T, int HD, bool BLOCKS>
int launch_one(const AttendRequest& r, const DeviceInfo& dev, cudaStream_t stream,
               std::string* err) {
  constexpr int U = unit_rows<T, HD>();
  AttendParams p{};
  p.q = r.q;
  p.k_ptrs = r.k_ptrs;
  p.v_ptrs = r.v_ptrs;
  p.n_pos = r.n_pos;
  p.max_n_pos = r.max_n_pos;
  p.xb = r.xb;
  p.n_heads = r.n_heads;
  p.n_kv = r.n_kv;
  p.kv_bytes = (uint32_t)(r.kv_stride * (int64_t)sizeof(T));
  p.scale_log2 = r.scale * kLog2e;
  p.block_ids = r.block_ids;
  p.n_sel = r.n_sel;
  while (BLOCKS && (1 << p.br_shift) < r.block_rows) ++p.br_shift;
  p.weight_ptrs = r.weight_ptrs;
  p.weight_stride = r.weight_stride;
  p.scores = r.scores;
  p.status = r.status;
  const int64_t rows = BLOCKS ? (int64_t)r.n_sel * r.block_rows : (int64_t)r.max_n_pos;
  const int64_t units = (rows + U - 1) / U;
  const int64_t items = (int64_t)r.batch * r.n_kv;
  if (!BLOCKS) p.score_pitch = score_pitch_for(r.max_n_pos);
  {
    const int64_t part_rows = BLOCKS ? list_part_rows_for(items, rows, U, dev)
                                     : part_rows_for(r.batch, r.n_kv, rows, U, dev);
    if (part_rows) {
      p.part_units = (int32_t)(part_rows / U);
      const int64_t parts = (rows + part_rows - 1) / part_rows;
      const int32_t outs = (r.n_heads / r.n_kv) * HD / 32;
      const int64_t shares = (BLOCKS ? 0 : (rows + kJoinRows - 1) / kJoinRows) + outs;
      if (items * parts > INT32_MAX || items * shares > INT32_MAX) {
        *err = "batch * n_kv_heads * max_n_pos too large";
        return GLA_ERR_NOT_SUPPORTED;
      }
      const int64_t heads = (int64_t)r.batch * r.n_heads;
      p.part = r.scores + heads * p.score_pitch;
      p.part_ml = reinterpret_cast<float2*>(p.part + heads * parts * r.head_dim);
      int rc = Launch<T, HD, BLOCKS, false>::run(p, items, (int)parts, stream, err);
      if (rc != GLA_OK) return rc;
      static ClusterKernel ck;
      return launch_clusters(attend_join_kernel, (unsigned)(items * shares), kJoinThreads, 0, 1,
                             ck, stream, "attention join", err, p, (int32_t)HD, U, outs,
                             (int32_t)shares);
    }
  }
  // Wide CTAs if they make more warps of an item, or as many without a cluster;
  // else slim ones, which spread over more SMs (an SM takes in 64 bytes a clock).
  const int sw = Launch<T, HD, BLOCKS, true>::cluster_size(items, units, dev);
  const int ss = Launch<T, HD, BLOCKS, false>::cluster_size(items, units, dev);
  const bool wide = items * sw <= dev.sms && (sw == 1 ? 2 >= ss : 2 * sw > ss);
  return wide ? Launch<T, HD, BLOCKS, true>::run(p, items, sw, stream, err)
              : Launch<T, HD, BLOCKS, false>::run(p, items, ss, stream, err);
}

template <int HD>
int by_type(const AttendRequest& r, const DeviceInfo& dev, cudaStream_t stream, std::string* err) {
  if (r.dtype == GLA_DTYPE_F16)
    return r.block_ids ? launch_one<__half, HD, true>(r, dev, stream, err)
                       : launch_one<__half, HD, false>(r, dev, stream, err);
  return r.block_ids ? launch_one<float, HD, true>(r, dev, stream, err)
                     : launch_one<float, HD, false>(r, dev, stream, err);
}

}  // namespace

size_t attend_workspace_floats(const AttendRequest& r, const DeviceInfo& dev) {
  const int unit = r.dtype == GLA_DTYPE_F16 ? unit_rows<__half, 64>() : unit_rows<float, 64>();
  const int64_t rows = r.block_ids ? (int64_t)r.n_sel * r.block_rows : (int64_t)r.max_n_pos;
  const int64_t part = r.block_ids
                           ? list_part_rows_for((int64_t)r.batch * r.n_kv, rows, unit, dev)
                           : part_rows_for(r.batch, r.n_kv, rows, unit, dev);
  const int64_t parts = part ? (rows + part - 1) / part : 0;
  const int64_t pitch = r.block_ids ? 0 : score_pitch_for(rows);
  const size_t heads = (size_t)r.batch * r.n_heads, each = (size_t)(pitch + parts * (r.head_dim + 2));
  constexpr size_t kMost = SIZE_MAX / 8;  // no device holds it: the allocation fails
  return each && heads > kMost / each ? kMost : heads * each;
}

int launch_attend(const AttendRequest& r, const DeviceInfo& dev, cudaStream_t stream,
                  std::string* err) {
  switch (r.head_dim) {
    case 64: return by_type<64>(r, dev, stream, err);
    case 96: return by_type<96>(r, dev, stream, err);
    default: return by_type<128>(r, dev, stream, err);
  }
}

}  // namespace gla
