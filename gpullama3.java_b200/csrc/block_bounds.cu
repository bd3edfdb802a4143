// block_bounds.cu - per-block bounds of the cached keys.
//
// bounds[j][g][0][d] = min, bounds[j][g][1][d] = max of k[t][g][d] over the
// rows t < n of block j (block_rows rows).  With them
//   q . k_t <= sum_d max(q_d lo_d, q_d hi_d)   for every row t of the block,
// the score gla_block_select_* ranks blocks by.  Minimum and maximum round
// nothing: bounds are exact in the cache's own type and do not depend on the
// order of the rows.
//
// HBM-bound: every key is read once.  16 lanes of a warp read one row's 16-byte
// chunks side by side, the other 16 the next row, eight loads under way each, and
// the two join by shuffles; a block of rows is the unit of work, so a short sequence
// still spreads over many warps.  16 sequences of up to 32,768 FP16 rows of 2 KB:
// 107 us, 6.3 TB/s (row pieces of 128 bytes 122 us, of 512 bytes 111); 4096 FP32
// rows of 2 KB 3.4 us (3.2 and 3.9).
#include "cache_ops.cuh"

namespace gla {

namespace {

// 16 bytes of cache elements: 8 halves or 4 floats.
template <class T>
struct Vec16;
template <>
struct Vec16<float> {
  __device__ __forceinline__ static void low(float4& a, const float4& b) {
    a.x = fminf(a.x, b.x), a.y = fminf(a.y, b.y), a.z = fminf(a.z, b.z), a.w = fminf(a.w, b.w);
  }
  __device__ __forceinline__ static void high(float4& a, const float4& b) {
    a.x = fmaxf(a.x, b.x), a.y = fmaxf(a.y, b.y), a.z = fmaxf(a.z, b.z), a.w = fmaxf(a.w, b.w);
  }
};
template <>
struct Vec16<__half> {
  __device__ __forceinline__ static uint32_t lo2(uint32_t a, uint32_t b) {
    const __half2 r = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ __forceinline__ static uint32_t hi2(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ __forceinline__ static void low(float4& a, const float4& b) {
    uint32_t* x = reinterpret_cast<uint32_t*>(&a);
    const uint32_t* y = reinterpret_cast<const uint32_t*>(&b);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lo2(x[i], y[i]);
  }
  __device__ __forceinline__ static void high(float4& a, const float4& b) {
    uint32_t* x = reinterpret_cast<uint32_t*>(&a);
    const uint32_t* y = reinterpret_cast<const uint32_t*>(&b);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = hi2(x[i], y[i]);
  }
};

__device__ __forceinline__ float4 shfl_xor4(float4 v, int m) {
  v.x = __shfl_xor_sync(0xffffffffu, v.x, m);
  v.y = __shfl_xor_sync(0xffffffffu, v.y, m);
  v.z = __shfl_xor_sync(0xffffffffu, v.z, m);
  v.w = __shfl_xor_sync(0xffffffffu, v.w, m);
  return v;
}

constexpr int kLanes = 16;  // chunks of a column group

// Work item: (sequence, block, column group); a group is kLanes chunks of 16
// bytes.  start_pos (or null): rows before it are unchanged, so the blocks
// wholly before it are left alone.
template <class T>
__global__ void __launch_bounds__(256)
    block_bounds_kernel(const T* const* __restrict__ k_ptrs, const int32_t* __restrict__ start_pos,
                        const int32_t* __restrict__ n_pos, int32_t max_n_pos,
                        T* const* __restrict__ bounds_ptrs, int32_t max_blocks, int32_t groups,
                        int32_t chunks_per_head, int32_t n_kv, int64_t kv_stride, int32_t br_shift,
                        int32_t* __restrict__ status) {
  pdl_wait();
  constexpr int kPer = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const int32_t n = clamped_rows(n_pos, b, max_n_pos, status);
  const T* k = k_ptrs[b];
  T* out = bounds_ptrs[b];
  if (!usable_ptrs(k, out, status)) return;
  const int32_t br = 1 << br_shift;
  const int32_t nb = (int32_t)(((int64_t)n + br - 1) >> br_shift);
  int32_t j0 = 0;
  if (start_pos) j0 = max(start_pos[b], 0) >> br_shift;
  const int64_t items = (int64_t)max_blocks * groups;
  const int64_t stride = (int64_t)gridDim.x * 8;
  for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += stride) {
    const int32_t jj = (int32_t)(it / groups);
    const int32_t j = j0 + jj;
    if (j >= nb) return;  // items ascend with the block
    const int32_t chunk = (int32_t)(it - (int64_t)jj * groups) * kLanes + lane % kLanes;
    const bool live = chunk < chunks_per_head * n_kv;
    const int64_t col = (int64_t)(live ? chunk : 0) * kPer;
    const int32_t row0 = j << br_shift, rows = min(br, n - row0);
    const T* src = k + (int64_t)row0 * kv_stride + col;
    constexpr int kStep = 32 / kLanes;  // rows side by side
    const int r0 = lane / kLanes;
    // rows past the last one repeat it: a repeated row changes no minimum
    float4 lo = __ldcg(reinterpret_cast<const float4*>(src + (int64_t)min(r0, rows - 1) * kv_stride));
    float4 hi = lo;
#pragma unroll 8
    for (int r = r0 + kStep; r < br; r += kStep) {
      const float4 x =
          __ldcg(reinterpret_cast<const float4*>(src + (int64_t)min(r, rows - 1) * kv_stride));
      Vec16<T>::low(lo, x);
      Vec16<T>::high(hi, x);
    }
#pragma unroll
    for (int m = kLanes; m <= 16; m <<= 1) {
      Vec16<T>::low(lo, shfl_xor4(lo, m));
      Vec16<T>::high(hi, shfl_xor4(hi, m));
    }
    if (live && r0 == 0) {
      const int32_t g = chunk / chunks_per_head, c = chunk - g * chunks_per_head;
      const int64_t width = (int64_t)chunks_per_head * kPer;
      const int64_t at = ((int64_t)j * n_kv + g) * 2 * width + (int64_t)c * kPer;
      *reinterpret_cast<float4*>(out + at) = lo;
      *reinterpret_cast<float4*>(out + at + width) = hi;
    }
  }
}

template <class T>
int launch_bounds(const BoundsRequest& r, cudaStream_t stream, std::string* err) {
  const int32_t chunks_per_head = r.head_dim * (int)sizeof(T) / 16;
  const int32_t groups = (chunks_per_head * r.n_kv + kLanes - 1) / kLanes;
  int32_t br_shift = 0;
  while ((1 << br_shift) < r.block_rows) ++br_shift;
  const int32_t max_blocks = (int32_t)(((int64_t)r.max_n_pos + r.block_rows - 1) / r.block_rows);
  const int64_t ctas = std::min<int64_t>(((int64_t)max_blocks * groups + 7) / 8, 1 << 20);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int32_t b0 = 0; b0 < r.batch; b0 += 65535) {  // gridDim.y
    cfg.gridDim = dim3((unsigned)ctas, (unsigned)std::min(r.batch - b0, 65535));
    cudaError_t e = cudaLaunchKernelEx(
        &cfg, block_bounds_kernel<T>, reinterpret_cast<const T* const*>(r.k_ptrs) + b0,
        r.start_pos ? r.start_pos + b0 : nullptr, r.n_pos + b0, r.max_n_pos,
        reinterpret_cast<T* const*>(r.bounds_ptrs) + b0, max_blocks, groups, chunks_per_head,
        r.n_kv, r.kv_stride, br_shift, r.status);
    if (e != cudaSuccess) {
      cudaGetLastError();
      *err = std::string("block bounds launch failed: ") + cudaGetErrorString(e);
      return GLA_ERR_CUDA;
    }
  }
  return GLA_OK;
}

}  // namespace

int launch_block_bounds(const BoundsRequest& r, cudaStream_t stream, std::string* err) {
  return r.dtype == GLA_DTYPE_F16 ? launch_bounds<__half>(r, stream, err)
                                  : launch_bounds<float>(r, stream, err);
}

}  // namespace gla
