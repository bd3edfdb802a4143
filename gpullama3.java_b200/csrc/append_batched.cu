// append_batched.cu - the new token of every sequence of a batch: RoPE of q
// and k, the key and value rows written to the sequences' caches (FP32 or
// FP16), and the bounds of the block that holds the new row brought up to
// date.  The cache row is apart from the position: after an eviction
// (evict.cu) a sequence holds fewer rows than it has seen tokens.
//
// Rotation: the same helpers, frequencies and roundings as rope.cu, so the
// FP32 rows equal gla_rope_append_f32's bit for bit.
//
// Latency-bound: a token is a few tens of KB.  What costs is the chain of
// double pow, cos and sin; the (cos, sin) pairs of a position are computed
// once per CTA, one pair a thread, and shared by its heads, and the CTAs of
// one sequence take kHeadsPerCta heads each.  Measured on one B200: 3.3 to 3.8 us
// for one sequence of the 1B shape, 5.2 us for 96 of the 8B shape, with bounds.
#include "cache_ops.cuh"
#include "gla_rope.cuh"

namespace gla {

namespace {

constexpr int kHeadsPerCta = 8;

__device__ __forceinline__ float to_cache(float x, float*) { return x; }
__device__ __forceinline__ __half to_cache(float x, __half*) { return __float2half_rn(x); }

__device__ __forceinline__ void widen(float* lo, float* hi, float x, bool first) {
  *lo = first ? x : fminf(*lo, x);
  *hi = first ? x : fmaxf(*hi, x);
}
__device__ __forceinline__ void widen(__half* lo, __half* hi, __half x, bool first) {
  *lo = first ? x : __hmin(*lo, x);
  *hi = first ? x : __hmax(*hi, x);
}

// Heads of a sequence: [0, n_kv) the kv heads, [n_kv, n_kv + n_heads) the q heads.
template <class T>
__global__ void __launch_bounds__(256)
    append_batched_kernel(const float* q, const float* __restrict__ k,
                          const float* __restrict__ v, float* q_out, T* const* __restrict__ k_ptrs,
                          T* const* __restrict__ v_ptrs, const int32_t* __restrict__ positions,
                          const int32_t* __restrict__ rows, T* const* __restrict__ bounds_ptrs,
                          int32_t br_shift, int32_t n_heads, int32_t n_kv, int32_t head_dim,
                          int64_t kv_stride, int32_t context_length, double theta, int32_t style,
                          int32_t* __restrict__ status) {
  __shared__ float2 s_turn[64];
  pdl_wait();
  const int b = blockIdx.y;
  const int32_t pos = positions[b];
  const int32_t row = rows ? rows[b] : pos;
  const int half = head_dim >> 1;
  if (pos < 0 || row < 0 || row >= context_length) {
    if (threadIdx.x == 0) atomicCAS(status, 0, GLA_ERR_INVALID_ARG);
    return;
  }
  T* kc = k_ptrs[b];
  T* vc = v_ptrs[b];
  T* bounds = bounds_ptrs ? bounds_ptrs[b] : nullptr;
  if (!usable_ptrs(kc, vc, status)) return;
  if (bounds_ptrs && !usable_ptrs(bounds, bounds, status)) return;
  if (threadIdx.x < half) {
    float fcr, fci;
    rope_cos_sin(pos, threadIdx.x, head_dim, theta, &fcr, &fci);
    s_turn[threadIdx.x] = make_float2(fcr, fci);
  }
  __syncthreads();
  const int head0 = blockIdx.x * kHeadsPerCta;
  const int heads = min(kHeadsPerCta, n_kv + n_heads - head0);
  for (int i = threadIdx.x; i < heads * half; i += blockDim.x) {
    const int hh = i / half, ic = i - hh * half;
    const int head = head0 + hh;
    const float2 t = s_turn[ic];
    int i0, i1;
    rope_pair(style, ic, head_dim, &i0, &i1);
    if (head >= n_kv) {
      const int64_t at = ((int64_t)b * n_heads + (head - n_kv)) * head_dim;
      float o0, o1;
      rope_rotate(q[at + i0], q[at + i1], t.x, t.y, &o0, &o1);
      q_out[at + i0] = o0;
      q_out[at + i1] = o1;
      continue;
    }
    const int64_t at = ((int64_t)b * n_kv + head) * head_dim;
    float o0, o1;
    rope_rotate(k[at + i0], k[at + i1], t.x, t.y, &o0, &o1);
    const T k0 = to_cache(o0, (T*)nullptr), k1 = to_cache(o1, (T*)nullptr);
    const int64_t dst = (int64_t)row * kv_stride + (int64_t)head * head_dim;
    kc[dst + i0] = k0;
    kc[dst + i1] = k1;
    vc[dst + i0] = to_cache(v[at + i0], (T*)nullptr);
    vc[dst + i1] = to_cache(v[at + i1], (T*)nullptr);
    if (bounds) {
      const bool first = (row & ((1 << br_shift) - 1)) == 0;
      T* lo = bounds + ((int64_t)(row >> br_shift) * n_kv + head) * 2 * head_dim;
      widen(lo + i0, lo + head_dim + i0, k0, first);
      widen(lo + i1, lo + head_dim + i1, k1, first);
    }
  }
}

template <class T>
int launch_append(const AppendRequest& r, cudaStream_t stream, std::string* err) {
  int32_t br_shift = 0;
  while (r.bounds_ptrs && (1 << br_shift) < r.block_rows) ++br_shift;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const unsigned gx = (unsigned)((r.n_kv + r.n_heads + kHeadsPerCta - 1) / kHeadsPerCta);
  for (int32_t b0 = 0; b0 < r.batch; b0 += 65535) {  // gridDim.y
    cfg.gridDim = dim3(gx, (unsigned)std::min(r.batch - b0, 65535));
    const int64_t qo = (int64_t)b0 * r.n_heads * r.head_dim, ko = (int64_t)b0 * r.n_kv * r.head_dim;
    cudaError_t e = cudaLaunchKernelEx(
        &cfg, append_batched_kernel<T>, r.q + qo, r.k + ko, r.v + ko, r.q_out + qo,
        reinterpret_cast<T* const*>(r.k_ptrs) + b0, reinterpret_cast<T* const*>(r.v_ptrs) + b0,
        r.positions + b0, r.rows ? r.rows + b0 : nullptr,
        r.bounds_ptrs ? reinterpret_cast<T* const*>(r.bounds_ptrs) + b0 : nullptr, br_shift,
        r.n_heads, r.n_kv, r.head_dim, r.kv_stride, r.context_length, r.theta, r.rope_style,
        r.status);
    if (e != cudaSuccess) {
      cudaGetLastError();
      *err = std::string("batched append launch failed: ") + cudaGetErrorString(e);
      return GLA_ERR_CUDA;
    }
  }
  return GLA_OK;
}

}  // namespace

int launch_append_batched(const AppendRequest& r, cudaStream_t stream, std::string* err) {
  return r.dtype == GLA_DTYPE_F16 ? launch_append<__half>(r, stream, err)
                                  : launch_append<float>(r, stream, err);
}

}  // namespace gla
