// api_cache.cu - the C ABI of the long-cache operators (include/gpullama_attn.h,
// "Long caches"): argument checks, the score workspace and dispatch.  Every
// entry point returns a status code; no exception crosses the ABI.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <string>

#include "gla_ctx.h"

using namespace gla;

namespace {

// Runs an entry point's body; an exception (only allocation can throw)
// becomes a status.
template <class F>
int32_t guarded(gla_ctx* ctx, F body) noexcept {
  if (!ctx) return GLA_ERR_INVALID_ARG;
  try {
    DeviceGuard dg(ctx->device);
    if (!dg.ok) return fail(ctx, GLA_ERR_CUDA, "cudaSetDevice failed");
    return body();
  } catch (...) {
    return GLA_ERR_OUT_OF_MEMORY;
  }
}

int check_heads(gla_ctx* ctx, int32_t batch, int32_t n_heads, int32_t n_kv, int32_t head_dim) {
  if (batch < 1) return fail(ctx, GLA_ERR_INVALID_ARG, "batch must be >= 1");
  if (n_heads < 1 || n_kv < 1)
    return fail(ctx, GLA_ERR_INVALID_ARG, "n_heads and n_kv_heads must be positive");
  if (n_heads % n_kv != 0)
    return fail(ctx, GLA_ERR_INVALID_ARG, "n_heads must be a multiple of n_kv_heads");
  if (n_heads / n_kv > 8) return fail(ctx, GLA_ERR_NOT_SUPPORTED, "kvMul must be at most 8");
  if (head_dim != 64 && head_dim != 96 && head_dim != 128)
    return fail(ctx, GLA_ERR_NOT_SUPPORTED, "head_dim must be 64, 96 or 128");
  return GLA_OK;
}

int check_stride(gla_ctx* ctx, int dtype, int32_t n_kv, int32_t head_dim, int64_t kv_stride) {
  if (kv_stride < (int64_t)n_kv * head_dim)
    return fail(ctx, GLA_ERR_INVALID_ARG, "kv_stride must be >= n_kv_heads * head_dim");
  if (kv_stride % (dtype == GLA_DTYPE_F16 ? 8 : 4) != 0)
    return fail(ctx, GLA_ERR_ALIGNMENT, "kv_stride must be a multiple of 16 bytes");
  if (kv_stride > (1 << 28)) return fail(ctx, GLA_ERR_NOT_SUPPORTED, "kv_stride above 2^28");
  return GLA_OK;
}

int check_block_rows(gla_ctx* ctx, int32_t block_rows) {
  if (block_rows != 16 && block_rows != 32 && block_rows != 64 && block_rows != 128)
    return fail(ctx, GLA_ERR_NOT_SUPPORTED, "block_rows must be 16, 32, 64 or 128");
  return GLA_OK;
}

int finish(gla_ctx* ctx, int rc, const std::string& err) {
  return rc == GLA_OK ? GLA_OK : fail(ctx, rc, err);
}

int32_t block_bounds(gla_ctx* ctx, int dtype, const void* const* k_ptrs, const int32_t* start_pos,
                     const int32_t* n_pos, int32_t max_n_pos, void* const* bounds_ptrs,
                     int32_t batch, int32_t n_kv_heads, int32_t head_dim, int64_t kv_stride,
                     int32_t block_rows) {
  return guarded(ctx, [&]() -> int {
    if (!k_ptrs || !n_pos || !bounds_ptrs) return fail(ctx, GLA_ERR_INVALID_ARG, "null pointer");
    if (max_n_pos < 1) return fail(ctx, GLA_ERR_INVALID_ARG, "max_n_pos must be >= 1");
    int rc = check_heads(ctx, batch, n_kv_heads, n_kv_heads, head_dim);
    if (rc == GLA_OK) rc = check_stride(ctx, dtype, n_kv_heads, head_dim, kv_stride);
    if (rc == GLA_OK) rc = check_block_rows(ctx, block_rows);
    if (rc != GLA_OK) return rc;
    BoundsRequest r{};
    r.dtype = dtype;
    r.k_ptrs = k_ptrs;
    r.start_pos = start_pos;
    r.n_pos = n_pos;
    r.max_n_pos = max_n_pos;
    r.bounds_ptrs = bounds_ptrs;
    r.batch = batch;
    r.n_kv = n_kv_heads;
    r.head_dim = head_dim;
    r.kv_stride = kv_stride;
    r.block_rows = block_rows;
    r.status = ctx->status;
    std::string err;
    return finish(ctx, launch_block_bounds(r, ctx->stream, &err), err);
  });
}

int32_t append_batched(gla_ctx* ctx, int dtype, const float* q, const float* k, const float* v,
                       float* q_out, void* const* k_ptrs, void* const* v_ptrs,
                       const int32_t* positions, const int32_t* rows, void* const* bounds_ptrs,
                       int32_t block_rows, int32_t batch, int32_t n_heads, int32_t n_kv_heads,
                       int32_t head_dim, int64_t kv_stride, int32_t context_length, float theta,
                       int32_t rope_style) {
  return guarded(ctx, [&]() -> int {
    if (!q || !k || !v || !q_out || !k_ptrs || !v_ptrs || !positions)
      return fail(ctx, GLA_ERR_INVALID_ARG, "null pointer");
    int rc = check_heads(ctx, batch, n_heads, n_kv_heads, head_dim);
    if (rc == GLA_OK) rc = check_stride(ctx, dtype, n_kv_heads, head_dim, kv_stride);
    if (rc == GLA_OK && bounds_ptrs) rc = check_block_rows(ctx, block_rows);
    if (rc != GLA_OK) return rc;
    if (context_length < 1) return fail(ctx, GLA_ERR_INVALID_ARG, "context_length must be >= 1");
    if (rope_style != GLA_ROPE_INTERLEAVED && rope_style != GLA_ROPE_NEOX)
      return fail(ctx, GLA_ERR_INVALID_ARG, "unknown rope_style");
    if (!(theta > 0.f) || !std::isfinite(theta))
      return fail(ctx, GLA_ERR_INVALID_ARG, "theta must be positive");
    AppendRequest r{};
    r.dtype = dtype;
    r.q = q;
    r.k = k;
    r.v = v;
    r.q_out = q_out;
    r.k_ptrs = k_ptrs;
    r.v_ptrs = v_ptrs;
    r.positions = positions;
    r.rows = rows;
    r.bounds_ptrs = bounds_ptrs;
    r.block_rows = block_rows;
    r.batch = batch;
    r.n_heads = n_heads;
    r.n_kv = n_kv_heads;
    r.head_dim = head_dim;
    r.kv_stride = kv_stride;
    r.context_length = context_length;
    r.theta = (double)theta;
    r.rope_style = rope_style;
    r.status = ctx->status;
    std::string err;
    return finish(ctx, launch_append_batched(r, ctx->stream, &err), err);
  });
}

int32_t block_select(gla_ctx* ctx, int dtype, const float* q, const void* const* bounds_ptrs,
                     const int32_t* n_pos, int32_t max_n_pos, int32_t* block_ids, int32_t batch,
                     int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t block_rows,
                     int32_t n_sel, int32_t n_first, int32_t n_last) {
  return guarded(ctx, [&]() -> int {
    if (!q || !bounds_ptrs || !n_pos || !block_ids)
      return fail(ctx, GLA_ERR_INVALID_ARG, "null pointer");
    if (max_n_pos < 1) return fail(ctx, GLA_ERR_INVALID_ARG, "max_n_pos must be >= 1");
    int rc = check_heads(ctx, batch, n_heads, n_kv_heads, head_dim);
    if (rc == GLA_OK) rc = check_block_rows(ctx, block_rows);
    if (rc != GLA_OK) return rc;
    if (n_sel < 1 || n_first < 0 || n_last < 0 || (int64_t)n_first + n_last > n_sel)
      return fail(ctx, GLA_ERR_INVALID_ARG,
                  "n_sel must be >= 1 and hold the n_first + n_last blocks that are always chosen");
    SelectRequest r{};
    r.dtype = dtype;
    r.q = q;
    r.bounds_ptrs = bounds_ptrs;
    r.n_pos = n_pos;
    r.max_n_pos = max_n_pos;
    r.block_ids = block_ids;
    r.batch = batch;
    r.n_heads = n_heads;
    r.n_kv = n_kv_heads;
    r.head_dim = head_dim;
    r.block_rows = block_rows;
    r.n_sel = n_sel;
    r.n_first = n_first;
    r.n_last = n_last;
    r.status = ctx->status;
    std::string err;
    return finish(ctx, launch_block_select(r, ctx->dev, ctx->stream, &err), err);
  });
}

int check_attend(gla_ctx* ctx, int dtype, const float* q, const void* const* k_ptrs,
                 const void* const* v_ptrs, const int32_t* n_pos, float* xb, int32_t max_n_pos,
                 int32_t batch, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                 int64_t kv_stride, float scale) {
  if (!q || !k_ptrs || !v_ptrs || !n_pos || !xb)
    return fail(ctx, GLA_ERR_INVALID_ARG, "null pointer");
  if (max_n_pos < 1) return fail(ctx, GLA_ERR_INVALID_ARG, "max_n_pos must be >= 1");
  if (!std::isfinite(scale)) return fail(ctx, GLA_ERR_INVALID_ARG, "scale must be finite");
  int rc = check_heads(ctx, batch, n_heads, n_kv_heads, head_dim);
  if (rc == GLA_OK) rc = check_stride(ctx, dtype, n_kv_heads, head_dim, kv_stride);
  if (rc != GLA_OK) return rc;
  if (!aligned16(q) || !aligned16(xb))
    return fail(ctx, GLA_ERR_ALIGNMENT, "q and xb must be 16-byte aligned");
  return GLA_OK;
}

AttendRequest attend_request(gla_ctx* ctx, int dtype, const float* q, const void* const* k_ptrs,
                             const void* const* v_ptrs, const int32_t* n_pos, int32_t max_n_pos,
                             float* xb, int32_t batch, int32_t n_heads, int32_t n_kv_heads,
                             int32_t head_dim, int64_t kv_stride, float scale) {
  AttendRequest r{};
  r.dtype = dtype;
  r.q = q;
  r.k_ptrs = k_ptrs;
  r.v_ptrs = v_ptrs;
  r.n_pos = n_pos;
  r.max_n_pos = max_n_pos;
  r.xb = xb;
  r.batch = batch;
  r.n_heads = n_heads;
  r.n_kv = n_kv_heads;
  r.head_dim = head_dim;
  r.kv_stride = kv_stride;
  r.scale = scale;
  r.status = ctx->status;
  return r;
}

// Grows the attention workspace (scores, parts).  An outgrown buffer lives until gla_destroy:
// kernels in flight and captured graphs may still use it.
int ensure_scores(gla_ctx* ctx, size_t floats) {
  if (floats <= ctx->scores_cap) return GLA_OK;
  if (stream_capturing(ctx->stream))
    return fail(ctx, GLA_ERR_INVALID_ARG,
                "attention workspace must grow; run the largest call once before capture");
  ctx->retired.reserve(ctx->retired.size() + 1);
  // doubling bounds what outgrown buffers hold to the size of the current one; where
  // there is no room for that, what the call needs will do
  size_t cap = std::max(floats, 2 * ctx->scores_cap);
  void* p = nullptr;
  cudaError_t e = cudaMalloc(&p, cap * sizeof(float));
  if (e != cudaSuccess && cap > floats) {
    cudaGetLastError();
    cap = floats;
    e = cudaMalloc(&p, cap * sizeof(float));
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(ctx, GLA_ERR_OUT_OF_MEMORY, "attention workspace allocation failed");
  }
  if (ctx->scores) ctx->retired.push_back(ctx->scores);
  ctx->scores = static_cast<float*>(p);
  ctx->scores_cap = cap;
  return GLA_OK;
}

int32_t decode_blocks(gla_ctx* ctx, int dtype, const float* q, const void* const* k_ptrs,
                      const void* const* v_ptrs, const int32_t* n_pos, const int32_t* block_ids,
                      int32_t n_sel, float* xb, int32_t batch,
                      int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t kv_stride,
                      int32_t block_rows, float scale) {
  return guarded(ctx, [&]() -> int {
    // the rows a list can reach are bounded by n_pos alone; a unit of rows
    // past the last one still has 32-bit row numbers
    constexpr int32_t max_n_pos = INT32_MAX - 255;
    int rc = check_attend(ctx, dtype, q, k_ptrs, v_ptrs, n_pos, xb, max_n_pos, batch, n_heads,
                          n_kv_heads, head_dim, kv_stride, scale);
    if (rc == GLA_OK) rc = check_block_rows(ctx, block_rows);
    if (rc != GLA_OK) return rc;
    if (!block_ids) return fail(ctx, GLA_ERR_INVALID_ARG, "null pointer");
    if (n_sel < 1 || (int64_t)n_sel * block_rows > INT32_MAX)
      return fail(ctx, GLA_ERR_INVALID_ARG, "n_sel must be >= 1 and n_sel * block_rows below 2^31");
    AttendRequest r = attend_request(ctx, dtype, q, k_ptrs, v_ptrs, n_pos, max_n_pos, xb, batch,
                                     n_heads, n_kv_heads, head_dim, kv_stride, scale);
    r.block_ids = block_ids;
    r.n_sel = n_sel;
    r.block_rows = block_rows;
    rc = ensure_scores(ctx, attend_workspace_floats(r, ctx->dev));
    if (rc != GLA_OK) return rc;
    r.scores = ctx->scores;
    std::string err;
    return finish(ctx, launch_attend(r, ctx->dev, ctx->stream, &err), err);
  });
}

int32_t decode_weights(gla_ctx* ctx, int dtype, const float* q, const void* const* k_ptrs,
                       const void* const* v_ptrs, const int32_t* n_pos, int32_t max_n_pos,
                       float* xb, float* const* weight_ptrs, int64_t weight_stride, int32_t batch,
                       int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t kv_stride,
                       float scale) {
  return guarded(ctx, [&]() -> int {
    int rc = check_attend(ctx, dtype, q, k_ptrs, v_ptrs, n_pos, xb, max_n_pos, batch, n_heads,
                          n_kv_heads, head_dim, kv_stride, scale);
    if (rc != GLA_OK) return rc;
    if (!weight_ptrs) return fail(ctx, GLA_ERR_INVALID_ARG, "null pointer");
    if (weight_stride < max_n_pos)
      return fail(ctx, GLA_ERR_INVALID_ARG, "weight_stride must be >= max_n_pos");
    AttendRequest r = attend_request(ctx, dtype, q, k_ptrs, v_ptrs, n_pos, max_n_pos, xb, batch,
                                     n_heads, n_kv_heads, head_dim, kv_stride, scale);
    r.weight_ptrs = weight_ptrs;
    r.weight_stride = weight_stride;
    rc = ensure_scores(ctx, attend_workspace_floats(r, ctx->dev));
    if (rc != GLA_OK) return rc;
    r.scores = ctx->scores;
    std::string err;
    return finish(ctx, launch_attend(r, ctx->dev, ctx->stream, &err), err);
  });
}

int32_t kv_evict(gla_ctx* ctx, int dtype, void* const* k_ptrs, void* const* v_ptrs,
                 float* const* weight_ptrs, int64_t weight_stride, const int32_t* n_pos,
                 int32_t max_n_pos, int32_t n_keep, int32_t n_recent, int32_t* kept,
                 void* const* k_out_ptrs, void* const* v_out_ptrs, float* const* weight_out_ptrs,
                 int64_t weight_out_stride, int32_t batch, int32_t n_kv_heads, int32_t head_dim,
                 int64_t kv_stride) {
  return guarded(ctx, [&]() -> int {
    if (!k_ptrs || !v_ptrs || !weight_ptrs || !n_pos || !kept)
      return fail(ctx, GLA_ERR_INVALID_ARG, "null pointer");
    if ((k_out_ptrs != nullptr) != (v_out_ptrs != nullptr) ||
        (k_out_ptrs != nullptr) != (weight_out_ptrs != nullptr))
      return fail(ctx, GLA_ERR_INVALID_ARG, "the output caches come all three or not at all");
    if (max_n_pos < 1) return fail(ctx, GLA_ERR_INVALID_ARG, "max_n_pos must be >= 1");
    if (n_keep < 1 || n_recent < 0 || n_recent > n_keep)
      return fail(ctx, GLA_ERR_INVALID_ARG, "n_keep must be >= 1 and 0 <= n_recent <= n_keep");
    if (weight_stride < max_n_pos)
      return fail(ctx, GLA_ERR_INVALID_ARG, "weight_stride must be >= max_n_pos");
    if (k_out_ptrs && weight_out_stride < std::min(n_keep, max_n_pos))
      return fail(ctx, GLA_ERR_INVALID_ARG, "weight_out_stride must hold the kept rows");
    int rc = check_heads(ctx, batch, n_kv_heads, n_kv_heads, head_dim);
    if (rc == GLA_OK) rc = check_stride(ctx, dtype, n_kv_heads, head_dim, kv_stride);
    if (rc != GLA_OK) return rc;
    EvictRequest r{};
    r.dtype = dtype;
    r.k_ptrs = k_ptrs;
    r.v_ptrs = v_ptrs;
    r.weight_ptrs = weight_ptrs;
    r.weight_stride = weight_stride;
    r.n_pos = n_pos;
    r.max_n_pos = max_n_pos;
    r.n_keep = n_keep;
    r.n_recent = n_recent;
    r.kept = kept;
    r.k_out_ptrs = k_out_ptrs;
    r.v_out_ptrs = v_out_ptrs;
    r.weight_out_ptrs = weight_out_ptrs;
    r.weight_out_stride = weight_out_stride;
    r.batch = batch;
    r.n_kv = n_kv_heads;
    r.head_dim = head_dim;
    r.kv_stride = kv_stride;
    r.status = ctx->status;
    std::string err;
    return finish(ctx, launch_evict(r, ctx->dev, ctx->stream, &err), err);
  });
}

const void* const* untyped(const uint16_t* const* p) {
  return reinterpret_cast<const void* const*>(p);
}
const void* const* untyped(const float* const* p) {
  return reinterpret_cast<const void* const*>(p);
}
void* const* untyped(uint16_t* const* p) { return reinterpret_cast<void* const*>(p); }
void* const* untyped(float* const* p) { return reinterpret_cast<void* const*>(p); }

}  // namespace

extern "C" {

#define GLA_CACHE_API(SUFFIX, T, DTYPE)                                                          \
  int32_t gla_block_bounds_##SUFFIX(                                                             \
      gla_ctx* ctx, const T* const* k_ptrs, const int32_t* start_pos, const int32_t* n_pos,      \
      int32_t max_n_pos, T* const* bounds_ptrs, int32_t batch, int32_t n_kv_heads,               \
      int32_t head_dim, int64_t kv_stride, int32_t block_rows) {                                 \
    return block_bounds(ctx, DTYPE, untyped(k_ptrs), start_pos, n_pos, max_n_pos,                \
                        untyped(bounds_ptrs), batch, n_kv_heads, head_dim, kv_stride,            \
                        block_rows);                                                             \
  }                                                                                              \
  int32_t gla_rope_append_batched_##SUFFIX(                                                      \
      gla_ctx* ctx, const float* q, const float* k, const float* v, float* q_out,                \
      T* const* k_ptrs, T* const* v_ptrs, const int32_t* positions, const int32_t* rows,         \
      T* const* bounds_ptrs, int32_t block_rows, int32_t batch, int32_t n_heads,                 \
      int32_t n_kv_heads, int32_t head_dim, int64_t kv_stride, int32_t context_length,           \
      float theta, int32_t rope_style) {                                                         \
    return append_batched(ctx, DTYPE, q, k, v, q_out, untyped(k_ptrs), untyped(v_ptrs),          \
                          positions, rows, untyped(bounds_ptrs), block_rows, batch, n_heads,     \
                          n_kv_heads, head_dim, kv_stride, context_length, theta, rope_style);   \
  }                                                                                              \
  int32_t gla_block_select_##SUFFIX(                                                             \
      gla_ctx* ctx, const float* q, const T* const* bounds_ptrs, const int32_t* n_pos,           \
      int32_t max_n_pos, int32_t* block_ids, int32_t batch, int32_t n_heads,                     \
      int32_t n_kv_heads, int32_t head_dim, int32_t block_rows, int32_t n_sel, int32_t n_first,  \
      int32_t n_last) {                                                                          \
    return block_select(ctx, DTYPE, q, untyped(bounds_ptrs), n_pos, max_n_pos, block_ids, batch, \
                        n_heads, n_kv_heads, head_dim, block_rows, n_sel, n_first, n_last);      \
  }                                                                                              \
  int32_t gla_decode_blocks_##SUFFIX(                                                            \
      gla_ctx* ctx, const float* q, const T* const* k_ptrs, const T* const* v_ptrs,              \
      const int32_t* n_pos, const int32_t* block_ids, int32_t n_sel, float* xb, int32_t batch,   \
      int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t kv_stride,                  \
      int32_t block_rows, float scale) {                                                         \
    return decode_blocks(ctx, DTYPE, q, untyped(k_ptrs), untyped(v_ptrs), n_pos,                 \
                         block_ids, n_sel, xb, batch, n_heads, n_kv_heads, head_dim, kv_stride,  \
                         block_rows, scale);                                                     \
  }                                                                                              \
  int32_t gla_decode_weights_##SUFFIX(                                                           \
      gla_ctx* ctx, const float* q, const T* const* k_ptrs, const T* const* v_ptrs,              \
      const int32_t* n_pos, int32_t max_n_pos, float* xb, float* const* weight_ptrs,             \
      int64_t weight_stride, int32_t batch, int32_t n_heads, int32_t n_kv_heads,                 \
      int32_t head_dim, int64_t kv_stride, float scale) {                                        \
    return decode_weights(ctx, DTYPE, q, untyped(k_ptrs), untyped(v_ptrs), n_pos, max_n_pos, xb, \
                          weight_ptrs, weight_stride, batch, n_heads, n_kv_heads, head_dim,      \
                          kv_stride, scale);                                                     \
  }                                                                                              \
  int32_t gla_kv_evict_##SUFFIX(                                                                 \
      gla_ctx* ctx, T* const* k_ptrs, T* const* v_ptrs, float* const* weight_ptrs,               \
      int64_t weight_stride, const int32_t* n_pos, int32_t max_n_pos, int32_t n_keep,            \
      int32_t n_recent, int32_t* kept, T* const* k_out_ptrs, T* const* v_out_ptrs,               \
      float* const* weight_out_ptrs, int64_t weight_out_stride, int32_t batch,                   \
      int32_t n_kv_heads, int32_t head_dim, int64_t kv_stride) {                                 \
    return kv_evict(ctx, DTYPE, untyped(k_ptrs), untyped(v_ptrs), weight_ptrs, weight_stride,    \
                    n_pos, max_n_pos, n_keep, n_recent, kept, untyped(k_out_ptrs),               \
                    untyped(v_out_ptrs), weight_out_ptrs, weight_out_stride, batch, n_kv_heads,  \
                    head_dim, kv_stride);                                                        \
  }

GLA_CACHE_API(f32kv, float, GLA_DTYPE_F32)
GLA_CACHE_API(f16kv, uint16_t, GLA_DTYPE_F16)

}  // extern "C"
