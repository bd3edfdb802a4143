// gla_ctx.h - the context behind the C ABI and the small helpers every entry
// point uses (api.cu, api_cache.cu).  Not installed; not part of the ABI.
#pragma once

#include <cuda_runtime.h>

#include <string>
#include <vector>

#include "gpullama_attn.h"
#include "gla_comm.h"
#include "gla_internal.h"
#include "gla_peer.h"

struct gla_ctx {
  int device = 0;
  cudaStream_t stream = nullptr;
  gla::DeviceInfo dev{};
  int32_t* status = nullptr;        // device status word
  int32_t* counters = nullptr;      // piece counters (zero between calls)
  size_t counters_cap = 0;
  uint64_t* parts = nullptr;        // piece slots (tagged 64-bit words, zeroed at allocation)
  size_t parts_cap = 0;             // words
  uint64_t* trace = nullptr;        // GLA_OPT_TRACE: per-CTA phase stamps of the last decode
  size_t trace_words = 0;
  float* records = nullptr;         // sharded decode: local records
  float* gathered = nullptr;        // sharded decode: all ranks' records
  size_t records_cap = 0;           // floats per rank
  uint16_t* ingest_ws = nullptr;    // prompt ingestion: FP16 q (and K/V) copies
  size_t ingest_cap = 0;            // halves
  gla::Comm comm;
  gla::PeerExchange xch;            // sharded decode: peer exchange buffers
  int32_t opt_early_kv = 2;         // GLA_OPT_EARLY_KV_PREFETCH
  int32_t opt_shard_exchange = 1;   // GLA_OPT_SHARD_EXCHANGE
  float* scores = nullptr;          // scores and parts (gla_decode_weights_*, _blocks_*)
  size_t scores_cap = 0;            // floats
  std::vector<void*> retired;       // outgrown scores: captured graphs may still name them
  std::string last_error;
};

namespace gla {

inline int fail(gla_ctx* ctx, int code, const std::string& msg) {
  if (ctx) ctx->last_error = msg;
  return code;
}

inline int cuda_fail(gla_ctx* ctx, cudaError_t e, const char* what) {
  return fail(ctx, GLA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The context's 256-byte status block: the device status word at 0, the
// decode call-epoch word (see DecodeWorkspace) at kEpochOffset.
constexpr size_t kEpochOffset = 64;

// Makes the context's device current for the duration of a call.
struct DeviceGuard {
  int prev = -1;
  int device;
  bool ok = true;
  explicit DeviceGuard(int dev) : device(dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
  }
  ~DeviceGuard() {
    if (prev >= 0 && prev != device) cudaSetDevice(prev);
  }
};

inline bool stream_capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(s, &st) != cudaSuccess) return false;
  return st != cudaStreamCaptureStatusNone;
}

}  // namespace gla
