// The library context behind llmr_ctx and the host helpers that every entry
// point uses: status messages, launch accounting, the tensor-map encoder.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <string>

#include "../../include/llmr_attn.h"

constexpr size_t kSyncInts = 1 + 65536;

// Bits of the context's device error word, read and cleared by llmr_sync.
enum : int {
  kErrTimeout = 1,  // a bounded wait expired
  kErrInput = 2,    // a device-side length, slot, position or page is out of range
  kErrPages = 4,    // the free list is shorter than the step needs
};

struct llmr_ctx {
  int device = 0;
  cudaStream_t stream = nullptr;
  bool own_stream = false;
  void *ws = nullptr;
  size_t ws_bytes = 0;
  int *d_err = nullptr;
  int *d_sync = nullptr;  // fused-prologue piece counters (self-resetting)
  unsigned long long *timeline = nullptr;  // LLMR_TIMELINE builds: event buffer
  uint64_t launches = 0;
  int num_sms = 0;    // SMs the persistent kernels may use (llmr_ctx_set_sm_budget)
  int total_sms = 0;  // SMs of the device
  bool prof_on = false;
  bool prof_valid = false;
  cudaEvent_t prof_ev[3] = {nullptr, nullptr, nullptr};
  std::string err;
};

namespace llmr {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t,
                                  void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *,
                                  CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

inline int fail(llmr_ctx *ctx, int code, const char *fmt, ...) {
  if (ctx) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    ctx->err = buf;
  }
  return code;
}

#define CUDA_TRY(ctx, call)                                                   \
  do {                                                                        \
    cudaError_t e_ = (call);                                                  \
    if (e_ != cudaSuccess)                                                    \
      return fail(ctx, LLMR_ECUDA, "%s: %s", #call, cudaGetErrorString(e_));  \
  } while (0)

// Checks the launch that was just enqueued.
inline int after_launch(llmr_ctx *ctx, const char *what) {
  ctx->launches++;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return fail(ctx, LLMR_ECUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return LLMR_OK;
}

// Launches a kernel that waits for its predecessor itself (griddep_wait before
// its first access to memory): its start-up overlaps the end of the kernel
// before it on the stream. cluster: CTAs per cluster.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_overlapped(void (*kern)(KArgs...), dim3 grid, int threads, int smem,
                                     cudaStream_t stream, int cluster, const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

inline EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

}  // namespace llmr
