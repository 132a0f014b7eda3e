// internal.h -- host-side helpers shared by the wisp_b200 translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <utility>

#include "wisp_b200.h"

namespace wb {

// Launches a kernel of the per-layer chain in plain stream order (errors are
// left for cudaGetLastError).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_k(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                            cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = nullptr;
  cfg.numAttrs = 0;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// The same launch as a programmatic dependent of the kernel before it on the
// stream: its CTAs may start while that kernel is still running (once all of
// that kernel's CTAs have started and triggered), and must execute
// griddepcontrol.wait (wb::pdl_wait) before they read anything that kernel,
// or any kernel before it, writes. Used for one edge only, router logits ->
// decode planner in the single-GPU decode chain: measured on B200 (CUDA
// graph, L2 flushed), making the gate/up kernel a dependent of the planner
// cost Mixtral b1 6 us, and the down kernel a dependent of gate/up gained
// nothing.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_k_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                                cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// The register path's unit plans of one grouped call, as the decode planner
// (route.cu) writes them in place of the grouped call's own planner
// (grouped.cu): the plan arrays in the call's workspace and the numbers that
// shape them.
struct DecodeUnits {
  int32_t* units_gu;
  int32_t* units_dn;
  uint8_t* xq;   // q16 input rows in the same workspace
  int per_gu, per_dn, cols, sk_rows, ks_dn, nk_dn, target;
};

// cuTensorMapEncodeTiled from the loaded driver (nullptr without one).
using TensorMapEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                       const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                       const cuuint32_t*, CUtensorMapInterleave,
                                       CUtensorMapSwizzle, CUtensorMapL2promotion,
                                       CUtensorMapFloatOOBfill);
TensorMapEncodeFn tensor_map_encoder();

// SMs of the current device, and a kernel's dynamic shared memory raised to
// `bytes` (both asked of the driver once per device: a call costs as much as a
// small kernel's launch).
inline cudaError_t device_sms(int* dev, int* sms) {
  static std::atomic<int> known[64];
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return e;
  const bool keep = *dev >= 0 && *dev < 64;
  if (keep && (*sms = known[*dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *dev);
  if (e == cudaSuccess && keep) known[*dev].store(*sms, std::memory_order_relaxed);
  return e;
}

// `raised`: the kernel's own record, one bit per device.
template <typename K>
inline cudaError_t raise_smem(K* kernel, int bytes, int dev, std::atomic<uint64_t>& raised) {
  const uint64_t bit = dev >= 0 && dev < 64 ? (uint64_t)1 << dev : 0;
  if (raised.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) raised.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Checks shared by the fp4 weight-set entry points (fp4.cu).
WispError fp4_validate(const WispFp4Config* c, const char* who, WispErrCtx* err);

// The same for fp8 (fp8.cu) and for a routing (select.cu).
WispError fp8_validate(const WispFp8Config* c, const char* who, WispErrCtx* err);
WispError fp8_check_mats(const WispFp8Mats* m, const char* who, const char* what, WispErrCtx* err);
WispError routing_validate(const WispRouting* r, int tokens, int n_experts, int top_k,
                           const char* who, WispErrCtx* err);

// wisp_b200_select_experts over the sum of `splits` sets of fp32 logits [tokens x
// n_experts] and logit_bias (may be NULL).
WispError launch_select(const WispRouting* r, const float* part, int splits,
                        const float* logit_bias, const float* bias, int tokens, int n_experts,
                        int top_k, int* idx, float* w, cudaStream_t st, WispErrCtx* err);

// Fill a WispErrCtx the way the reference's WISP_ERR_SET does
// (csrc/core/wisp_engine.h:66-72) and return the code.
inline WispError set_err(WispErrCtx* err, WispError code, const char* file, int line,
                         const char* fmt, ...) {
  if (err) {
    err->code = code;
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err->message, sizeof(err->message), fmt, ap);
    va_end(ap);
    err->file = file;
    err->line = line;
  }
  return code;
}

}  // namespace wb

#define WB_FAIL(code, ...) ::wb::set_err(err, code, __FILE__, __LINE__, __VA_ARGS__)

#define WB_CUDA_CHECK(call)                                                          \
  do {                                                                               \
    cudaError_t _e = (call);                                                         \
    if (_e != cudaSuccess)                                                           \
      return WB_FAIL(WISP_ERR_CUDA, "CUDA error: %s", cudaGetErrorString(_e));       \
  } while (0)
