// ops_common.cuh -- what the operator files (ops_*.cu) share: element types,
// the device guard and the boundary that turns C++ failures into statuses.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <exception>
#include <memory>
#include <new>
#include <string>

#include "../../include/svl_gpu.h"
#include "common.cuh"
#include "model.cuh"

namespace svl {

// Makes `device` current for a scope; the caller's device comes back after it.
struct DeviceGuard {
  int before = -1;
  cudaError_t status = cudaSuccess;
  explicit DeviceGuard(int device) {
    status = cudaGetDevice(&before);
    if (status == cudaSuccess && before != device) status = cudaSetDevice(device);
    else if (status == cudaSuccess) before = -1;  // nothing to restore
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};

// Frees a handle's memory.  cudaFree inside another stream's capture is refused and
// breaks that capture unless the thread says that it may happen there; a handle can go at
// any time, with its owner's last reference.
inline void free_block(int device, void* block) {
  if (!block) return;
  DeviceGuard on(device);
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  const bool swapped = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
  cudaFree(block);
  if (swapped) cudaThreadExchangeStreamCaptureMode(&mode);
}

inline int refuse(int status, const std::string& message, char* err, size_t err_len) {
  set_err(err, err_len, message);
  return status;
}

inline int cuda_failure(cudaError_t e, char* err, size_t err_len) {
  cudaGetLastError();  // a refused launch or allocation is not sticky
  return refuse(e == cudaErrorMemoryAllocation ? SVL_LIMIT_EXCEEDED : SVL_INTERNAL,
                std::string("CUDA error: ") + cudaGetErrorString(e), err, err_len);
}

// Runs the body of a C entry point; no exception leaves it.
template <typename F>
int guarded(char* err, size_t err_len, F&& body) {
  try {
    return body();
  } catch (const std::bad_alloc&) {
    return refuse(SVL_LIMIT_EXCEEDED, "out of host memory", err, err_len);
  } catch (const std::exception& e) {
    return refuse(SVL_INTERNAL, e.what(), err, err_len);
  }
}

inline uint32_t dtype_size(uint32_t dtype) { return dtype == SVL_DTYPE_F32 ? 4 : 2; }
inline bool is_operand_dtype(uint32_t dtype) { return dtype <= SVL_DTYPE_F16; }

// Exact widening to FP32 and one rounding (nearest even) back.
SVL_DEV float widen(float x) { return x; }
SVL_DEV float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
SVL_DEV float widen(__half x) { return __half2float(x); }
template <typename T>
SVL_DEV T narrow(float x);
template <>
SVL_DEV float narrow<float>(float x) {
  return x;
}
template <>
SVL_DEV __nv_bfloat16 narrow<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
SVL_DEV __half narrow<__half>(float x) {
  return __float2half_rn(x);
}

}  // namespace svl
