// Host helpers of the handle-free operators declared in gptoss_decode_b200.h.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/gptoss_decode_b200.h"

namespace gptoss {

// decode.cu: error text that gptoss_decode_last_error(NULL) returns on this thread
int decode_error(int code, const char *fmt, ...);

// The device that holds `ptr` becomes current for the scope; `code` is 0 or the error that
// the entry point returns.  An operator's launch goes to the GPU of its output, whatever
// device the calling thread has selected.
class OnDeviceOf {
 public:
  OnDeviceOf(const void *ptr, const char *what) {
    cudaPointerAttributes attr = {};
    cudaError_t e = cudaPointerGetAttributes(&attr, ptr);
    if (e != cudaSuccess) {
      cudaGetLastError();  // not sticky: the next call starts clean
      code = decode_error(GPTOSS_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
      return;
    }
    if (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged) {
      code = decode_error(GPTOSS_E_INVALID, "%s is not device memory", what);
      return;
    }
    e = cudaGetDevice(&before_);
    if (e == cudaSuccess && attr.device != before_) {
      e = cudaSetDevice(attr.device);
      switched_ = e == cudaSuccess;
    }
    if (e != cudaSuccess) {
      cudaGetLastError();
      code = decode_error(GPTOSS_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
      return;
    }
    device = attr.device;
  }
  ~OnDeviceOf() {
    if (switched_) cudaSetDevice(before_);
  }
  OnDeviceOf(const OnDeviceOf &) = delete;
  OnDeviceOf &operator=(const OnDeviceOf &) = delete;

  int code = 0;
  int device = -1;

 private:
  int before_ = -1;
  bool switched_ = false;
};

// Result of a launch (cudaLaunchKernelEx) or of a call before it -> status code of the entry
// point.  The thread's last error is not asked: it may be left over from something else.
inline int launch_result(const char *what, cudaError_t e) {
  if (e == cudaSuccess) return GPTOSS_OK;
  cudaGetLastError();  // not sticky: the next call starts clean
  return decode_error(GPTOSS_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Multiprocessors of the device (looked up once per device).
int sm_count(int device);

// token_attention.cu: prompt attention of sequences with a few query rows each
int launch_token_attention(const gptoss_attention_args_t &a, int sms, cudaStream_t st);

inline bool aligned(const void *p, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

}  // namespace gptoss
