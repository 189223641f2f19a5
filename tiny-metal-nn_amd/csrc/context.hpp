// context.hpp -- what the library's host files share: the context, the
// thread-local error message and device buffers.
#pragma once

#include <hip/hip_runtime.h>

#include <mutex>
#include <string>

#include "tmnn_hip.h"

namespace tmnn_hip {

// Sets the calling thread's message (tmnn_last_error) and returns `code`.
int fail(int code, const std::string &msg);

struct DevBuf {
  void *ptr = nullptr;
  size_t bytes = 0;
  bool borrowed = false;  // ptr is a region of the device scratch (never freed or grown)
  DevBuf() = default;
  DevBuf(const DevBuf &) = delete;
  DevBuf &operator=(const DevBuf &) = delete;
  ~DevBuf() {
    if (ptr && !borrowed) (void)hipFree(ptr);
  }
  hipError_t ensure(size_t want) {
    if (want <= bytes) return hipSuccess;
    if (borrowed) return hipErrorInvalidValue;  // a scratch region never grows
    if (ptr) {
      (void)hipFree(ptr);
      ptr = nullptr;
      bytes = 0;
    }
    const size_t rounded = (want + 255) / 256 * 256;
    hipError_t e = hipMalloc(&ptr, rounded);
    if (e == hipSuccess)
      bytes = rounded;
    else
      (void)hipGetLastError();  // returned here; the next launch's check must not find it
    return e;
  }
  template <class T>
  T *as() const {
    return static_cast<T *>(ptr);
  }
};

}  // namespace tmnn_hip

#define TMNN_HIP_TRY(expr)                                                   \
  do {                                                                       \
    hipError_t e_ = (expr);                                                  \
    if (e_ != hipSuccess)                                                    \
      return fail(TMNN_ERR_GPU, std::string(#expr) + ": " + hipGetErrorString(e_)); \
  } while (0)

struct tmnn_context {
  int device = 0;
  hipStream_t stream = nullptr;
  int cu_count = 0;
  uint64_t mem_bytes = 0;
  std::string name;
  unsigned char *scratch = nullptr;  // this device's copy of the step scratch (device address)
  // Pinned host memory of the host-pointer calls whose arrays fit (stage_in /
  // stage_out): inputs, then outputs, then the step's loss (kStageTotal
  // bytes, freed with the context). One call at a time holds it (StageLease).
  unsigned char *stage = nullptr;
  std::mutex stage_mu;
};
