// logits_host.hpp -- what the host files of the class-logit operators share: the
// handle, host arrays' way to the device and back, and the guard of C entries.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <new>
#include <vector>

#include "arg_types.hpp"
#include "context.hpp"
#include "tmnn_hip.h"

struct tmnn_logits {
  tmnn_context *ctx = nullptr;
  tmnn_hip::DevBuf work;    // part sums, part keys, listed logits
  tmnn_hip::DevBuf arena;   // arrays of the host-pointer calls
  std::mutex host_mu;       // the arena belongs to one host-pointer call
  std::mutex mu;            // the fields below, and the order of calls that share `work`
  bool used = false;        // a call has taken the workspace, the last one on `last`
  hipStream_t last = nullptr;  // (only compared for a capture: the stream may be gone)
  bool recorded = false;    // `done` follows the last such call that no capture took
  hipEvent_t done = nullptr;
};

namespace tmnn_hip {

inline hipStream_t stream_of(tmnn_logits *h, void *stream) {
  return stream == TMNN_STREAM_CONTEXT ? h->ctx->stream : static_cast<hipStream_t>(stream);
}

// The host arrays of a call and their places in the handle's arena.
class HostArrays {
 public:
  enum Dir { kIn, kOut, kRoom };
  // `rows` x `width` bytes, `pitch` bytes from row to row on the host; packed on the device
  template <class P>
  void add(P *&slot, Dir dir, int64_t rows, size_t width, size_t pitch) {
    if (!slot || rows == 0 || width == 0) return;
    items_.push_back({const_cast<void *>(static_cast<const void *>(slot)),
                      const_cast<void **>(reinterpret_cast<const void *const *>(&slot)), dir, rows,
                      width, rows == 1 ? width : pitch, bytes_, {}});
    bytes_ += (static_cast<size_t>(rows) * width + 255) / 256 * 256;
  }
  template <class P>
  void add(P *&slot, Dir dir, int64_t rows, size_t width) {
    add(slot, dir, rows, width, width);
  }
  // room on the device alone
  void room(void *&slot, size_t bytes) {
    items_.push_back({nullptr, &slot, kRoom, 1, bytes, bytes, bytes_, {}});
    bytes_ += (bytes + 255) / 256 * 256;
  }
  // Rows that are not adjacent on the host are packed there (a copy of rows over a pitch takes
  // the runtime a transfer a row).
  int enter(tmnn_logits *h) {
    TMNN_HIP_TRY(h->arena.ensure(std::max<size_t>(bytes_, 256)));
    for (Item &i : items_) {
      char *d = h->arena.as<char>() + i.at;
      *i.slot = d;
      const size_t bytes = static_cast<size_t>(i.rows) * i.width;
      if (i.pitch != i.width) i.packed.resize(bytes);
      if (i.dir != kIn) continue;
      const char *from = static_cast<const char *>(i.host);
      for (int64_t r = 0; i.pitch != i.width && r < i.rows; ++r)
        std::memcpy(i.packed.data() + r * i.width, from + r * i.pitch, i.width);
      TMNN_HIP_TRY(hipMemcpyAsync(d, i.pitch != i.width ? i.packed.data() : from, bytes,
                                  hipMemcpyHostToDevice, h->ctx->stream));
    }
    return TMNN_OK;
  }
  // Enqueues the copies out; `place` puts them where they belong once they are there.
  int leave(tmnn_logits *h) {
    for (Item &i : items_)
      if (i.dir == kOut)
        TMNN_HIP_TRY(hipMemcpyAsync(i.pitch != i.width ? i.packed.data() : i.host,
                                    h->arena.as<char>() + i.at,
                                    static_cast<size_t>(i.rows) * i.width, hipMemcpyDeviceToHost,
                                    h->ctx->stream));
    return TMNN_OK;
  }
  void place() const {
    for (const Item &i : items_)
      for (int64_t r = 0; i.dir == kOut && i.pitch != i.width && r < i.rows; ++r)
        std::memcpy(static_cast<char *>(i.host) + r * i.pitch, i.packed.data() + r * i.width, i.width);
  }

 private:
  struct Item {
    void *host;
    void **slot;
    Dir dir;
    int64_t rows;
    size_t width, pitch, at;
    std::vector<char> packed;
  };
  std::vector<Item> items_;
  size_t bytes_ = 0;
};

template <class Run>
int on_host(tmnn_logits *h, HostArrays &arrays, Run run) {
  std::lock_guard<std::mutex> lock(h->host_mu);
  int rc = arrays.enter(h);
  if (rc == TMNN_OK) rc = run();
  if (rc == TMNN_OK) rc = arrays.leave(h);
  const hipError_t e = hipStreamSynchronize(h->ctx->stream);
  if (rc == TMNN_OK && e != hipSuccess)
    rc = fail(TMNN_ERR_GPU, std::string("hipStreamSynchronize: ") + hipGetErrorString(e));
  if (rc == TMNN_OK) arrays.place();
  return rc;
}

// No exception leaves a C entry point.
template <class F>
int guarded(F f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return fail(TMNN_ERR_RUNTIME, "out of host memory");
  } catch (const std::exception &e) {
    return fail(TMNN_ERR_RUNTIME, e.what());
  }
}
template <class F>
int entry(tmnn_logits *h, F f) {
  return guarded([&] { return h ? f() : fail(TMNN_ERR_INVALID_ARGUMENT, "logits handle is null"); });
}

}  // namespace tmnn_hip
