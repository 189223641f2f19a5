// logits.hip -- host side of the class-logit operators (include/tmnn_hip.h):
// argument checks, the choice of kernel and split, the workspace, and the
// host-pointer forms.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <new>
#include <vector>

#include "context.hpp"
#include "distill_kernel.hpp"
#include "logprob_kernel.hpp"
#include "tmnn_hip.h"

using namespace tmnn_hip;

namespace {

// Workspace of the calls that split rows: at most kMaxSplit parts at a time.
constexpr int kMaxSplit = 4096;
constexpr size_t kSumBytes = kMaxSplit * sizeof(float4);
constexpr int64_t kSplitKeys = 1 << 20;  // threads of these parts
constexpr size_t kKeyBytes = static_cast<size_t>(kSplitKeys) * sizeof(uint64_t);
constexpr size_t kListBytes = static_cast<size_t>(kMaxSplit) * kMaxTeacher * sizeof(float);

}  // namespace

struct tmnn_logits {
  tmnn_context *ctx = nullptr;
  DevBuf work;              // part sums, part keys, listed logits
  DevBuf arena;             // arrays of the host-pointer calls
  std::mutex host_mu;       // the arena belongs to one host-pointer call
  std::mutex mu;            // the fields below, and the order of calls that share `work`
  bool used = false;        // a call has taken the workspace, the last one on `last`
  hipStream_t last = nullptr;  // (only compared for a capture: the stream may be gone)
  bool recorded = false;    // `done` follows the last such call that no capture took
  hipEvent_t done = nullptr;
};

namespace {

size_t dtype_size(int32_t dtype) { return dtype == TMNN_DTYPE_F32 ? 4 : 2; }

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether a row of d_logits lies over a part of the logits other than its own place (at one address,
// with one row stride). Rows of both may interleave.
template <class A>
bool overlaps(const A *a) {
  typedef __int128 wide;  // strides are the caller's
  const wide size = static_cast<wide>(dtype_size(a->dtype)), n = a->rows, width = a->classes * size;
  const wide s = a->row_stride * size, ds = a->d_row_stride * size;
  const wide z = reinterpret_cast<uintptr_t>(a->logits), d = reinterpret_cast<uintptr_t>(a->d_logits);
  if (z == d) return n > 1 && s != ds;
  if (d >= z + (n - 1) * s + width || z >= d + (n - 1) * ds + width) return false;
  // the first row of logits that ends after `at`, whether there is one that begins before its end
  auto meets = [&](wide at) {
    const wide i = at < z + width ? 0 : (at - z - width) / s + 1;
    return i < n && z + i * s < at + width;
  };
  if (s == ds) {
    // rows are shifted by whole strides against each other, or lie alike in all: against the
    // rows beside it, the first row of d_logits that is not before the logits says it for all
    const wide j = d >= z ? 0 : std::min<wide>(n - 1, (z - d) / ds);
    return meets(d + j * ds) || (j + 1 < n && meets(d + (j + 1) * ds));
  }
  for (wide j = 0; j < n; ++j)
    if (meets(d + j * ds)) return true;
  return false;
}

template <class A>
int check_matrix(const A *a, const char *what, bool written) {
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (a->struct_size != sizeof(A)) return bad("struct_size mismatch");
  if (a->dtype < TMNN_DTYPE_F32 || a->dtype > TMNN_DTYPE_BF16) return bad("invalid dtype");
  if (a->index_dtype != TMNN_INDEX_I32 && a->index_dtype != TMNN_INDEX_I64)
    return bad("invalid index_dtype");
  if (a->rows < 0 || a->rows > INT32_MAX) return bad("rows must be in [0, 2^31)");
  if (a->classes < 1 || a->classes > TMNN_LOGITS_MAX_CLASSES)
    return bad("classes must be in [1, 2^24]");
  if (a->row_stride < a->classes) return bad("row_stride must be at least classes");
  if (a->d_logits && a->d_row_stride < a->classes)
    return bad("d_row_stride must be at least classes");
  // c = log2(e) / T stays an ordinary number
  if (!(a->temperature >= 1e-6f && a->temperature <= 1e6f))
    return bad("temperature must be in [1e-6, 1e6]");
  if (a->rows == 0) return TMNN_OK;
  if (!a->logits) return bad("logits is null");
  const size_t size = dtype_size(a->dtype);
  if (!aligned(a->logits, size) || !aligned(a->d_logits, size))
    return bad("logits and d_logits must be aligned to their type");
  // one row's gradient would lie over another row's logits, which it may not have read yet
  if (a->d_logits == a->logits && a->rows > 1 && a->d_row_stride != a->row_stride)
    return bad("d_logits in the place of the logits needs their row_stride");
  if (written && a->d_logits && overlaps(a))
    return bad("d_logits overlaps the logits (their own place, with their row_stride, is allowed)");
  return TMNN_OK;
}

int check_logprobs(const tmnn_token_logprobs_args *a, bool back, bool host) {
  const char *what = back ? "token_logprobs_backward" : "token_logprobs";
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (!a) return bad("args is null");
  // (host arrays are written once everything has been read)
  const int rc = check_matrix(a, what, back && !host);
  if (rc != TMNN_OK) return rc;
  if (a->top_k < 0 || a->top_k > TMNN_LOGITS_MAX_TOP) return bad("top_k must be in [0, 128]");
  if (a->rows == 0) return TMNN_OK;
  if (!aligned(a->tokens, a->index_dtype == TMNN_INDEX_I64 ? 8 : 4))
    return bad("tokens must be aligned to their type");
  for (const void *p : {static_cast<const void *>(a->logprob), static_cast<const void *>(a->entropy),
                        static_cast<const void *>(a->rank), static_cast<const void *>(a->stats),
                        static_cast<const void *>(a->top_ids),
                        static_cast<const void *>(a->top_logprobs),
                        static_cast<const void *>(a->d_logprob),
                        static_cast<const void *>(a->d_entropy),
                        static_cast<const void *>(a->d_top_logprobs)})
    if (!aligned(p, 4)) return bad("arrays of 32-bit values must be 4-byte aligned");
  if (back) {
    if (!a->d_logits) return bad("d_logits is null");
    if (!a->stats) return bad("stats is null");
    if (a->d_logprob && !a->tokens) return bad("d_logprob needs tokens");
    if (a->d_entropy && !a->entropy) return bad("d_entropy needs entropy");
    if (a->d_top_logprobs && a->top_k > 0 && !a->top_ids) return bad("d_top_logprobs needs top_ids");
    return TMNN_OK;
  }
  if (!a->top_ids != !a->top_logprobs) return bad("top_ids and top_logprobs go together");
  if (a->top_k > 0 && !a->top_ids) return bad("top_k > 0 needs top_ids and top_logprobs");
  return TMNN_OK;
}

int check_distill(const tmnn_distill_args *a, bool back, bool host) {
  const char *what = back ? "distill_backward" : "distill";
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (!a) return bad("args is null");
  const int rc = check_matrix(a, what, !host);
  if (rc != TMNN_OK) return rc;
  if (a->teacher_kind != TMNN_TEACHER_LOGITS && a->teacher_kind != TMNN_TEACHER_LOGPROBS)
    return bad("invalid teacher_kind");
  if (a->teacher_k < 1 || a->teacher_k > TMNN_LOGITS_MAX_TEACHER)
    return bad("teacher_k must be in [1, 256]");
  if (a->rows == 0) return TMNN_OK;
  if (!a->teacher_ids || !a->teacher) return bad("teacher_ids and teacher must not be null");
  if (!aligned(a->teacher_ids, a->index_dtype == TMNN_INDEX_I64 ? 8 : 4))
    return bad("teacher_ids must be aligned to their type");
  if (!aligned(a->teacher, 4) || !aligned(a->row_weights, 4) || !aligned(a->loss, 4))
    return bad("arrays of 32-bit values must be 4-byte aligned");
  if (!host && !aligned(a->stats, 16)) return bad("stats must be 16-byte aligned");
  if (back) {
    if (!a->d_logits) return bad("d_logits is null");
    if (!a->stats) return bad("stats is null");
    if (!a->row_weights) return bad("row_weights (the loss's gradient) is null");
  } else if (!a->loss && !a->stats && !a->d_logits) {
    return bad("nothing to compute");
  }
  return TMNN_OK;
}

// The workspace for the kernels that `launch` enqueues on `st`, where rows are in parts: after the
// last call that used it, whichever stream that went to. The event is recorded at once: later the
// stream may be captured, or destroyed and its handle given to another. It costs a call 1 us (64 x
// 131072 fp32 with 20 alternatives 18.0 -> 19.1), with a fence for the host, which it does not need, 3.
template <class F>
int with_workspace(tmnn_logits *h, hipStream_t st, int parts, F launch) {
  if (parts == 1) return launch();  // (one block a row: nothing goes through it)
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (st) TMNN_HIP_TRY(hipStreamIsCapturing(st, &cap));  // (the null stream cannot be captured)
  const bool captured = cap != hipStreamCaptureStatusNone;
  if (captured && h->used && h->last != st)
    return fail(TMNN_ERR_UNSUPPORTED,
                "a captured stream needs a logits handle of its own (another stream used this one)");
  if (!captured && h->recorded) {
    const hipError_t e = hipStreamWaitEvent(st, h->done, 0);
    if (e != hipSuccess) (void)hipGetLastError();  // returned here; a later check must not find it
    if (e == hipErrorStreamCaptureIsolation)
      return fail(TMNN_ERR_UNSUPPORTED,
                  "the stream of this logits handle's last call is being captured: another stream "
                  "needs another handle meanwhile");
    if (e != hipSuccess)
      return fail(TMNN_ERR_GPU, std::string("hipStreamWaitEvent: ") + hipGetErrorString(e));
  }
  h->used = true;
  h->last = st;
  int rc = launch();
  if (!captured) {
    const hipError_t e = hipEventRecord(h->done, st);
    if (e == hipSuccess)
      h->recorded = true;
    else
      (void)hipGetLastError();
    if (e != hipSuccess && rc == TMNN_OK)
      rc = fail(TMNN_ERR_GPU, std::string("hipEventRecord: ") + hipGetErrorString(e));
  }
  return rc;
}

// ---- kernels by size ---------------------------------------------------------------

// Lanes of a row in registers, 16 classes a lane (fewer where one lane holds all); 0: the
// row is too long.
int group_lanes(int64_t classes) {
  int g = 1;
  while (g <= kWave && static_cast<int64_t>(g) * 16 < classes) g *= 2;
  return g <= kWave ? g : 0;
}

// Threads of a block by the vectors of its part. A block's sums and selection cost the
// same whatever they end, so short parts go to few threads; a long part goes to
// many, which finish together. us at 64 / 128 / 256 / 512 / 1024 threads: log-probabilities
// with 20 alternatives of 16384 x 5003 bf16 (625 vectors) 82 / 70 / 106 / 200 / 335, 8192 x
// 20011 (2501) 137 / 110 / 99 / 134 / 221, 4096 x 131072 (16384) 506 / 388 / 268 / 218 / 209.
int sum_threads(int64_t vecs) {
  return vecs < 512 ? 64 : vecs < 1536 ? 128 : vecs < 5000 ? 256 : vecs < 12288 ? 512 : 1024;
}
// A block that only writes a gradient: four vectors a thread (16384 x 5003 bf16 75 / 69 / 77 /
// 98 / 137, 4096 x 131072 431 / 435 / 420 / 407 / 385).
int map_threads(int64_t vecs) {
  return vecs < 512 ? 64 : vecs < 1024 ? 128 : vecs < 2048 ? 256 : vecs < 4096 ? 512 : 1024;
}
// Sums and gradient in one block. Up to 8 vectors a thread stay in registers in between, while
// several blocks of up to 256 threads share a unit then (16384 x 8192 bf16, 1024 vectors, kept at
// 128 threads 111, read again at 128 / 256 131 / 129; f32, 2048 vectors, kept at 256 187, read
// again 238); longer rows are read again (8192 x 65536 bf16, 8192 vectors, kept at 1024 threads
// 567, read again at 512 / 1024 484 / 455; 8192 x 20011 at 128 / 256 / 512 223 / 198 / 212).
int both_threads(int64_t vecs) {
  return vecs <= 512 ? 64 : vecs <= 1024 ? 128 : vecs < 4096 ? 256 : vecs < 8192 ? 512 : 1024;
}
constexpr int kKeptVecs = 8;

struct Split {
  int threads, parts, part_len;
};

// Threads of a block, at least so many, and blocks of a row, which a second kernel joins or not.
// Few rows go to one block each, with four vectors a thread, where its time alone is less than
// that of shorter parts and the kernel that joins them: up to 4096 vectors, and up to 16384 where
// there would be fewer than four parts. us in parts / in one block, log-probabilities without
// alternatives and distillation: 1 x 32768 bf16 (4096 vectors) 5.6 / 5.0 and 9.3 / 7.9, 1 x 65536
// 5.7 / 7.0 and 9.4 / 10.7, 128 x 65536 8.3 / 8.2 and 13.3 / 13.0, 200 x 131072 17.3 / 14.3 and
// 29.5 / 25.3. The gradient of log-probabilities, whose parts leave a peaked row's best class to a
// second kernel, 1 x 32768 bf16 4.6 / 4.4, 200 x 131072 25.6 / 22.9, and less host work in one.
// Rows that would not be split gain from the threads alone while their blocks share a unit easily:
// 512 x 8192 bf16 5.6 / 4.4 and 9.7 / 9.1, but 512 x 32768 fp32 13.2 / 14.8.
Split split_of(int64_t rows, int64_t classes, int n, int (*threads)(int64_t), int at_least,
               int64_t blocks, bool joined) {
  Split s;
  const int64_t vecs = (classes + n - 1) / n;
  const int64_t one = 2 * rows > blocks ? 2048 : 4 * rows > blocks ? 16384 : 4096;
  if (joined && rows <= blocks && vecs <= one) {
    s = {64, 1, static_cast<int>(classes)};
    while (s.threads < 1024 && (s.threads * kLogitVecs < vecs || s.threads < at_least)) s.threads *= 2;
    return s;
  }
  int64_t parts = 1;
  if (rows < blocks) parts = std::min<int64_t>(blocks / rows, vecs / (2 * 256));
  parts = std::max<int64_t>(parts, (classes + kMaxPartLen - 1) / kMaxPartLen);
  parts = std::min<int64_t>(std::max<int64_t>(parts, 1), kMaxParts);
  int64_t len = (classes + parts - 1) / parts;
  if (parts > 1) len = (len + 255) / 256 * 256;
  s.part_len = static_cast<int>(len);
  s.parts = static_cast<int>((classes + len - 1) / len);
  s.threads = threads((len + n - 1) / n);
  while (s.threads < at_least) s.threads *= 2;
  return s;
}

// Blocks that few rows are split into, with at least 512 vectors each: two a unit (64 x 131072
// fp32, 20 alternatives, part and join kernel: 11.4 + 7.5 us, with 1024 blocks 9.9 + 9.4).
constexpr int64_t kSplitBlocks = 512;
// Alternatives up to which rows stay in registers: each costs a round over the row there, all of
// them one selection in a block of 64 threads and more. us in registers / in blocks, by the lanes
// of a row:
//   64  65536 x 600 bf16, fp32 with 1 66 / 64, 69 / 63, with 2 77 / 68, 77 / 64; 65536 x 1000 with 2
//       78 / 69, 81 / 70
//   32  65536 x 510 bf16 with 4 53 / 70 and with 20 144 / 79
//   16  131072 x 250 bf16 with 3 44 / 119, 20 137 / 138, 32 201 / 469, 64 373 / 917, 128 719 / 955; fp32
//       with 20 137 / 125, 32 202 / 129, 64 375 / 907
//   8   131072 x 128 bf16 with 20 69 / 257, 64 188 / 292, 128 359 / 435
// (a block selects among the maxima of its threads that have classes, and a row of 250 has few:
// it bounds 32 and more of them badly).
int group_top(int g) { return g <= 16 ? kMaxTop : g == 32 ? 4 : 0; }

// Rows of one launch: at most 2^31 threads, and the workspace of its parts.
template <class F>
int in_slices(int64_t rows, int64_t threads_per_row, int parts, F launch) {
  int64_t step = std::max<int64_t>(1, (1ll << 31) / threads_per_row - 1);
  if (parts > 1)
    step = std::min<int64_t>(step, std::min<int64_t>(kMaxSplit / parts, kSplitKeys / threads_per_row));
  for (int64_t at = 0; at < rows; at += step) {
    launch(at, static_cast<int32_t>(std::min(step, rows - at)));
    TMNN_HIP_TRY(hipGetLastError());
  }
  return TMNN_OK;
}

dim3 group_grid(int64_t rows, int g) {  // (rows of one lane pass 2^31 - per)
  const int64_t per = kGroupThreads / g;
  return dim3(static_cast<uint32_t>((rows + per - 1) / per));
}

#define TMNN_BY_GROUP(g, CALL)                          \
  switch (g) {                                          \
    case 1:                                             \
      if (a.classes <= n) {                             \
        CALL(1, 1);                                     \
      } else if (a.classes <= 8) {                      \
        CALL(1, 8 / n);                                 \
      } else {                                          \
        CALL(1, 16 / n);                                \
      }                                                 \
      break;                                            \
    case 2: CALL(2, 16 / n); break;                     \
    case 4: CALL(4, 16 / n); break;                     \
    case 8: CALL(8, 16 / n); break;                     \
    case 16: CALL(16, 16 / n); break;                   \
    case 32: CALL(32, 16 / n); break;                   \
    default: CALL(64, 16 / n); break;                   \
  }
#define TMNN_BY_THREADS(nt, CALL) \
  switch (nt) {                   \
    case 64: CALL(64); break;     \
    case 128: CALL(128); break;   \
    case 256: CALL(256); break;   \
    case 512: CALL(512); break;   \
    default: CALL(1024); break;   \
  }

template <class T>
LogprobArgs logprob_slice(const LogprobArgs &a, int64_t at, int32_t rows) {
  LogprobArgs s = a;
  auto move = [&](auto *&p, int64_t n) {
    if (p) p += at * n;
  };
  s.rows = rows;
  s.logits = static_cast<const T *>(a.logits) + at * a.row_stride;
  if (a.tokens) s.tokens = static_cast<const char *>(a.tokens) + at * (a.wide_index ? 8 : 4);
  move(s.logprob, 1);
  move(s.entropy, 1);
  move(s.rank, 1);
  move(s.stats, 2);
  move(s.top_ids, a.top_k);
  move(s.top_logprobs, a.top_k);
  move(s.d_logprob, 1);
  move(s.d_entropy, 1);
  move(s.d_top, a.top_k);
  move(s.entropy_in, 1);
  move(s.stats_in, 2);
  move(s.top_in, a.top_k);
  if (a.d_logits) s.d_logits = static_cast<T *>(a.d_logits) + at * a.d_row_stride;
  return s;
}

template <class T>
int run_logprobs(tmnn_logits *h, LogprobArgs a, int64_t rows, hipStream_t st) {
  constexpr int n = Row<T>::n;
  const int g = group_lanes(a.classes);
  if (g != 0 && a.top_k <= group_top(g)) {
    return in_slices(rows, g, 1, [&](int64_t at, int32_t r) {
      const LogprobArgs s = logprob_slice<T>(a, at, r);
#define CALL(G, NV) \
  hipLaunchKernelGGL((logprob_group_kernel<T, G, NV>), group_grid(r, G), dim3(kGroupThreads), 0, st, s)
      TMNN_BY_GROUP(g, CALL)
#undef CALL
    });
  }
  const Split sp = split_of(rows, a.classes, n, sum_threads, 2 * a.top_k, kSplitBlocks, true);
  a.parts = sp.parts;
  a.part_len = sp.part_len;
  a.part_threads = sp.threads;
  a.part_sum = static_cast<float4 *>(h->work.ptr);
  a.part_key = reinterpret_cast<uint64_t *>(static_cast<char *>(h->work.ptr) + kSumBytes);
  const int64_t threads = static_cast<int64_t>(sp.threads) * a.parts;
  return with_workspace(h, st, a.parts, [&] {
    return in_slices(rows, threads, a.parts, [&](int64_t at, int32_t r) {
      const LogprobArgs s = logprob_slice<T>(a, at, r);
#define CALL(NT) \
  hipLaunchKernelGGL((logprob_block_kernel<T, NT>), dim3(r * a.parts), dim3(NT), 0, st, s)
      TMNN_BY_THREADS(sp.threads, CALL)
#undef CALL
      if (a.parts > 1)
        hipLaunchKernelGGL((logprob_join_kernel<T>), dim3(r), dim3(kJoinThreads), 0, st, s);
    });
  });
}

template <class T>
int run_logprobs_grad(tmnn_logits *h, LogprobArgs a, int64_t rows, hipStream_t st) {
  constexpr int n = Row<T>::n;
  if (const int g = group_lanes(a.classes)) {
    return in_slices(rows, g, 1, [&](int64_t at, int32_t r) {
      const LogprobArgs s = logprob_slice<T>(a, at, r);
#define CALL(G, NV)                                                                          \
  hipLaunchKernelGGL((logprob_grad_group_kernel<T, G, NV>), group_grid(r, G), dim3(kGroupThreads), 0, \
                     st, s)
      TMNN_BY_GROUP(g, CALL)
#undef CALL
    });
  }
  const Split sp = split_of(rows, a.classes, n, map_threads, a.d_top ? a.top_k + 1 : 1, kSplitBlocks,
                            true);
  a.parts = sp.parts;
  a.part_len = sp.part_len;
  a.part_sum = static_cast<float4 *>(h->work.ptr);
  const int64_t threads = static_cast<int64_t>(sp.threads) * a.parts;
  return with_workspace(h, st, a.parts, [&] {
    return in_slices(rows, threads, a.parts, [&](int64_t at, int32_t r) {
      const LogprobArgs s = logprob_slice<T>(a, at, r);
#define CALL(NT) \
  hipLaunchKernelGGL((logprob_grad_block_kernel<T, NT>), dim3(r * a.parts), dim3(NT), 0, st, s)
      TMNN_BY_THREADS(sp.threads, CALL)
#undef CALL
      if (a.parts > 1)
        hipLaunchKernelGGL((logprob_grad_best_kernel<T>), dim3(r), dim3(kBestThreads), 0, st, s);
    });
  });
}

template <class T>
DistillArgs distill_slice(const DistillArgs &a, int64_t at, int32_t rows) {
  DistillArgs s = a;
  s.rows = rows;
  s.logits = static_cast<const T *>(a.logits) + at * a.row_stride;
  s.ids = static_cast<const char *>(a.ids) + at * a.k * (a.wide_index ? 8 : 4);
  s.teacher = a.teacher + at * a.k;
  if (a.weights) s.weights = a.weights + at;
  if (a.loss) s.loss = a.loss + at;
  if (a.stats) s.stats = a.stats + at * 4;
  if (a.d_logits) s.d_logits = static_cast<T *>(a.d_logits) + at * a.d_row_stride;
  return s;
}

template <class T>
int run_distill(tmnn_logits *h, DistillArgs a, int64_t rows, bool back, hipStream_t st) {
  constexpr int n = Row<T>::n;
  const bool tail = a.kind == TMNN_TEACHER_LOGPROBS;
  if (const int g = group_lanes(a.classes)) {
    return in_slices(rows, g, 1, [&](int64_t at, int32_t r) {
      const DistillArgs s = distill_slice<T>(a, at, r);
#define LAUNCH(G, NV, TAIL, BACK)                                                            \
  hipLaunchKernelGGL((distill_group_kernel<T, G, NV, TAIL, BACK>), group_grid(r, G),         \
                     dim3(kGroupThreads), 0, st, s)
#define CALL(G, NV)                                                                          \
  if (tail && back) LAUNCH(G, NV, true, true);                                               \
  else if (tail) LAUNCH(G, NV, true, false);                                                 \
  else if (back) LAUNCH(G, NV, false, true);                                                 \
  else LAUNCH(G, NV, false, false)
      TMNN_BY_GROUP(g, CALL)
#undef CALL
#undef LAUNCH
    });
  }
  const Split sp = split_of(rows, a.classes, n, back ? map_threads : a.d_logits ? both_threads : sum_threads,
                            a.k, kSplitBlocks, !back);
  a.parts = sp.parts;
  a.part_len = sp.part_len;
  if (back)
    return in_slices(rows, static_cast<int64_t>(sp.threads) * a.parts, 1,
                     [&](int64_t at, int32_t r) {
                       const DistillArgs s = distill_slice<T>(a, at, r);
#define CALL(NT)                                                                                    \
  if (tail)                                                                                         \
    hipLaunchKernelGGL((distill_grad_block_kernel<T, NT, true>), dim3(r * a.parts), dim3(NT), 0, st, \
                       s);                                                                          \
  else                                                                                              \
    hipLaunchKernelGGL((distill_grad_block_kernel<T, NT, false>), dim3(r * a.parts), dim3(NT), 0,   \
                       st, s)
                       TMNN_BY_THREADS(sp.threads, CALL)
#undef CALL
                     });
  const bool keep = a.parts == 1 && a.d_logits && sp.threads <= 256 &&
                    a.classes <= static_cast<int64_t>(sp.threads) * n * kKeptVecs;
  a.part_sum = static_cast<float2 *>(h->work.ptr);
  a.list_z = reinterpret_cast<float *>(static_cast<char *>(h->work.ptr) + kSumBytes + kKeyBytes);
  const int64_t threads = static_cast<int64_t>(sp.threads) * a.parts;
  return with_workspace(h, st, a.parts, [&] {
    return in_slices(rows, threads, a.parts, [&](int64_t at, int32_t r) {
      const DistillArgs s = distill_slice<T>(a, at, r);
      const size_t bits = (static_cast<size_t>(sp.part_len) + 31) / 32 * 4;
#define LAUNCH(NT, TAIL, KEEP)                                                               \
  hipLaunchKernelGGL((distill_block_kernel<T, NT, TAIL, KEEP>), dim3(r * a.parts), dim3(NT), \
      TAIL ? bits : 0, st, s)
#define CALL(NT)                                                  \
  if (tail && keep) LAUNCH(NT, true, (NT <= 256 ? kKeptVecs : 0)); \
  else if (tail) LAUNCH(NT, true, 0);                              \
  else if (keep) LAUNCH(NT, false, (NT <= 256 ? kKeptVecs : 0));   \
  else LAUNCH(NT, false, 0)
      TMNN_BY_THREADS(sp.threads, CALL)
#undef CALL
#undef LAUNCH
      if (a.parts > 1) {
        const dim3 grid(r * (a.d_logits ? a.parts : 1));
#define CALL(NT)                                                                            \
  if (tail)                                                                                 \
    hipLaunchKernelGGL((distill_join_kernel<T, NT, true>), grid, dim3(NT), 0, st, s);       \
  else                                                                                      \
    hipLaunchKernelGGL((distill_join_kernel<T, NT, false>), grid, dim3(NT), 0, st, s)
        TMNN_BY_THREADS(sp.threads, CALL)
#undef CALL
      }
    });
  });
}

// ---- calls on device memory -----------------------------------------------------------

int logprobs_device(tmnn_logits *h, const tmnn_token_logprobs_args &u, bool back, hipStream_t st) {
  LogprobArgs a{};
  a.logits = u.logits;
  a.row_stride = u.row_stride;
  a.tokens = u.tokens;
  a.wide_index = u.index_dtype == TMNN_INDEX_I64;
  a.classes = static_cast<int32_t>(u.classes);
  a.top_k = u.top_k;
  a.parts = 1;
  a.inv_t = static_cast<float>(1.0 / u.temperature);
  a.c = static_cast<float>(1.4426950408889634 / u.temperature);
  if (back) {
    a.d_logprob = u.d_logprob;
    a.d_entropy = u.d_entropy;
    a.d_top = u.top_k > 0 ? u.d_top_logprobs : nullptr;
    a.entropy_in = u.entropy;
    a.stats_in = u.stats;
    a.top_in = u.top_ids;
    a.d_logits = u.d_logits;
    a.d_row_stride = u.d_row_stride;
  } else {
    a.logprob = u.logprob;
    a.entropy = u.entropy;
    a.rank = u.rank;
    a.stats = u.stats;
    a.top_ids = u.top_ids;
    a.top_logprobs = u.top_logprobs;
  }
  std::lock_guard<std::mutex> lock(h->mu);
  switch (u.dtype) {
    case TMNN_DTYPE_F32:
      return back ? run_logprobs_grad<float>(h, a, u.rows, st) : run_logprobs<float>(h, a, u.rows, st);
    case TMNN_DTYPE_F16:
      return back ? run_logprobs_grad<_Float16>(h, a, u.rows, st)
                  : run_logprobs<_Float16>(h, a, u.rows, st);
    default:
      return back ? run_logprobs_grad<__bf16>(h, a, u.rows, st) : run_logprobs<__bf16>(h, a, u.rows, st);
  }
}

int distill_device(tmnn_logits *h, const tmnn_distill_args &u, bool back, hipStream_t st) {
  DistillArgs a{};
  a.logits = u.logits;
  a.row_stride = u.row_stride;
  a.ids = u.teacher_ids;
  a.teacher = u.teacher;
  a.weights = u.row_weights;
  a.wide_index = u.index_dtype == TMNN_INDEX_I64;
  a.kind = u.teacher_kind;
  a.classes = static_cast<int32_t>(u.classes);
  a.k = u.teacher_k;
  a.parts = 1;
  a.t = u.temperature;
  a.inv_t64 = 1.0 / static_cast<double>(u.temperature);
  a.inv_t = static_cast<float>(a.inv_t64);
  a.c = static_cast<float>(1.4426950408889634 / u.temperature);
  a.loss = back ? nullptr : u.loss;
  a.stats = u.stats;
  a.d_logits = u.d_logits;
  a.d_row_stride = u.d_row_stride;
  std::lock_guard<std::mutex> lock(h->mu);
  switch (u.dtype) {
    case TMNN_DTYPE_F32:
      return run_distill<float>(h, a, u.rows, back, st);
    case TMNN_DTYPE_F16:
      return run_distill<_Float16>(h, a, u.rows, back, st);
    default:
      return run_distill<__bf16>(h, a, u.rows, back, st);
  }
}

hipStream_t stream_of(tmnn_logits *h, void *stream) {
  return stream == TMNN_STREAM_CONTEXT ? h->ctx->stream : static_cast<hipStream_t>(stream);
}

// ---- calls on host memory ---------------------------------------------------------------

// The host arrays of a call and their places in the handle's arena.
class HostArrays {
 public:
  enum Dir { kIn, kOut };
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

int logprobs_host(tmnn_logits *h, tmnn_token_logprobs_args u, bool back) {
  const size_t size = dtype_size(u.dtype), index = u.index_dtype == TMNN_INDEX_I64 ? 8 : 4;
  const size_t k = static_cast<size_t>(u.top_k);
  const auto out = back ? HostArrays::kIn : HostArrays::kOut;
  HostArrays m;
  m.add(u.logits, HostArrays::kIn, u.rows, u.classes * size, u.row_stride * size);
  m.add(u.tokens, HostArrays::kIn, u.rows, index);
  m.add(u.entropy, out, u.rows, 4);
  m.add(u.stats, out, u.rows, 8);
  m.add(u.top_ids, out, u.rows, 4 * k);
  if (back) {
    m.add(u.d_logprob, HostArrays::kIn, u.rows, 4);
    m.add(u.d_entropy, HostArrays::kIn, u.rows, 4);
    m.add(u.d_top_logprobs, HostArrays::kIn, u.rows, 4 * k);
    m.add(u.d_logits, HostArrays::kOut, u.rows, u.classes * size, u.d_row_stride * size);
  } else {
    m.add(u.logprob, HostArrays::kOut, u.rows, 4);
    m.add(u.rank, HostArrays::kOut, u.rows, 4);
    m.add(u.top_logprobs, HostArrays::kOut, u.rows, 4 * k);
    u.d_logits = nullptr;
  }
  u.row_stride = u.d_row_stride = u.classes;
  return on_host(h, m, [&] { return logprobs_device(h, u, back, h->ctx->stream); });
}

int distill_host(tmnn_logits *h, tmnn_distill_args u, bool back) {
  const size_t size = dtype_size(u.dtype), index = u.index_dtype == TMNN_INDEX_I64 ? 8 : 4;
  const size_t k = static_cast<size_t>(u.teacher_k);
  HostArrays m;
  m.add(u.logits, HostArrays::kIn, u.rows, u.classes * size, u.row_stride * size);
  m.add(u.teacher_ids, HostArrays::kIn, u.rows, index * k);
  m.add(u.teacher, HostArrays::kIn, u.rows, 4 * k);
  m.add(u.row_weights, HostArrays::kIn, u.rows, 4);
  m.add(u.stats, back ? HostArrays::kIn : HostArrays::kOut, u.rows, 16);
  if (back)
    u.loss = nullptr;
  else
    m.add(u.loss, HostArrays::kOut, u.rows, 4);
  m.add(u.d_logits, HostArrays::kOut, u.rows, u.classes * size, u.d_row_stride * size);
  u.row_stride = u.d_row_stride = u.classes;
  return on_host(h, m, [&] { return distill_device(h, u, back, h->ctx->stream); });
}

// No exception leaves a C entry point.
template <class F>
int entry(tmnn_logits *h, F f) {
  if (!h) return fail(TMNN_ERR_INVALID_ARGUMENT, "logits handle is null");
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return fail(TMNN_ERR_RUNTIME, "out of host memory");
  } catch (const std::exception &e) {
    return fail(TMNN_ERR_RUNTIME, e.what());
  }
}

int token_logprobs(tmnn_logits *h, const tmnn_token_logprobs_args *args, bool back, bool host,
                   void *stream) {
  return entry(h, [&] {
    const int rc = check_logprobs(args, back, host);
    if (rc != TMNN_OK || args->rows == 0) return rc;
    TMNN_HIP_TRY(hipSetDevice(h->ctx->device));
    return host ? logprobs_host(h, *args, back)
                : logprobs_device(h, *args, back, stream_of(h, stream));
  });
}

int distill(tmnn_logits *h, const tmnn_distill_args *args, bool back, bool host, void *stream) {
  return entry(h, [&] {
    const int rc = check_distill(args, back, host);
    if (rc != TMNN_OK || args->rows == 0) return rc;
    TMNN_HIP_TRY(hipSetDevice(h->ctx->device));
    return host ? distill_host(h, *args, back) : distill_device(h, *args, back, stream_of(h, stream));
  });
}

}  // namespace

extern "C" {

int tmnn_logits_create(tmnn_context *ctx, tmnn_logits **out) {
  if (!out) return fail(TMNN_ERR_INVALID_ARGUMENT, "out is null");
  *out = nullptr;
  if (!ctx) return fail(TMNN_ERR_INVALID_ARGUMENT, "context is null");
  TMNN_HIP_TRY(hipSetDevice(ctx->device));
  std::unique_ptr<tmnn_logits> h(new (std::nothrow) tmnn_logits());
  if (!h) return fail(TMNN_ERR_RUNTIME, "out of host memory");
  h->ctx = ctx;
  TMNN_HIP_TRY(h->work.ensure(kSumBytes + kKeyBytes + kListBytes));
  // orders kernels of one device; the host reads nothing after it
  TMNN_HIP_TRY(hipEventCreateWithFlags(&h->done, hipEventDisableTiming | hipEventDisableSystemFence));
  *out = h.release();
  return TMNN_OK;
}

int tmnn_logits_destroy(tmnn_logits *h) {
  if (!h) return TMNN_OK;
  (void)hipSetDevice(h->ctx->device);
  if (h->recorded && hipEventSynchronize(h->done) != hipSuccess) (void)hipGetLastError();
  if (h->done) (void)hipEventDestroy(h->done);
  delete h;
  return TMNN_OK;
}

int tmnn_token_logprobs(tmnn_logits *h, const tmnn_token_logprobs_args *args) {
  return token_logprobs(h, args, false, true, nullptr);
}
int tmnn_token_logprobs_device(tmnn_logits *h, const tmnn_token_logprobs_args *args, void *stream) {
  return token_logprobs(h, args, false, false, stream);
}
int tmnn_token_logprobs_backward(tmnn_logits *h, const tmnn_token_logprobs_args *args) {
  return token_logprobs(h, args, true, true, nullptr);
}
int tmnn_token_logprobs_backward_device(tmnn_logits *h, const tmnn_token_logprobs_args *args,
                                        void *stream) {
  return token_logprobs(h, args, true, false, stream);
}
int tmnn_distill(tmnn_logits *h, const tmnn_distill_args *args) {
  return distill(h, args, false, true, nullptr);
}
int tmnn_distill_device(tmnn_logits *h, const tmnn_distill_args *args, void *stream) {
  return distill(h, args, false, false, stream);
}
int tmnn_distill_backward(tmnn_logits *h, const tmnn_distill_args *args) {
  return distill(h, args, true, true, nullptr);
}
int tmnn_distill_backward_device(tmnn_logits *h, const tmnn_distill_args *args, void *stream) {
  return distill(h, args, true, false, stream);
}

}  // extern "C"
