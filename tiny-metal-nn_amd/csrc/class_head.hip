// class_head.hip -- host side of the class head (include/tmnn_hip.h): argument
// checks, launches by the plan (head_plan.hpp), and the host-pointer forms.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <memory>
#include <string>

#include "class_loss_kernel.hpp"
#include "f8_kernel.hpp"
#include "head_plan.hpp"
#include "logits_host.hpp"
#include "narrow_kernel.hpp"
#include "tmnn_hip.h"

using namespace tmnn_hip;

namespace {

// ---- tiles --------------------------------------------------------------------------

// waves, blocks of a wave, stages
template <class E, bool XT, bool YT>
using Large = TileShape<E, 2, 4, 8, 4, 2, XT, YT>;  // 256 classes x 256 rows
template <class E, bool XT, bool YT>
using Wide = TileShape<E, 4, 2, 4, 4, 3, XT, YT>;  // 256 x 128
template <class E, bool XT, bool YT>
using Middle = TileShape<E, 2, 2, 4, 4, 2, XT, YT>;  // 128 x 128
template <class E, bool XT, bool YT>
using Flat = TileShape<E, 4, 1, 2, 4, 3, XT, YT>;  // 128 x 64
template <class E, bool XT, bool YT>
using Small = TileShape<E, 4, 1, 2, 2, 4, XT, YT>;  // 128 x 32
template <class S>
constexpr bool planned(int bc, int br) {  // as `choose` takes it
  return S::BC == bc && S::BR == br;
}
static_assert(planned<Large<F16, false, false>>(256, 256) && planned<Wide<F16, false, false>>(256, 128) &&
                  planned<Middle<F16, false, false>>(128, 128) && planned<Flat<F16, false, false>>(128, 64) &&
                  planned<Small<F16, false, false>>(128, 32),
              "");

template <class S, class Steps, class Epi, class StepArgs>
struct TileLaunch {
  static int run(const TileArgs &a, const StepArgs &sa, const Epi &epi, int device, hipStream_t st) {
    // more LDS than a kernel gets unasked, asked for once a device
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << (device & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
      TMNN_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(tile_kernel<S, Steps, Epi, StepArgs>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds));
      done.fetch_or(bit, std::memory_order_relaxed);
    }
    const int64_t blocks = static_cast<int64_t>(a.tiles_r) * a.tiles_c * a.parts;
    hipLaunchKernelGGL((tile_kernel<S, Steps, Epi, StepArgs>), dim3(static_cast<uint32_t>(blocks)),
                       dim3(S::kThreads), S::kLds, st, a, sa, epi);
    TMNN_HIP_TRY(hipGetLastError());
    return TMNN_OK;
  }
};

struct NoArgs {
  int32_t unused;
};

template <class S, class Epi>
int run_plain(const TileArgs &a, const Epi &epi, int device, hipStream_t st) {
  return TileLaunch<S, PlainSteps<S>, Epi, NoArgs>::run(a, NoArgs{}, epi, device, st);
}

// Both operands' k contiguous.
template <class E, class Epi>
int run_rows(const TileArgs &a, Shape s, const Epi &epi, int device, hipStream_t st) {
  switch (s) {
    case kLarge: return run_plain<Large<E, false, false>>(a, epi, device, st);
    case kWide: return run_plain<Wide<E, false, false>>(a, epi, device, st);
    case kMiddle: return run_plain<Middle<E, false, false>>(a, epi, device, st);
    case kFlat: return run_plain<Flat<E, false, false>>(a, epi, device, st);
    default: return run_plain<Small<E, false, false>>(a, epi, device, st);
  }
}

// The gradients' products: d and the table, or both transposed.
template <bool XT, class Epi>
int run_grad(const TileArgs &a, Shape s, const Epi &epi, int device, hipStream_t st) {
  switch (s) {
    case kLarge: return run_plain<Large<F16, XT, true>>(a, epi, device, st);
    case kWide: return run_plain<Wide<F16, XT, true>>(a, epi, device, st);
    default: return run_plain<Middle<F16, XT, true>>(a, epi, device, st);
  }
}

// ---- arguments ------------------------------------------------------------------------

struct Extent {  // rows of `width` bytes, `stride` bytes apart
  const void *p;
  int64_t rows, width, stride;
  const char *name;
};

bool meet(const Extent &a, const Extent &b) {
  typedef __int128 wide;
  if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  const wide pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  const wide ea = pa + static_cast<wide>(a.rows - 1) * a.stride + a.width;
  const wide eb = pb + static_cast<wide>(b.rows - 1) * b.stride + b.width;
  if (pa >= eb || pb >= ea) return false;
  if (a.rows > 1 && b.rows > 1 && a.stride == b.stride) {  // rows between each other's
    wide off = (pb - pa) % a.stride;
    if (off < 0) off += a.stride;
    if (off >= a.width && off + b.width <= a.stride) return false;
  }
  return true;
}

// Each of `out` against `in` and the others of `out`.
int apart(const char *what, std::initializer_list<Extent> out, std::initializer_list<Extent> in) {
  for (const Extent &o : out) {
    for (const Extent &i : in)
      if (meet(o, i))
        return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + o.name + " overlaps " + i.name);
    for (const Extent &p : out)
      if (&p < &o && meet(o, p))
        return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + o.name + " overlaps " + p.name);
  }
  return TMNN_OK;
}

int check_sizes(const char *what, int64_t rows, int64_t classes, int64_t dims) {
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (rows < 0 || rows > TMNN_HEAD_MAX_ROWS) return bad("rows must be in [0, 2^24]");
  if (classes < 1 || classes > TMNN_LOGITS_MAX_CLASSES) return bad("classes must be in [1, 2^24]");
  if (dims < 1 || dims > TMNN_HEAD_MAX_DIMS) return bad("dims must be in [1, 2^16]");
  // (the threads of a launch are counted in 32 bits)
  if (rows * classes > int64_t{1} << 38) return bad("rows x classes must be at most 2^38");
  return TMNN_OK;
}

constexpr int64_t kMostStride = int64_t{1} << 40;  // elements: addresses stay 64-bit numbers

int check_loss(const tmnn_class_loss_args *a, bool back) {
  const char *what = back ? "class_loss_backward" : "class_loss";
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (!a) return bad("args is null");
  if (a->struct_size != sizeof(*a)) return bad("struct_size mismatch");
  if (a->dtype < TMNN_DTYPE_F32 || a->dtype > TMNN_DTYPE_BF16) return bad("invalid dtype");
  if (a->index_dtype != TMNN_INDEX_I32 && a->index_dtype != TMNN_INDEX_I64) return bad("invalid index_dtype");
  const int rc = check_sizes(what, a->rows, a->classes, a->dims);
  if (rc != TMNN_OK) return rc;
  // c = log2(e) / T stays an ordinary number
  if (!(a->temperature >= 1e-6f && a->temperature <= 1e6f)) return bad("temperature must be in [1e-6, 1e6]");
  if (a->feature_stride < a->dims || a->feature_stride > kMostStride || a->table_stride < a->dims ||
      a->table_stride > kMostStride)
    return bad("strides must be at least dims");
  if (a->d_features && (a->d_feature_stride < a->dims || a->d_feature_stride > kMostStride))
    return bad("d_feature_stride must be at least dims");
  if (a->d_table && (a->d_table_stride < a->dims || a->d_table_stride > kMostStride))
    return bad("d_table_stride must be at least dims");
  return TMNN_OK;
}

int check_loss_arrays(const tmnn_class_loss_args *a, bool back, bool host) {
  const char *what = back ? "class_loss_backward" : "class_loss";
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  const int64_t size = static_cast<int64_t>(dtype_size(a->dtype));
  if (a->rows > 0 && !a->d_features && !a->d_table && (back || (!a->loss && !a->stats)))
    return bad("nothing to compute");
  if (!a->table) return bad("table is null");
  if (a->rows > 0) {
    if (!a->features) return bad("features is null");
    if (!a->labels) return bad("labels is null");
    if (back && !a->stats) return bad("stats is null");
    if (back && !a->row_weights) return bad("row_weights (the loss's gradient) is null");
  }
  for (const void *p : {a->features, a->table, static_cast<const void *>(a->d_features),
                        static_cast<const void *>(a->d_table)})
    if (!aligned(p, size)) return bad("features, table and gradients must be aligned to their type");
  if (!aligned(a->labels, a->index_dtype == TMNN_INDEX_I64 ? 8 : 4))
    return bad("labels must be aligned to their type");
  if (!aligned(a->row_weights, 4) || !aligned(a->loss, 4)) return bad("arrays of 32-bit values must be 4-byte aligned");
  if (!host && !aligned(a->stats, 16)) return bad("stats must be 16-byte aligned");
  if (host && !aligned(a->stats, 4)) return bad("arrays of 32-bit values must be 4-byte aligned");
  const int64_t n = a->rows, w = a->dims * size;
  const Extent x{a->features, n, w, a->feature_stride * size, "features"};
  const Extent y{a->table, a->classes, w, a->table_stride * size, "the table"};
  const int64_t index = a->index_dtype == TMNN_INDEX_I64 ? 8 : 4;
  const Extent l{a->labels, 1, n * index, 0, "labels"}, rw{a->row_weights, 1, n * 4, 0, "row_weights"};
  const Extent s{a->stats, 1, n * 16, 0, "stats"}, lo{back ? nullptr : a->loss, 1, n * 4, 0, "loss"};
  const Extent dx{a->d_features, n, w, a->d_feature_stride * size, "d_features"};
  const Extent dy{a->d_table, a->classes, w, a->d_table_stride * size, "d_table"};
  const Extent ws{host ? nullptr : a->workspace, 1, a->workspace_bytes, 0, "the workspace"};
  if (back) return apart(what, {dx, dy, ws}, {x, y, l, rw, s});
  return apart(what, {lo, s, dx, dy, ws}, {x, y, l, rw});
}

// ---- class loss ---------------------------------------------------------------------------

template <class T>
int run_reduce(const GradScale &s, void *out, int64_t ld, const float *slabs, int64_t slab_ld, int32_t parts, int64_t rows,
               int64_t cols, hipStream_t st) {
  ReduceArgs r{s, out, ld, slabs, static_cast<int32_t>(slab_ld), parts, static_cast<int32_t>(rows),
               static_cast<int32_t>(cols), 1};
  // (four parts a thread at least, and threads enough for two blocks a unit)
  while (r.lanes < 16 && r.lanes * 4 < parts && parts_of(rows * slab_ld / 4, 256 / r.lanes) < 2 * kUnits) r.lanes *= 2;
  const int64_t blocks = std::min<int64_t>(parts_of(rows * slab_ld / 4, 256 / r.lanes), 8 * kUnits);
  hipLaunchKernelGGL((class_reduce_kernel<T>), dim3(static_cast<uint32_t>(std::max<int64_t>(blocks, 1))), dim3(256), 0, st,
                     r);
  TMNN_HIP_TRY(hipGetLastError());
  return TMNN_OK;
}

template <int DP, int PL, int PD, int RJ, class Op>
int run_walk(const WalkArgs &a, int32_t parts, const Op &op, int device, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (device & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    TMNN_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(walk_kernel<DP, PL, PD, RJ, Op>),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, WalkTile<DP, PL>::kLds));
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL((walk_kernel<DP, PL, PD, RJ, Op>), dim3(static_cast<uint32_t>(static_cast<int64_t>(a.blocks) * parts)),
                     dim3(kWalkThreads), (WalkTile<DP, PL>::kLds), st, a, op);
  TMNN_HIP_TRY(hipGetLastError());
  return TMNN_OK;
}

// Features of up to 128 dims, both sides laid out.
template <class T, int DP>
int run_narrow(tmnn_logits *h, const tmnn_class_loss_args &a, const LossPlan &p, const RowInfo &row, float c, float inv_t,
               const Exponents *exps, hipStream_t st) {
  constexpr int PL = sizeof(T) == 4 ? 2 : 1, PD = __is_same(T, __bf16) ? 1 : 2;
  const int device = h->ctx->device;
  char *ws = static_cast<char *>(a.workspace);
  const int32_t n = static_cast<int32_t>(a.rows), v = static_cast<int32_t>(a.classes), dims = static_cast<int32_t>(a.dims);
  const int64_t x_plane = a.rows * DP * 2, y_plane = a.classes * DP * 2;
  float4 *stats = reinterpret_cast<float4 *>(a.stats ? reinterpret_cast<char *>(a.stats) : ws + p.at_stats);
  if (p.sums || a.d_features) {
    RowsShared g{};
    g.exps = exps;
    g.row = row;
    g.c = c;
    g.inv_t = inv_t;
    g.loss = p.sums ? a.loss : nullptr;
    g.stats = p.sums && (a.stats || a.d_table) ? stats : nullptr;
    if (p.parts_r > 1) {
      g.part_sum = reinterpret_cast<float2 *>(ws + p.at_part_sum);
      g.own = reinterpret_cast<float *>(ws + p.at_part_own);
      g.part_out = reinterpret_cast<float *>(ws + p.at_part_out);
    }
    const T *table = static_cast<const T *>(a.table);
    T *out = static_cast<T *>(a.d_features);
    const WalkArgs w{ws + p.at_x, ws + p.at_y, x_plane, y_plane, n, v, p.blocks_r,
                     static_cast<int32_t>(parts_of(p.tiles_r, p.parts_r))};
    auto walk = [&](auto op) {
      static_cast<RowsShared &>(op) = g;
      op.table = table;
      op.table_ld = a.table_stride;
      op.out = out;
      op.out_ld = a.d_feature_stride;
      op.dims = dims;
      return run_walk<DP, PL, PD, 1>(w, p.parts_r, op, device, st);
    };
    const int rc = out ? walk(RowsWalk<T, true>{}) : walk(RowsWalk<T, false>{});
    if (rc != TMNN_OK) return rc;
    if (p.parts_r > 1) {
      const dim3 groups(static_cast<uint32_t>(parts_of(n, 256 / (DP / 4))));
      if (p.parts_r <= kFewParts)
        hipLaunchKernelGGL((walk_join_few_kernel<T, DP>), groups, dim3(256), 0, st, g, n, p.parts_r, table,
                           a.table_stride, out, a.d_feature_stride, dims);
      else
        hipLaunchKernelGGL((walk_join_kernel<T, DP>), dim3(static_cast<uint32_t>(n)), dim3(256), 0, st, g, n, p.parts_r,
                           table, a.table_stride, out, a.d_feature_stride, dims);
      TMNN_HIP_TRY(hipGetLastError());
    }
  }
  if (!a.d_table) return TMNN_OK;
  float *slabs = p.slabs_y ? reinterpret_cast<float *>(ws + p.at_slab_y) : nullptr;
  const GradScale scale{exps, row, inv_t, 0};
  const WalkArgs w{ws + p.at_y, ws + p.at_w, y_plane, x_plane, v, n, p.blocks_t,
                   static_cast<int32_t>(parts_of(p.tiles_t, p.parts_t))};
  auto walk = [&](auto rj) {
    constexpr int RJ = decltype(rj)::value;
    TableWalk<T, RJ> t{};
    t.exps = exps;
    t.row = row;
    t.c = c;
    t.stats = stats;
    t.scale = scale;
    t.out = static_cast<T *>(a.d_table);
    t.out_ld = a.d_table_stride;
    t.dims = dims;
    t.slabs = slabs;
    t.slab_ld = static_cast<int32_t>(p.slab_ld);
    return run_walk<DP, PL, PD, RJ>(w, p.parts_t, t, device, st);
  };
  const int rc = p.wide_t ? walk(std::integral_constant<int, 2>{}) : walk(std::integral_constant<int, 1>{});
  if (rc != TMNN_OK || !slabs) return rc;
  return run_reduce<T>(scale, a.d_table, a.d_table_stride, slabs, p.slab_ld, p.parts_t, v, dims, st);
}

int run_terms(const LossPlan &p, const RowInfo &row, float c, const float4 *stats, int64_t n, int64_t v, char *ws, _Float16 *d,
              int64_t plane, hipStream_t st) {
  TermsArgs t{row, c, stats, reinterpret_cast<const float *>(ws + p.at_z), static_cast<int32_t>(n), static_cast<int32_t>(v),
              static_cast<int32_t>(p.k_d / 8), 1, 1, p.k_d, p.ld_d, p.planes_d, plane, d};
  while (t.lanes < 256 && t.lanes < t.chunks) t.lanes *= 2;
  const int64_t groups = parts_of(n, 256 / t.lanes);
  // (two vectors a thread at least, and blocks for eight a unit)
  t.splits = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(parts_of(8 * kUnits, groups), t.chunks / (2 * t.lanes))));
  hipLaunchKernelGGL(class_terms_kernel, dim3(static_cast<uint32_t>(groups * t.splits)), dim3(256), 0, st, t);
  TMNN_HIP_TRY(hipGetLastError());
  return TMNN_OK;
}

template <class T>
int run_loss(tmnn_logits *h, const tmnn_class_loss_args &a, const LossPlan &p, bool back, hipStream_t st) {
  const int device = h->ctx->device;
  const int64_t n = a.rows, v = a.classes, size = sizeof(T);
  char *ws = static_cast<char *>(a.workspace);
  RowInfo row{a.labels, a.row_weights, a.index_dtype == TMNN_INDEX_I64, static_cast<int32_t>(v)};
  const float c = static_cast<float>(1.4426950408889634 / a.temperature);
  const float inv_t = static_cast<float>(1.0 / a.temperature);
  const Exponents *exps = nullptr;

  if (p.lay_x || p.lay_y || p.weighted) {
    LayArgs l{};
    const bool keep = !p.f32 && a.dtype == TMNN_DTYPE_F16;  // fp16 products take fp16 operands as they are
    const int planes = p.planes;
    auto blocks = [&](int64_t rows) {
      int lanes = 1;
      while (lanes < 256 && lanes < p.ld / 8) lanes *= 2;
      return static_cast<int32_t>(std::min<int64_t>(parts_of(std::max<int64_t>(rows, 1), 256 / lanes), 2048));
    };
    // (16 rows of a wave's vectors a block: four loads each on their way, four times)
    auto scale_parts = [&](int64_t rows) {
      return static_cast<int32_t>(std::min<int64_t>(parts_of(rows * parts_of(a.dims, 8), 16 * 256), kScaleParts));
    };
    const int32_t dims = static_cast<int32_t>(a.dims), ld = static_cast<int32_t>(p.ld);
    l.part[0] = {a.features, a.feature_stride, static_cast<int32_t>(n), dims, p.lay_x ? ws + p.at_x : nullptr,
                 p.weighted ? ws + p.at_w : nullptr, ld, !keep, planes,
                 p.lay_x || p.weighted ? blocks(n) : 0, !keep || (p.weighted && !p.narrow) ? scale_parts(n) : 0};
    l.part[1] = {a.table, a.table_stride, static_cast<int32_t>(v), dims, p.lay_y ? ws + p.at_y : nullptr, nullptr,
                 ld, !keep, planes, p.lay_y ? blocks(v) : 0, !keep ? scale_parts(v) : 0};
    l.row = row;
    l.most = reinterpret_cast<uint32_t *>(ws + p.at_most);
    l.most_w = reinterpret_cast<int32_t *>(ws + p.at_most) + 2 * kScaleParts;
    l.by_weight = !p.narrow;
    l.parts_w = static_cast<int32_t>(std::min<int64_t>(parts_of(n, 256), kScaleParts));
    l.exps = reinterpret_cast<Exponents *>(ws + p.at_exps);
    if (p.scaled) exps = l.exps;
    const dim3 grid(l.part[0].blocks + l.part[1].blocks);
    if (p.scaled) {
      hipLaunchKernelGGL((class_scale_kernel<T>), dim3(l.part[0].parts + l.part[1].parts + l.parts_w), dim3(256), 0, st, l);
      hipLaunchKernelGGL((class_lay_kernel<T, true>), grid, dim3(256), 0, st, l);
    } else {
      hipLaunchKernelGGL((class_lay_kernel<T, false>), grid, dim3(256), 0, st, l);
    }
    TMNN_HIP_TRY(hipGetLastError());
  }

  if (p.narrow) {
    switch (p.ld) {
      case 32: return run_narrow<T, 32>(h, a, p, row, c, inv_t, exps, st);
      case 64: return run_narrow<T, 64>(h, a, p, row, c, inv_t, exps, st);
      default: return run_narrow<T, 128>(h, a, p, row, c, inv_t, exps, st);
    }
  }
  const LossOperands o = loss_operands(a, p);
  float4 *stats = reinterpret_cast<float4 *>(a.stats ? reinterpret_cast<char *>(a.stats) : ws + p.at_stats);

  if (p.sums) {
    SumsEpilogue e{exps, row, c, reinterpret_cast<float2 *>(ws + p.at_sums),
                   reinterpret_cast<float *>(ws + p.at_own), p.keep ? reinterpret_cast<float *>(ws + p.at_z) : nullptr, p.k_d};
    const TileArgs t = sums_product(a, p, o);
    int rc;
    if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16))
      rc = p.scaled ? run_rows<F16>(t, p.t_sums.shape, e, device, st) : run_rows<BF16>(t, p.t_sums.shape, e, device, st);
    else
      rc = run_rows<F16>(t, p.t_sums.shape, e, device, st);
    if (rc != TMNN_OK) return rc;
    JoinArgs j{row, e.sums, e.own, static_cast<int32_t>(n), p.t_sums.c, 1, c, inv_t, a.loss,
               a.stats || p.grad ? stats : nullptr};
    while (j.lanes < 64 && j.lanes * 4 < j.tiles) j.lanes *= 2;
    hipLaunchKernelGGL(class_join_kernel, dim3(static_cast<uint32_t>(parts_of(n, 256 / j.lanes))), dim3(256), 0, st, j);
    TMNN_HIP_TRY(hipGetLastError());
  }
  if (!p.grad) return TMNN_OK;

  auto *d = reinterpret_cast<_Float16 *>(ws + p.at_d);
  const int64_t d_plane = n * p.ld_d;
  const GradScale by_row{exps, row, inv_t, 1}, by_all{exps, row, inv_t, 0};
  for (int64_t first = 0; first < v; first += p.piece) {
    const LossPiece q = piece_of(p, v, first);
    int rc;
    if (p.keep) {
      rc = run_terms(p, row, c, stats, n, v, ws, d, d_plane, st);
    } else {
      GradEpilogue g{exps, row, c, stats, static_cast<int32_t>(first), static_cast<int32_t>(q.width), p.ld_d, p.planes_d, d_plane, d};
      rc = run_rows<F16>(d_product(a, p, o, q), q.d.shape, g, device, st);
    }
    if (rc != TMNN_OK) return rc;
    if (a.d_features) {
      GradOut<T> out{by_row, static_cast<T *>(a.d_features), a.d_feature_stride,
                     p.slabs_x ? reinterpret_cast<float *>(ws + p.at_slab_x) : nullptr, static_cast<int32_t>(p.slab_ld),
                     first > 0};
      rc = run_grad<false>(features_product(a, p, o, q), q.x.shape, out, device, st);
      if (rc != TMNN_OK) return rc;
    }
    if (a.d_table) {
      T *to = static_cast<T *>(a.d_table) + first * a.d_table_stride;
      GradOut<T> out{by_all, to, a.d_table_stride, p.slabs_y ? reinterpret_cast<float *>(ws + p.at_slab_y) : nullptr,
                     static_cast<int32_t>(p.slab_ld), 0};
      rc = run_grad<true>(table_product(a, p, o, q), q.y.shape, out, device, st);
      if (rc != TMNN_OK) return rc;
      if (p.slabs_y) {
        rc = run_reduce<T>(by_all, to, a.d_table_stride, out.slabs, p.slab_ld, q.y.parts, q.count, a.dims, st);
        if (rc != TMNN_OK) return rc;
      }
    }
  }
  if (a.d_features && p.slabs_x)
    return run_reduce<T>(by_row, a.d_features, a.d_feature_stride, reinterpret_cast<float *>(ws + p.at_slab_x), p.slab_ld,
                         p.t_x.parts, n, a.dims, st);
  return TMNN_OK;
}

// Without rows the table's gradient is 0.
__global__ __launch_bounds__(256) void class_zero_kernel(char *out, int64_t stride, int64_t rows, int64_t width) {
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < rows * width;
       at += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = at / width;
    reinterpret_cast<int16_t *>(out + r * stride)[at - r * width] = 0;
  }
}

int loss_device(tmnn_logits *h, const tmnn_class_loss_args &a, bool back, hipStream_t st) {
  if (a.rows == 0) {
    if (!a.d_table) return TMNN_OK;
    const int64_t size = static_cast<int64_t>(dtype_size(a.dtype));
    hipLaunchKernelGGL(class_zero_kernel, dim3(1024), dim3(256), 0, st, static_cast<char *>(a.d_table),
                       a.d_table_stride * size, a.classes, a.dims * size / 2);
    TMNN_HIP_TRY(hipGetLastError());
    return TMNN_OK;
  }
  const LossPlan p = plan_loss(a, back);
  const char *what = back ? "class_loss_backward" : "class_loss";
  if (!a.workspace || !aligned(a.workspace, 256) || a.workspace_bytes < p.bytes)
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": the workspace must be 256-byte aligned and hold " +
                                               std::to_string(p.bytes) + " bytes");
  switch (a.dtype) {
    case TMNN_DTYPE_F32: return run_loss<float>(h, a, p, back, st);
    case TMNN_DTYPE_F16: return run_loss<_Float16>(h, a, p, back, st);
    default: return run_loss<__bf16>(h, a, p, back, st);
  }
}

int loss_host(tmnn_logits *h, tmnn_class_loss_args u, bool back) {
  const size_t size = dtype_size(u.dtype), index = u.index_dtype == TMNN_INDEX_I64 ? 8 : 4, w = u.dims * size;
  HostArrays m;
  m.add(u.features, HostArrays::kIn, u.rows, w, u.feature_stride * size);
  m.add(u.table, HostArrays::kIn, u.classes, w, u.table_stride * size);
  m.add(u.labels, HostArrays::kIn, u.rows, index);
  m.add(u.row_weights, HostArrays::kIn, u.rows, 4);
  m.add(u.stats, back ? HostArrays::kIn : HostArrays::kOut, u.rows, 16);
  if (back)
    u.loss = nullptr;
  else
    m.add(u.loss, HostArrays::kOut, u.rows, 4);
  m.add(u.d_features, HostArrays::kOut, u.rows, w, u.d_feature_stride * size);
  m.add(u.d_table, HostArrays::kOut, u.classes, w, u.d_table_stride * size);
  u.feature_stride = u.table_stride = u.d_feature_stride = u.d_table_stride = u.dims;
  // (planned for the places that the arrays will have: aligned)
  tmnn_class_loss_args on_device = u;
  on_device.features = on_device.table = nullptr;
  u.workspace_bytes = u.rows > 0 ? plan_loss(on_device, back).bytes : 256;
  m.room(u.workspace, u.workspace_bytes);
  return on_host(h, m, [&] { return loss_device(h, u, back, h->ctx->stream); });
}

int class_loss(tmnn_logits *h, const tmnn_class_loss_args *args, bool back, bool host, void *stream) {
  return entry(h, [&] {
    int rc = check_loss(args, back);
    if (rc == TMNN_OK) rc = check_loss_arrays(args, back, host);
    if (rc != TMNN_OK || (args->rows == 0 && !args->d_table)) return rc;
    TMNN_HIP_TRY(hipSetDevice(h->ctx->device));
    return host ? loss_host(h, *args, back) : loss_device(h, *args, back, stream_of(h, stream));
  });
}

// ---- logits from 8-bit operands ------------------------------------------------------------

int check_logits(const tmnn_class_logits_f8_args *a) {
  const char *what = "class_logits_f8";
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (!a) return bad("args is null");
  if (a->struct_size != sizeof(*a)) return bad("struct_size mismatch");
  if (a->dtype < TMNN_DTYPE_F32 || a->dtype > TMNN_DTYPE_BF16) return bad("invalid dtype");
  if (a->scale_dtype != TMNN_SCALE_F32 && a->scale_dtype != TMNN_SCALE_E8M0) return bad("invalid scale_dtype");
  const int rc = check_sizes(what, a->rows, a->classes, a->dims);
  if (rc != TMNN_OK) return rc;
  if (a->feature_stride < a->dims || a->feature_stride > kMostStride || a->table_stride < a->dims ||
      a->table_stride > kMostStride)
    return bad("strides must be at least dims");
  if (a->logit_stride < a->classes || a->logit_stride > kMostStride) return bad("logit_stride must be at least classes");
  return TMNN_OK;
}

int check_logits_arrays(const tmnn_class_logits_f8_args *a, bool host) {
  const char *what = "class_logits_f8";
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (a->rows == 0) return TMNN_OK;
  if (!a->features || !a->feature_scales || !a->table || !a->table_scales || !a->logits)
    return bad("features, table, their scales and logits must not be null");
  const int64_t size = static_cast<int64_t>(dtype_size(a->dtype)), n = a->rows, v = a->classes;
  if (!aligned(a->logits, size)) return bad("logits must be aligned to their type");
  const int64_t s = a->scale_dtype == TMNN_SCALE_F32 ? 4 : 1;
  if (!aligned(a->feature_scales, s) || !aligned(a->table_scales, s)) return bad("scales must be aligned to their type");
  const int64_t blocks = parts_of(a->dims, kScaleBlock);
  return apart(what,
               {{a->logits, n, v * size, a->logit_stride * size, "logits"},
                {host ? nullptr : a->workspace, 1, a->workspace_bytes, 0, "the workspace"}},
               {{a->features, n, a->dims, a->feature_stride, "features"},
                {a->table, v, a->dims, a->table_stride, "the table"},
                {a->feature_scales, 1, n * blocks * s, 0, "feature_scales"},
                {a->table_scales, 1, parts_of(v, kScaleBlock) * blocks * s, 0, "table_scales"}});
}

template <class S, bool WIDE, class T>
int run_f8(const TileArgs &t, const F8Scales &s, const LogitsOut<T> &o, bool power, int device, hipStream_t st) {
  return power ? TileLaunch<S, F8Steps<S, true, WIDE>, LogitsOut<T>, F8Scales>::run(t, s, o, device, st)
               : TileLaunch<S, F8Steps<S, false, WIDE>, LogitsOut<T>, F8Scales>::run(t, s, o, device, st);
}

template <class T>
int run_logits(tmnn_logits *h, const tmnn_class_logits_f8_args &a, const LogitsPlan &p, hipStream_t st) {
  const int device = h->ctx->device;
  const int64_t n = a.rows, v = a.classes;
  char *ws = static_cast<char *>(a.workspace);
  if (p.lay_x || p.lay_y) {
    F8LayArgs l{};
    l.in[0] = static_cast<const uint8_t *>(a.features);
    l.in[1] = static_cast<const uint8_t *>(a.table);
    l.stride[0] = a.feature_stride;
    l.stride[1] = a.table_stride;
    l.rows[0] = static_cast<int32_t>(n);
    l.rows[1] = static_cast<int32_t>(v);
    l.dims = static_cast<int32_t>(a.dims);
    l.ld = static_cast<int32_t>(p.ld);
    l.out[0] = p.lay_x ? reinterpret_cast<uint8_t *>(ws + p.at_x) : nullptr;
    l.out[1] = p.lay_y ? reinterpret_cast<uint8_t *>(ws + p.at_y) : nullptr;
    hipLaunchKernelGGL(f8_lay_kernel, dim3(8 * kUnits), dim3(256), 0, st, l);
    TMNN_HIP_TRY(hipGetLastError());
  }
  const TileArgs t = logits_product(a, p);
  const F8Scales s{a.feature_scales, a.table_scales, static_cast<int32_t>(p.steps),
                   static_cast<int32_t>(parts_of(v, kScaleBlock)),
                   static_cast<int32_t>(a.dims - (p.steps - 1) * kScaleBlock)};
  float *slabs = p.t.parts > 1 ? reinterpret_cast<float *>(ws + p.at_slabs) : nullptr;
  const LogitsOut<T> o{static_cast<T *>(a.logits), a.logit_stride, slabs, static_cast<int32_t>(p.slab_ld)};
  const bool power = a.scale_dtype == TMNN_SCALE_E8M0;
  constexpr bool wide = sizeof(T) == 4;
  int rc;
  switch (p.t.shape) {
    case kLarge:
      if constexpr (!wide) {  // (fp32 logits are never planned so: 256 x 256 widened takes too many registers)
        rc = run_f8<Large<F8, false, false>, false>(t, s, o, power, device, st);
        break;
      }
    case kWide: rc = run_f8<Wide<F8, false, false>, wide>(t, s, o, power, device, st); break;
    case kMiddle: rc = run_f8<Middle<F8, false, false>, wide>(t, s, o, power, device, st); break;
    case kFlat: rc = run_f8<Flat<F8, false, false>, true>(t, s, o, power, device, st); break;
    default: rc = run_f8<Small<F8, false, false>, true>(t, s, o, power, device, st); break;
  }
  if (rc != TMNN_OK || !slabs) return rc;
  SumSlabsArgs j{slabs, a.logits, a.logit_stride, static_cast<int32_t>(p.slab_ld), p.t.parts, static_cast<int32_t>(n),
                 static_cast<int32_t>(v)};
  const int64_t blocks = std::min<int64_t>(parts_of(n * v, 256), 8 * kUnits);
  hipLaunchKernelGGL((f8_join_kernel<T>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, st, j);
  TMNN_HIP_TRY(hipGetLastError());
  return TMNN_OK;
}

int logits_device(tmnn_logits *h, const tmnn_class_logits_f8_args &a, hipStream_t st) {
  const LogitsPlan p = plan_logits(a);
  if (p.bytes > 0 && (!a.workspace || !aligned(a.workspace, 256) || a.workspace_bytes < p.bytes))
    return fail(TMNN_ERR_INVALID_ARGUMENT, "class_logits_f8: the workspace must be 256-byte aligned and hold " +
                                               std::to_string(p.bytes) + " bytes");
  switch (a.dtype) {
    case TMNN_DTYPE_F32: return run_logits<float>(h, a, p, st);
    case TMNN_DTYPE_F16: return run_logits<_Float16>(h, a, p, st);
    default: return run_logits<__bf16>(h, a, p, st);
  }
}

int logits_host(tmnn_logits *h, tmnn_class_logits_f8_args u) {
  const size_t size = dtype_size(u.dtype), s = u.scale_dtype == TMNN_SCALE_F32 ? 4 : 1;
  const int64_t blocks = parts_of(u.dims, kScaleBlock);
  HostArrays m;
  m.add(u.features, HostArrays::kIn, u.rows, u.dims, u.feature_stride);
  m.add(u.table, HostArrays::kIn, u.classes, u.dims, u.table_stride);
  m.add(u.feature_scales, HostArrays::kIn, u.rows, blocks * s);
  m.add(u.table_scales, HostArrays::kIn, parts_of(u.classes, kScaleBlock), blocks * s);
  m.add(u.logits, HostArrays::kOut, u.rows, u.classes * size, u.logit_stride * size);
  u.feature_stride = u.table_stride = u.dims;
  u.logit_stride = u.classes;
  tmnn_class_logits_f8_args on_device = u;
  on_device.features = on_device.table = nullptr;
  u.workspace_bytes = plan_logits(on_device).bytes;
  if (u.workspace_bytes > 0) m.room(u.workspace, u.workspace_bytes);
  return on_host(h, m, [&] { return logits_device(h, u, h->ctx->stream); });
}

int class_logits(tmnn_logits *h, const tmnn_class_logits_f8_args *args, bool host, void *stream) {
  return entry(h, [&] {
    int rc = check_logits(args);
    if (rc == TMNN_OK) rc = check_logits_arrays(args, host);
    if (rc != TMNN_OK || args->rows == 0) return rc;
    TMNN_HIP_TRY(hipSetDevice(h->ctx->device));
    return host ? logits_host(h, *args) : logits_device(h, *args, stream_of(h, stream));
  });
}

// ---- quantisation -----------------------------------------------------------------------------

int check_quantize(const tmnn_quantize_f8_args *a) {
  const char *what = "quantize_f8";
  auto bad = [&](const char *m) {
    return fail(TMNN_ERR_INVALID_ARGUMENT, std::string(what) + ": " + m);
  };
  if (!a) return bad("args is null");
  if (a->struct_size != sizeof(*a)) return bad("struct_size mismatch");
  if (a->dtype < TMNN_DTYPE_F32 || a->dtype > TMNN_DTYPE_BF16) return bad("invalid dtype");
  if (a->scale_dtype != TMNN_SCALE_F32 && a->scale_dtype != TMNN_SCALE_E8M0) return bad("invalid scale_dtype");
  if (a->block_rows != 1 && a->block_rows != kScaleBlock) return bad("block_rows must be 1 or 128");
  const int rc = check_sizes(what, a->rows, 1, a->dims);
  if (rc != TMNN_OK) return rc;
  if (a->stride < a->dims || a->stride > kMostStride || a->value_stride < a->dims || a->value_stride > kMostStride)
    return bad("strides must be at least dims");
  if (a->rows == 0) return TMNN_OK;
  if (!a->input || !a->values || !a->scales) return bad("input, values and scales must not be null");
  const int64_t size = static_cast<int64_t>(dtype_size(a->dtype)), s = a->scale_dtype == TMNN_SCALE_F32 ? 4 : 1;
  if (!aligned(a->input, size) || !aligned(a->scales, s)) return bad("input and scales must be aligned to their type");
  const int64_t blocks = parts_of(a->rows, a->block_rows) * parts_of(a->dims, kScaleBlock);
  return apart(what,
               {{a->values, a->rows, a->dims, a->value_stride, "values"}, {a->scales, 1, blocks * s, 0, "scales"}},
               {{a->input, a->rows, a->dims * size, a->stride * size, "input"}});
}

template <class T, bool POWER>
int run_quantize(const tmnn_quantize_f8_args &u, hipStream_t st) {
  QuantizeArgs a{u.input, u.stride, static_cast<int32_t>(u.rows), static_cast<int32_t>(u.dims),
                 static_cast<int32_t>(parts_of(u.dims, kScaleBlock)), static_cast<uint8_t *>(u.values), u.value_stride,
                 u.scales};
  if (u.block_rows == 1) {
    const int64_t blocks = std::min<int64_t>(parts_of(u.rows * a.blocks, 16), 1 << 20);
    hipLaunchKernelGGL((f8_rows_kernel<T, POWER>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, st, a);
  } else {
    const int64_t blocks = parts_of(u.rows, kScaleBlock) * a.blocks;
    hipLaunchKernelGGL((f8_table_kernel<T, POWER>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, st, a);
  }
  TMNN_HIP_TRY(hipGetLastError());
  return TMNN_OK;
}

int quantize_device(const tmnn_quantize_f8_args &u, hipStream_t st) {
  const bool power = u.scale_dtype == TMNN_SCALE_E8M0;
  switch (u.dtype) {
    case TMNN_DTYPE_F32: return power ? run_quantize<float, true>(u, st) : run_quantize<float, false>(u, st);
    case TMNN_DTYPE_F16: return power ? run_quantize<_Float16, true>(u, st) : run_quantize<_Float16, false>(u, st);
    default: return power ? run_quantize<__bf16, true>(u, st) : run_quantize<__bf16, false>(u, st);
  }
}

int quantize_host(tmnn_logits *h, tmnn_quantize_f8_args u) {
  const size_t size = dtype_size(u.dtype), s = u.scale_dtype == TMNN_SCALE_F32 ? 4 : 1;
  HostArrays m;
  m.add(u.input, HostArrays::kIn, u.rows, u.dims * size, u.stride * size);
  m.add(u.values, HostArrays::kOut, u.rows, u.dims, u.value_stride);
  m.add(u.scales, HostArrays::kOut, parts_of(u.rows, u.block_rows), parts_of(u.dims, kScaleBlock) * s);
  u.stride = u.value_stride = u.dims;
  return on_host(h, m, [&] { return quantize_device(u, h->ctx->stream); });
}

int quantize(tmnn_logits *h, const tmnn_quantize_f8_args *args, bool host, void *stream) {
  return entry(h, [&] {
    const int rc = check_quantize(args);
    if (rc != TMNN_OK || args->rows == 0) return rc;
    TMNN_HIP_TRY(hipSetDevice(h->ctx->device));
    return host ? quantize_host(h, *args) : quantize_device(*args, stream_of(h, stream));
  });
}

}  // namespace

extern "C" {

int tmnn_class_loss_workspace(const tmnn_class_loss_args *args, int32_t backward, int64_t *bytes) {
  return guarded([&] {
    if (!bytes) return fail(TMNN_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = 0;
    const int rc = check_loss(args, backward != 0);
    if (rc == TMNN_OK && args->rows > 0) *bytes = plan_loss(*args, backward != 0).bytes;
    return rc;
  });
}
int tmnn_class_loss(tmnn_logits *h, const tmnn_class_loss_args *args) {
  return class_loss(h, args, false, true, nullptr);
}
int tmnn_class_loss_device(tmnn_logits *h, const tmnn_class_loss_args *args, void *stream) {
  return class_loss(h, args, false, false, stream);
}
int tmnn_class_loss_backward(tmnn_logits *h, const tmnn_class_loss_args *args) {
  return class_loss(h, args, true, true, nullptr);
}
int tmnn_class_loss_backward_device(tmnn_logits *h, const tmnn_class_loss_args *args, void *stream) {
  return class_loss(h, args, true, false, stream);
}
int tmnn_class_logits_f8_workspace(const tmnn_class_logits_f8_args *args, int64_t *bytes) {
  return guarded([&] {
    if (!bytes) return fail(TMNN_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = 0;
    const int rc = check_logits(args);
    if (rc == TMNN_OK && args->rows > 0) *bytes = plan_logits(*args).bytes;
    return rc;
  });
}
int tmnn_class_logits_f8(tmnn_logits *h, const tmnn_class_logits_f8_args *args) {
  return class_logits(h, args, true, nullptr);
}
int tmnn_class_logits_f8_device(tmnn_logits *h, const tmnn_class_logits_f8_args *args, void *stream) {
  return class_logits(h, args, false, stream);
}
int tmnn_quantize_f8(tmnn_logits *h, const tmnn_quantize_f8_args *args) { return quantize(h, args, true, nullptr); }
int tmnn_quantize_f8_device(tmnn_logits *h, const tmnn_quantize_f8_args *args, void *stream) {
  return quantize(h, args, false, stream);
}

}  // extern "C"
