// class_loss_kernel.hpp -- softmax cross entropy of features against a table of
// classes, without a tensor of logits of the caller's, and its gradients.
//
// Of a row h with label l, logits z_v = h . W_v, c = log2(e) / T, m = max z:
//   R = sum_{v != l} 2^(c (z_v - m)),  e = 2^(c (z_l - m)),  S = R + e
//   loss = w ln(S / e): ln(1 + R) where the label is the best class (exact for small losses)
//   d_v = w / T (p_v - [v = l]),  p_v = 2^(c (z_v - m)) / S,  d_l = -w / T R / S
// The label's term is kept out of the sums, so that neither a small loss nor 1 - p of a
// confident row is a difference of two numbers near 1.
//
// The logits are a tile product (tile_product.hpp) whose epilogue sums a tile up to (max, sum) per
// row; a second kernel joins the tiles of a row. The backward pass computes the logits again (or, of a call of
// both, reads up to 512 MB of them back), for a piece of the classes at a time, writes d of the piece in
// 16 bits, and multiplies it with the table (d_features) and with the features (d_table).
//
// Numbers in 16 bits. Products take fp16 operands wherever a gradient is formed, also of
// bf16 inputs: a bf16 matrix times the power of two that brings its largest magnitude to 2^14 is
// exact in fp16 for elements down to 2^-32 of the largest, and d keeps 11 bits instead of 8 (with
// d in bf16 its rounding would add as much error as that of the results). fp32 inputs become two
// fp16 terms, 22 bits, and three products, at a third of the rate of fp16, three times that of the fp32 matrix
// instructions (154 TFLOP/s in a large product). fp16 inputs of few rows, or of few dims, have d in two terms:
// there its 11 bits would show beside those of the results. d is held as 2^14 m d T / w, m in [1, 2) being w's mantissa: its
// exponent goes to the result (d_features: exactly, rows of any weight keep their bits) or to the features (d_table: rows of
// weights far below the largest lose bits of theirs, as small features do).
// A fixed point of 2^14 means that d ends at 2^-39: a class of probability p has at most 39 + log2 p bits, in one term
// 11 of them from 2^-28 on, in two 22 from 2^-17 on.
#pragma once

#include "head_plan.hpp"
#include "tile_product.hpp"

namespace tmnn_hip {

constexpr int kDTerm = 14;         // d is held times 2^14

// Powers of two that the operands of the logits and the weighted features were multiplied with, and
// the largest weight's. Where nothing was (a null pointer), all are 0.
struct Exponents {
  int32_t x, y, w, weighted;
};
static_assert(sizeof(Exponents) == kExponentBytes, "its place in the workspace");

struct RowInfo {  // of the rows of a call
  const void *labels;
  const float *weights;  // nullable: 1
  int32_t wide;          // labels of 64 bits
  int32_t classes;
  __device__ __forceinline__ int32_t label(int64_t r) const {  // -1: none; `classes`: out of range
    if (wide) {
      const int64_t l = static_cast<const int64_t *>(labels)[r];
      return l < 0 ? -1 : l < classes ? static_cast<int32_t>(l) : classes;
    }
    const int32_t l = static_cast<const int32_t *>(labels)[r];
    return l < 0 ? -1 : l < classes ? l : classes;
  }
  __device__ __forceinline__ float weight(int64_t r) const { return weights ? weights[r] : 1.f; }
  // Whether a row counts, in two loads without a branch: a label's sign, and the weight or something in its place.
  struct Counts {
    int32_t sign;
    float weight;
  };
  __device__ __forceinline__ Counts counts(int64_t r) const {
    const float *w = weights ? weights : static_cast<const float *>(labels);
    return {static_cast<const int32_t *>(labels)[wide ? 2 * r + 1 : r], w[r]};
  }
  __device__ __forceinline__ bool used(const Counts &v) const { return v.sign >= 0 && (!weights || v.weight != 0.f); }
};

// w = m 2^e with |m| in [1, 2); what is not finite keeps e = 0.
__device__ __forceinline__ int weight_exponent(float w) {
  return w == 0.f || !__builtin_isfinite(w) ? 0 : __builtin_amdgcn_frexp_expf(w) - 1;
}

__device__ __forceinline__ float exponent_factor(int e) {  // 2^e, held to normal numbers
  return ldexpf(1.f, e < -126 ? -126 : e > 126 ? 126 : e);
}

template <class T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}

// ---- operands laid out --------------------------------------------------------------------

struct LayPart {
  const void *in;
  int64_t stride;      // elements
  int32_t rows, dims;
  char *out;           // [plane][rows][ld], nullable
  char *weighted;      // the same, rows times 2^exponent of their weights or as they are, and 0 where they do
                       // not count; nullable
  int32_t ld;          // elements, a multiple of 64: columns from dims on are 0
  int32_t scaled;      // `out` is scaled by its largest magnitude (`weighted` always is)
  int32_t planes;      // 1, or 2 (high, low)
  int32_t blocks;      // that lay it out
  int32_t parts;       // blocks that look for its largest magnitude, up to kScaleParts
};

struct LayArgs {
  LayPart part[2];     // features, table
  RowInfo row;
  uint32_t *most;      // [2][kScaleParts] largest finite magnitudes, as bits
  int32_t *most_w;     // [parts_w] largest weight exponents
  int32_t parts_w;
  int32_t by_weight;   // `weighted` is multiplied
  Exponents *exps;
};

// Threads that take a row of 8-element vectors together, so that short rows go several to a block.
__device__ __forceinline__ int row_lanes(int chunks) {
  int lanes = 1;
  while (lanes < 256 && lanes < chunks) lanes *= 2;
  return lanes;
}

template <class T>
__device__ __forceinline__ uint32_t magnitude(T v) {  // its bits, 0 for what is not finite
  const uint32_t b = __builtin_bit_cast(uint32_t, to_f32(v)) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0;
}

// The largest finite magnitude of each operand, one per block, and of the weights. Rows that do not count may hold
// anything and take no part. One pass over both: 554 MB of
// 4096 x 2048 and 131072 x 2048 bf16 in 117 us, 4.7 TB/s.
template <class T>
__global__ __launch_bounds__(256) void class_scale_kernel(LayArgs a) {
  __shared__ uint32_t top[4];
  const int parts_x = a.part[0].parts, parts_y = a.part[1].parts;
  const int which = static_cast<int>(blockIdx.x) < parts_x ? 0 : static_cast<int>(blockIdx.x) < parts_x + parts_y ? 1 : 2;
  const int block = blockIdx.x - (which > 0 ? parts_x : 0) - (which > 1 ? parts_y : 0);
  uint32_t most = 0;
  if (which < 2) {
    const LayPart &p = a.part[which];
    typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const int chunks = (p.dims + 7) / 8, lanes = row_lanes(chunks), per = 256 / lanes;
    const int64_t step = static_cast<int64_t>(p.parts) * per;
    auto used = [&](const RowInfo::Counts &v) { return which == 1 || a.row.used(v); };
    // (of the table's rows, which all count, some row's)
    auto counts = [&](int64_t r) { return a.row.counts(which == 1 ? 0 : r); };
    for (int c = threadIdx.x % lanes; c < chunks; c += lanes) {
      const T *at = static_cast<const T *>(p.in) + c * 8;
      auto scan = [&](auto load) {
        auto top_of = [&](const V &v, const RowInfo::Counts &in) {
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[i]));
          most = max(most, used(in) ? top : 0);
        };
        int64_t r = static_cast<int64_t>(block) * per + threadIdx.x / lanes;
        for (; r + 3 * step < p.rows; r += 4 * step) {  // four loads on their way
          V v[4];
          RowInfo::Counts in[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            v[u] = load(at + (r + u * step) * p.stride);
            in[u] = counts(r + u * step);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) top_of(v[u], in[u]);
        }
        for (; r < p.rows; r += step) top_of(load(at + r * p.stride), counts(r));
      };
      const int last = p.dims - 1 - c * 8;
      if (last >= 7)
        scan([](const T *x) { return *reinterpret_cast<const V *>(x); });
      else  // (a row's end: its last value in place of those past it, without a branch)
        scan([=](const T *x) {
          V v;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = x[min(i, last)];
          return v;
        });
    }
  } else {
    // (exponents shifted by 1000, 0 being none)
    for (int64_t r = static_cast<int64_t>(block) * 256 + threadIdx.x; r < a.part[0].rows; r += 256ll * a.parts_w) {
      if (a.row.used(a.row.counts(r))) most = max(most, static_cast<uint32_t>(weight_exponent(a.row.weight(r)) + 1000));
    }
  }
#pragma unroll
  for (int s = 32; s > 0; s /= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), s)));
  if (threadIdx.x % 64 == 0) top[threadIdx.x / 64] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    most = max(max(top[0], top[1]), max(top[2], top[3]));
    if (which < 2)
      a.most[which * kScaleParts + block] = most;
    else
      a.most_w[block] = static_cast<int32_t>(most) - 1000;
  }
}

__device__ __forceinline__ int block_max_256(int v, int *room) {
#pragma unroll
  for (int s = 32; s > 0; s /= 2) v = max(v, __shfl_xor(v, s));
  if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = v;
  __syncthreads();
  v = max(max(room[0], room[1]), max(room[2], room[3]));
  __syncthreads();
  return v;
}

__device__ __forceinline__ int largest(const int *v, int n, int least) {
  for (int i = threadIdx.x; i < n; i += 256) least = max(least, v[i]);
  return least;
}

// The exponent that brings a magnitude (its bits) to [2^14, 2^15).
__device__ __forceinline__ int scale_exponent(int bits) {
  if (bits == 0) return 0;
  const int e = 14 - (__builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, bits)) - 1);
  return e > 126 ? 126 : e;
}

// Lays both operands out: scaled, in fp16 terms (or copied as they are), rows at
// multiples of 128 bytes. Read once and written once: those 554 MB in 206 us, 5.4 TB/s.
template <class T, bool SCALED>
__global__ __launch_bounds__(256) void class_lay_kernel(LayArgs a) {
  __shared__ int room[4];
  const int which = blockIdx.x < static_cast<uint32_t>(a.part[0].blocks) ? 0 : 1;
  const LayPart &p = a.part[which];
  const int block = which ? blockIdx.x - a.part[0].blocks : blockIdx.x;
  int e = 0, seen = 0, top_w = 0;
  if constexpr (SCALED) {
    int exps[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (a.part[k].parts > 0)
        exps[k] = scale_exponent(block_max_256(largest(reinterpret_cast<const int *>(a.most) + k * kScaleParts,
                                                       a.part[k].parts, 0), room));
    top_w = block_max_256(largest(a.most_w, a.parts_w, -1000), room);
    seen = exps[which];
    e = p.scaled ? seen : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0)
      *a.exps = {a.part[0].scaled ? exps[0] : 0, a.part[1].scaled ? exps[1] : 0, top_w, exps[0] * (a.by_weight | a.part[0].scaled)};
  }
  const int chunks = p.ld / 8;
  const int lanes = row_lanes(chunks), per = 256 / lanes;
  typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const int64_t plane = static_cast<int64_t>(p.rows) * p.ld;
  for (int64_t r = static_cast<int64_t>(block) * per + threadIdx.x / lanes; r < p.rows;
       r += static_cast<int64_t>(p.blocks) * per) {
    const T *row = static_cast<const T *>(p.in) + r * p.stride;
    float factor = 0.f;
    bool used = false;
    if (SCALED && p.weighted) {
      const float w = a.row.weight(r);
      used = a.row.label(r) >= 0 && w != 0.f;
      factor = used ? a.by_weight == 0 ? 1.f : ldexpf(1.f, max(weight_exponent(w) - top_w, -149)) : 0.f;
    }
    for (int c = threadIdx.x % lanes; c < chunks; c += lanes) {
      V v = {};
      if (c * 8 + 8 <= p.dims) {
        v = *reinterpret_cast<const V *>(row + c * 8);
      } else {
        for (int i = 0; i < 8; ++i)
          if (c * 8 + i < p.dims) v[i] = row[c * 8 + i];
      }
      const int64_t at = r * p.ld + c * 8;
      if constexpr (!SCALED) {
        *reinterpret_cast<V *>(reinterpret_cast<T *>(p.out) + at) = v;
      } else {
        f16x8 high, low;
        float f[8];
        if (p.out) {
          const float s = exponent_factor(e);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = to_f32(v[i]) * s;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            high[i] = static_cast<_Float16>(f[i]);
            low[i] = static_cast<_Float16>(f[i] - static_cast<float>(high[i]));
          }
          *reinterpret_cast<f16x8 *>(reinterpret_cast<_Float16 *>(p.out) + at) = high;
          if (p.planes == 2) *reinterpret_cast<f16x8 *>(reinterpret_cast<_Float16 *>(p.out) + plane + at) = low;
        }
        if (p.weighted) {
          const float s = exponent_factor(a.by_weight ? seen : e);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float g = used ? to_f32(v[i]) * s * factor : 0.f;  // (a row without weight may hold anything)
            high[i] = static_cast<_Float16>(g);
            low[i] = static_cast<_Float16>(g - static_cast<float>(high[i]));
          }
          *reinterpret_cast<f16x8 *>(reinterpret_cast<_Float16 *>(p.weighted) + at) = high;
          if (p.planes == 2)
            *reinterpret_cast<f16x8 *>(reinterpret_cast<_Float16 *>(p.weighted) + plane + at) = low;
        }
      }
    }
  }
}

// ---- the logits' epilogues -----------------------------------------------------------------

__device__ __forceinline__ float logit_scale(const Exponents *e) { return e ? exponent_factor(-(e->x + e->y)) : 1.f; }

// A tile's rows as (max, sum) over the classes other than the label's, and the label's logit. The logits' products
// bound it: 4096 x 2048 x 131072 bf16, 2.2 TFLOP, in 1.85 ms, 1.19 PFLOP/s (the same matrix product by the library,
// which writes the logits, runs at 1.5).
struct SumsEpilogue {
  const Exponents *exps;  // nullable: operands as they are
  RowInfo row;
  float c;
  float2 *sums;           // [rows][tiles_c]
  float *own;             // [rows] the label's logit
  float *z;               // [rows][z_ld] the logits, nullable
  int64_t z_ld;

  template <class S>
  __device__ __forceinline__ void finish(const TileArgs &a, const TilePlace &p, f32x4t (&acc)[S::FC][S::FR],
                                         int c0, int r0, int wc, int wr, int lane) const {
    float2 *part = reinterpret_cast<float2 *>(tile_lds);  // [WC][BR]
    const float inv = logit_scale(exps);
    const int g4 = 4 * (lane / 16);
#pragma unroll
    for (int j = 0; j < S::FR; ++j) {
      const int r = r0 + j * 16 + lane % 16;
      const int label = r < a.rows ? row.label(r) : -1;
      float m = -3.4e38f, s = 0.f;
#pragma unroll
      for (int i = 0; i < S::FC; ++i) {
        const int four = c0 + i * 16 + g4;
        acc[i][j] *= inv;
        if (z && r < a.rows && four < z_ld) *reinterpret_cast<f32x4t *>(z + r * z_ld + four) = acc[i][j];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = four + e;
          float v = acc[i][j][e];
          if (col == label) own[r] = v;
          v = col == label || col >= a.cols ? -__builtin_inff() : v;
          acc[i][j][e] = v;
          m = fmaxf(m, v);
        }
      }
#pragma unroll
      for (int i = 0; i < S::FC; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f((acc[i][j][e] - m) * c);
#pragma unroll
      for (int x = 16; x < 64; x *= 2) {
        const float mo = __shfl_xor(m, x), so = __shfl_xor(s, x);
        const float top = fmaxf(m, mo);
        s = s * __builtin_amdgcn_exp2f((m - top) * c) + so * __builtin_amdgcn_exp2f((mo - top) * c);
        m = top;
      }
      if (lane < 16) part[wc * S::BR + wr * S::FR * 16 + j * 16 + lane] = float2{m, s};
    }
    __syncthreads();
    for (int t = threadIdx.x; t < S::BR; t += S::kThreads) {
      const int r = p.r * S::BR + t;
      if (r >= a.rows) continue;
      float2 v = part[t];
#pragma unroll
      for (int w = 1; w < S::WC; ++w) {
        const float2 o = part[w * S::BR + t];
        const float top = fmaxf(v.x, o.x);
        v.y = v.y * __builtin_amdgcn_exp2f((v.x - top) * c) + o.y * __builtin_amdgcn_exp2f((o.x - top) * c);
        v.x = top;
      }
      sums[static_cast<int64_t>(r) * a.tiles_c + p.c] = v;
    }
  }
};

struct JoinArgs {
  RowInfo row;
  const float2 *sums;
  const float *own;
  int32_t rows, tiles, lanes;  // lanes of a row, a power of two
  float c, inv_t;
  float *loss;                 // nullable
  float4 *stats;               // (m, S, R / S, 0)
};

// The label's logit in a row's end: NaN without such a class, and where it is not finite, so that all that comes
// of it is NaN too. (An infinite one would end as a loss of 0 or infinity beside sums that look sound.)
__device__ __forceinline__ float own_logit(float z, int label, int classes) {
  return label < classes && __builtin_isfinite(z) ? z : __builtin_nanf("");
}

__global__ __launch_bounds__(256) void class_join_kernel(JoinArgs a) {
  const int lane = threadIdx.x % a.lanes;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (256 / a.lanes) + threadIdx.x / a.lanes;
  const bool here = r < a.rows;
  const int label = here ? a.row.label(r) : -1;
  float m = -3.4e38f, s = 0.f;
  if (here)
    for (int t = lane; t < a.tiles; t += 8 * a.lanes) {  // (eight loads on their way)
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = t + u * a.lanes < a.tiles ? a.sums[r * a.tiles + t + u * a.lanes] : float2{-3.4e38f, 0.f};
      float top = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, v[u].x);
      s *= __builtin_amdgcn_exp2f((m - top) * a.c);
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u].y * __builtin_amdgcn_exp2f((v[u].x - top) * a.c);
      m = top;
    }
  for (int x = 1; x < a.lanes; x *= 2) {
    const float mo = __shfl_xor(m, x), so = __shfl_xor(s, x);
    const float top = fmaxf(m, mo);
    s = s * __builtin_amdgcn_exp2f((m - top) * a.c) + so * __builtin_amdgcn_exp2f((mo - top) * a.c);
    m = top;
  }
  if (!here || lane != 0) return;
  float loss = 0.f, big = m, total = s, missing = 1.f;
  if (label >= 0) {
    const float z = own_logit(a.own[r], label, a.row.classes);
    big = fmaxf(m, z);
    s *= __builtin_amdgcn_exp2f((m - big) * a.c);
    total = s + __builtin_amdgcn_exp2f((z - big) * a.c);
    missing = s / total;
    loss = z >= m ? log1pf(s) : logf(total) + (m - z) * a.inv_t;
    const float w = a.row.weight(r);
    loss = w == 0.f ? 0.f : loss * w;
  }
  if (a.loss) a.loss[r] = loss;
  if (a.stats) a.stats[r] = float4{big, total, missing, 0.f};
}

// What a row's d is made of.
struct GradRow {
  int label;
  bool used;
  float big, share, mine;
  __device__ __forceinline__ GradRow(const RowInfo &row, const float4 *stats, int r, int first) {
    const float w = row.weight(r);
    const int l = row.label(r);
    label = l - first;
    used = l >= 0 && w != 0.f;
    const float4 st = stats[r];
    float f = __builtin_isfinite(w) ? __builtin_amdgcn_frexp_mantf(w) * (2.f * (1 << kDTerm)) : w;
    if (l == row.classes) f = __builtin_nanf("");
    big = st.x;
    share = f / st.y;
    mine = -f * st.z;
  }
  // of the logit z of class `col` of `cols`
  __device__ __forceinline__ float operator()(float z, int col, int cols, float c) const {
    float v = __builtin_amdgcn_exp2f((z - big) * c) * share;
    v = col == label ? mine : v;
    return used && col < cols ? v : 0.f;
  }
};

// The piece's d in fp16 terms, times 2^14, the weight's mantissa and T / w. A quarter of those classes, with 268 MB of
// d written: 0.52 ms, 1.06 PFLOP/s.
struct GradEpilogue {
  const Exponents *exps;
  RowInfo row;
  float c;
  const float4 *stats;
  int32_t first;       // class of the piece's first column
  int32_t width;       // columns to write: those past the piece are 0
  int64_t ld;
  int32_t planes;
  int64_t plane;       // elements
  _Float16 *d;         // [plane][rows][ld]

  template <class S>
  __device__ __forceinline__ void finish(const TileArgs &a, const TilePlace &, f32x4t (&acc)[S::FC][S::FR],
                                         int c0, int r0, int, int, int lane) const {
    const float inv = logit_scale(exps);
    const int g4 = 4 * (lane / 16);
#pragma unroll
    for (int j = 0; j < S::FR; ++j) {
      const int r = r0 + j * 16 + lane % 16;
      if (r >= a.rows) continue;
      const GradRow d_of(row, stats, r, first);
#pragma unroll
      for (int i = 0; i < S::FC; ++i) {
        const int col = c0 + i * 16 + g4;
        if (col >= width) continue;
        f16x4 high, low;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = d_of(acc[i][j][e] * inv, col + e, a.cols, c);
          high[e] = static_cast<_Float16>(v);
          low[e] = static_cast<_Float16>(v - static_cast<float>(high[e]));
        }
        const int64_t at = static_cast<int64_t>(r) * ld + col;
        *reinterpret_cast<f16x4 *>(d + at) = high;
        if (planes == 2) *reinterpret_cast<f16x4 *>(d + plane + at) = low;
      }
    }
  }
};

// The same from logits that the sums' pass kept: one pass, 515 x 50021 in 30 us (154 MB, 5.1 TB/s), which adds
// 20 us to the sums' pass.
struct TermsArgs {
  RowInfo row;
  float c;
  const float4 *stats;
  const float *z;      // [rows][ld]
  int32_t rows, cols;
  int32_t chunks;      // of 8 columns of a row, those past `cols` give 0
  int32_t lanes, splits;  // threads that take a row together, a power of two; blocks that do
  int64_t z_ld, ld;
  int32_t planes;
  int64_t plane;
  _Float16 *d;
};

__global__ __launch_bounds__(256) void class_terms_kernel(TermsArgs a) {
  const int r = static_cast<int>(blockIdx.x / a.splits) * (256 / a.lanes) + threadIdx.x / a.lanes;
  if (r >= a.rows) return;
  const GradRow d_of(a.row, a.stats, r, 0);
  const float *z = a.z + r * a.z_ld;
  _Float16 *d = a.d + r * a.ld;
  for (int k = blockIdx.x % a.splits * a.lanes + threadIdx.x % a.lanes; k < a.chunks; k += a.splits * a.lanes) {
    f32x4t in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) in[h] = *reinterpret_cast<const f32x4t *>(z + k * 8 + 4 * h);
    f16x8 high, low;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = d_of(in[i / 4][i % 4], k * 8 + i, a.cols, a.c);
      high[i] = static_cast<_Float16>(v);
      low[i] = static_cast<_Float16>(v - static_cast<float>(high[i]));
    }
    *reinterpret_cast<f16x8 *>(d + k * 8) = high;
    if (a.planes == 2) *reinterpret_cast<f16x8 *>(d + a.plane + k * 8) = low;
  }
}

// ---- the gradients' epilogues ----------------------------------------------------------------

// What a sum of products is multiplied with: 2^e / T, e of the row (d_features) or of all (d_table).
struct GradScale {
  const Exponents *exps;  // nullable
  RowInfo row;
  float inv_t;
  int32_t by_row;
  __device__ __forceinline__ float operator()(float v, int r, const Exponents &e, bool &none) const {
    int k = -kDTerm;
    none = false;
    if (by_row) {
      const float w = row.weight(r);
      none = row.label(r) < 0 || w == 0.f;
      k += weight_exponent(w) - e.y;
    } else {
      k += e.w - e.weighted;
    }
    return none ? 0.f : ldexpf(v * inv_t, k);
  }
};

template <class T>
__device__ __forceinline__ void store_four(T *p, const float (&v)[4], int n) {
  typedef T V __attribute__((ext_vector_type(4)));
  typedef V VU __attribute__((aligned(sizeof(T))));
  if (n >= 4) {
    V o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = static_cast<T>(v[i]);
    *reinterpret_cast<VU *>(p) = o;
  } else {
    for (int i = 0; i < n; ++i) p[i] = static_cast<T>(v[i]);
  }
}

// The finished gradient, or, where it comes in parts, sums in fp32 that class_reduce_kernel ends. For that quarter
// d_features takes 0.42 ms (1.31 PFLOP/s), d_table 0.465 (1.18).
template <class T>
struct GradOut {
  GradScale scale;
  T *out;          // [rows][cols]
  int64_t ld;
  float *slabs;    // [part][rows][slab_ld], nullable
  int32_t slab_ld;
  int32_t add;     // to what the slabs hold (pieces after the first)

  template <class S>
  __device__ __forceinline__ void finish(const TileArgs &a, const TilePlace &p, f32x4t (&acc)[S::FC][S::FR],
                                         int c0, int r0, int, int, int lane) const {
    const int g4 = 4 * (lane / 16);
    Exponents e = {};
    if (!slabs && scale.exps) e = *scale.exps;
#pragma unroll
    for (int j = 0; j < S::FR; ++j) {
      const int r = r0 + j * 16 + lane % 16;
      if (r >= a.rows) continue;
#pragma unroll
      for (int i = 0; i < S::FC; ++i) {
        const int col = c0 + i * 16 + g4;
        if (col >= a.cols) continue;
        if (slabs) {
          f32x4t *s = reinterpret_cast<f32x4t *>(slabs + (static_cast<int64_t>(p.part) * a.rows + r) * slab_ld + col);
          *s = add ? *s + acc[i][j] : acc[i][j];
        } else {
          float v[4];
          bool none;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = scale(acc[i][j][k], r, e, none);
          store_four<T>(out + r * ld + col, v, a.cols - col);
        }
      }
    }
  }
};

struct ReduceArgs {
  GradScale scale;
  void *out;
  int64_t ld;
  const float *slabs;
  int32_t slab_ld, parts, rows, cols;
  int32_t lanes;  // threads that share a sum's parts, a power of two
};

// Many parts of few sums go to several threads a sum, in a fixed order: 150 x 64 sums of 335 parts 88 -> 5.4 us,
// 1000 x 64 of 64 parts 19 -> 4.9.
template <class T>
__global__ __launch_bounds__(256) void class_reduce_kernel(ReduceArgs a) {
  __shared__ f32x4t shared[256];
  const int64_t per = a.slab_ld / 4, n = per * a.rows;
  const int width = 256 / a.lanes, lane = threadIdx.x / width;
  const Exponents e = a.scale.exps ? *a.scale.exps : Exponents{};
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * width; first < n;
       first += static_cast<int64_t>(gridDim.x) * width) {
    const int64_t at = first + threadIdx.x % width;
    f32x4t sum = {0.f, 0.f, 0.f, 0.f};
    if (at < n) {
      const f32x4t *s = reinterpret_cast<const f32x4t *>(a.slabs) + at;
      int p = lane;
      for (; p + 3 * a.lanes < a.parts; p += 4 * a.lanes) {  // four loads on their way
        f32x4t v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = s[(p + u * a.lanes) * n];
#pragma unroll
        for (int u = 0; u < 4; ++u) sum += v[u];
      }
      for (; p < a.parts; p += a.lanes) sum += s[p * n];
    }
    for (int x = a.lanes / 2; x > 0; x /= 2) {
      shared[threadIdx.x] = sum;
      __syncthreads();
      if (lane < x) sum += shared[threadIdx.x + x * width];
      __syncthreads();
    }
    const int r = static_cast<int>(at / per), c = static_cast<int>(at - r * per) * 4;
    if (at >= n || lane > 0 || c >= a.cols) continue;
    float v[4];
    bool none;
    for (int k = 0; k < 4; ++k) v[k] = a.scale(sum[k], r, e, none);
    store_four<T>(static_cast<T *>(a.out) + r * a.ld + c, v, a.cols - c);
  }
}

}  // namespace tmnn_hip
