// narrow_kernel.hpp -- the class head for features of up to 128 dims: loss and
// d_features in one walk over the table, d_table in one walk over the rows, with
// neither logits nor d ever in memory.
//
// A wave holds 16 items (rows, or classes for d_table; of many classes 32) in registers and walks over the other
// side's items in tiles of 64 that the block shares in LDS:
//   z = x y^T          16 x 16 x 32 products; a lane gets 4 neighbouring items y of one item x
//   d = f(z)           the softmax's terms or its gradient, in fp16 (two terms for fp32 inputs)
//   o += d y           the same tile read transposed: which values of k a lane holds does not matter as
//                      long as both operands agree, so d goes from the first product's result
//                      straight into the second one's operand
// For wide features this would hold dims / 16 accumulators of the second product a 16 x 16 block; up to
// 128 dims they fit beside the rest. The walk over the table keeps a running maximum, as an online
// softmax does, and the label's class out of its sums.
//
// The walk over the table holds a class's part relative to the row's best other class, the walk over the rows p itself
// times 2^14 and the row's weight over the largest one's power of two: there a class has at most 39 + log2 p bits, and
// rows of smaller weights as many fewer.
//
// Products and exponentials take turns on a unit. 4096 x 128 x 131072 bf16, 275 GFLOP a walk: 328 to 336 us for loss and
// d_features (0.83 PFLOP/s), 352 for d_table; 262144 x 64 x 1000 bf16, 67 GFLOP a walk: 123 and 144 us (0.5).
#pragma once

#include <type_traits>

#include "class_loss_kernel.hpp"

namespace tmnn_hip {

constexpr int kWalkThreads = kWalkWaves * 64;
constexpr int kWalkStages = 2;

constexpr float kLowest = -3.4e38f;  // a maximum of nothing

// Both sides laid out as [plane][items][DP] in fp16.
struct WalkArgs {
  const char *x, *y;
  int64_t x_plane, y_plane;  // bytes
  int32_t nx, ny;
  int32_t blocks;            // of kWalkWaves * 16 RJ items x
  int32_t part_tiles;        // tiles of y of one part
};

// Which 16 bytes of an item lie at a place in LDS: reads of 16 items' same chunk meet no bank twice. (The transposing
// reads meet one twice, a third of LDS's busy time. An order without that, by the counters too, was no faster, 65536 x
// 64 x 1000 fp32 62 us and 63, and its registers leave room for three waves where four were: 4096 x 128 x 131072
// bf16 325 and 360.)
template <int DP>
__device__ __forceinline__ int walk_swizzle(int item) {
  return DP == 32 ? (item >> 2) & 3 : DP == 64 ? (item >> 1) & 7 : item & 15;
}

template <int DP, int PL>
struct WalkTile {
  static constexpr int kRow = DP * 2, kPlane = kWalkItems * kRow, kBytes = PL * kPlane;
  static constexpr int kLds = kWalkStages * (kBytes + kWalkItems * 16);  // (the items' numbers behind the tiles)
  static constexpr int kLoads = kBytes / 1024 / kWalkWaves;
  static constexpr int kChunks = DP / 8, kItems = 64 / kChunks;  // of a load
  static_assert(kBytes % (1024 * kWalkWaves) == 0, "every wave loads as much");
};

// The largest of four lanes 16 apart. (Written out, with the waits that these instructions need around them:
// of the builtins' two results the compiler keeps one.)
__device__ __forceinline__ float max_of_four(float v) {
  float a = v, b = v;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  a = b = fmaxf(a, b);
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}

// Eight values in fp16, of one lane: with two terms the high ones are cut and the low ones take the rest.
template <int PL>
__device__ __forceinline__ void to_terms(const f32x4t &a, const f32x4t &b, f16x8 (&t)[PL]) {
  if constexpr (PL == 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[0][e] = static_cast<_Float16>(a[e]);
      t[0][4 + e] = static_cast<_Float16>(b[e]);
    }
  } else {
    typedef __fp16 h2 __attribute__((ext_vector_type(2)));
    union {
      h2 h[4];
      f16x8 v;
    } u;
    u.h[0] = __builtin_amdgcn_cvt_pkrtz(a[0], a[1]);
    u.h[1] = __builtin_amdgcn_cvt_pkrtz(a[2], a[3]);
    u.h[2] = __builtin_amdgcn_cvt_pkrtz(b[0], b[1]);
    u.h[3] = __builtin_amdgcn_cvt_pkrtz(b[2], b[3]);
    t[0] = u.v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[1][e] = static_cast<_Float16>(__builtin_fmaf(-static_cast<float>(u.v[e]), 1.f, a[e]));
      t[1][4 + e] = static_cast<_Float16>(__builtin_fmaf(-static_cast<float>(u.v[4 + e]), 1.f, b[e]));
    }
  }
}

// `n` groups of products, the reads of each beside the products of the one before.
template <int n, int reads, int products>
__device__ __forceinline__ void ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
#pragma unroll
  for (int s = 0; s < n; ++s) {
    if (s + 1 < n) __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, products, 0);
  }
}

// PL, PD: terms of the operands and of d (d of fp16 gradients, which hold as many bits as one term, goes in two).
// RJ: 16 items x of a wave, or 32. 32 halve the reads from LDS; with 16 a call has twice the blocks, of
// half the registers, so that some multiply while others take exponentials.
template <int DP, int PL, int PD, int RJ, class Op>
__global__ __launch_bounds__(kWalkThreads, RJ == 1 ? (DP <= 64 ? 4 : 3) : DP <= 64 ? 3 : 2) void walk_kernel(WalkArgs a, Op op) {
  typedef WalkTile<DP, PL> W;
  constexpr int KS = DP / 32, FD = DP / 16;
  constexpr int kInfo = Op::kInfo ? kWalkItems * 16 : 0;
  char *const lds = tile_lds;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int block = blockIdx.x % a.blocks, part = blockIdx.x / a.blocks;
  const int r0 = (block * kWalkWaves + wave) * (16 * RJ);
  const int tiles = (a.ny + kWalkItems - 1) / kWalkItems;
  const int from = part * a.part_tiles, to = min(tiles, from + a.part_tiles);

  // this wave's items; those past the end are 0
  f16x8 hx[RJ][KS][PL];
#pragma unroll
  for (int j = 0; j < RJ; ++j) {
    const int r = r0 + j * 16 + lane % 16;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int p = 0; p < PL; ++p)
        hx[j][k][p] = r < a.nx ? *reinterpret_cast<const f16x8 *>(a.x + p * a.x_plane + static_cast<int64_t>(r) * W::kRow +
                                                                 k * 64 + lane / 16 * 16)
                               : f16x8{};
  }

  // loads of a tile into a stage
  const uint32_t first = __builtin_amdgcn_readfirstlane(lds_address(lds));
  uint32_t off[W::kLoads];
  int item[W::kLoads];
#pragma unroll
  for (int q = 0; q < W::kLoads; ++q) {
    const int piece = q * kWalkWaves + wave;  // of 1 KB
    item[q] = piece % (W::kPlane / 1024) * W::kItems + lane / W::kChunks;
    off[q] = static_cast<uint32_t>(item[q] * W::kRow + 16 * ((lane % W::kChunks) ^ walk_swizzle<DP>(item[q])));
  }
  auto load = [&](int tile, int stage) {
#pragma unroll
    for (int q = 0; q < W::kLoads; ++q) {
      const int p = (q * kWalkWaves + wave) / (W::kPlane / 1024);
      const char *b = a.y + p * a.y_plane + static_cast<int64_t>(tile) * kWalkItems * W::kRow;
      i32x4t rsrc;
      rsrc[0] = static_cast<int32_t>(reinterpret_cast<uintptr_t>(b));
      rsrc[1] = static_cast<int32_t>((reinterpret_cast<uintptr_t>(b) >> 32) & 0xffff);
      rsrc[2] = 0x7fffffff;
      rsrc[3] = 0x00020000;
      const uint32_t o = tile < to && tile * kWalkItems + item[q] < a.ny ? off[q] : kOutside;
      asm volatile(
          "s_mov_b32 m0, %0\n\t"
          "s_nop 0\n\t"
          "buffer_load_dwordx4 %1, %2, 0 offen lds"
          :
          : "s"(first + stage * W::kBytes + (q * kWalkWaves + wave) * 1024), "v"(o), "s"(rsrc)
          : "memory");
    }
  };

  f32x4t out[FD][RJ];
#pragma unroll
  for (int f = 0; f < FD; ++f)
#pragma unroll
    for (int j = 0; j < RJ; ++j) out[f][j] = f32x4t{0.f, 0.f, 0.f, 0.f};
  op.begin(r0, a.nx, lane);

  load(from, 0);
  int stage = 0;
  auto walk = [&](int tile, auto edge) {  // edge: the tile may end before its 64 items
    char *info = lds + kWalkStages * W::kBytes + stage * kInfo;
    if constexpr (Op::kInfo) op.put_info(info, tile * kWalkItems, a.ny);
    // the tile has arrived (and its items' numbers), and all waves are done with the one before
    wait_and_meet<0>();
    load(tile + 1, stage ^ 1);
    const char *y = lds + stage * W::kBytes;
    f32x4t z[4][RJ];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < RJ; ++j) z[i][j] = f32x4t{0.f, 0.f, 0.f, 0.f};
    // fragments are read one pair of products ahead
    auto read_z = [&](f16x8 (&fy)[PL], int s) {
      const int k = s / 4, it = s % 4 * 16 + lane % 16;
#pragma unroll
      for (int p = 0; p < PL; ++p)
        fy[p] = *reinterpret_cast<const f16x8 *>(y + p * W::kPlane + it * W::kRow +
                                                 16 * ((k * 4 + lane / 16) ^ walk_swizzle<DP>(it)));
    };
    f16x8 fy[2][PL];
    read_z(fy[0], 0);
#pragma unroll
    for (int s = 0; s < KS * 4; ++s) {
      const int k = s / 4, i = s % 4;
      if (s + 1 < KS * 4) read_z(fy[(s + 1) % 2], s + 1);
#pragma unroll
      for (int t = 0; t < (PL == 2 ? 3 : 1); ++t)  // (a result is not needed by the product right behind it)
#pragma unroll
        for (int j = 0; j < RJ; ++j)
          z[i][j] = Fragment<F16>::mul(fy[s % 2][t == 1], hx[j][k][t == 2], z[i][j]);
    }
    ahead<KS * 4, PL, (PL == 2 ? 3 : 1) * RJ>();
    op.template transform<decltype(edge)::value>(z, out, info, tile * kWalkItems, a.ny, lane);
    if constexpr (Op::kGradient) {
      f16x8 dx[2][RJ][PD];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int j = 0; j < RJ; ++j) to_terms<PD>(z[2 * kk][j], z[2 * kk + 1][j], dx[kk][j]);
      __builtin_amdgcn_sched_barrier(0);
      auto read_t = [&](f16x8 (&ft)[PL], int s) {
        const int kk = s / FD, f = s % FD, t = lane % 16;
#pragma unroll
        for (int p = 0; p < PL; ++p) {
          union {
            s16x4 half[2];
            f16x8 v;
          } u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int it = 32 * kk + 16 * h + 4 * (lane / 16) + t / 4;
            const char *at = y + p * W::kPlane + it * W::kRow +
                             16 * ((2 * f + (t % 4) / 2) ^ walk_swizzle<DP>(it)) + (t % 2) * 8;
            u.half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(__attribute__((address_space(3))) char *)at);
          }
          ft[p] = u.v;
        }
      };
      f16x8 ft[2][PL];
      read_t(ft[0], 0);
#pragma unroll
      for (int s = 0; s < 2 * FD; ++s) {
        const int kk = s / FD, f = s % FD;
        if (s + 1 < 2 * FD) read_t(ft[(s + 1) % 2], s + 1);
#pragma unroll
        for (int t = 0; t < PL + PD - 1; ++t)  // high and high, y low, d low
#pragma unroll
          for (int j = 0; j < RJ; ++j)
            out[f][j] = Fragment<F16>::mul(ft[s % 2][PL == 2 && t == 1], dx[kk][j][t > 0 && t == PL + PD - 2], out[f][j]);
      }
      ahead<2 * FD, 2 * PL, (PL + PD - 1) * RJ>();
    }
    stage ^= 1;
  };
  for (int tile = from; tile < to - 1; ++tile) walk(tile, std::false_type{});
  if (from < to) walk(to - 1, std::true_type{});
  wait_and_meet<0>();  // (the last load's zeros)
  op.template finish<FD>(out, a, r0, part, lane);
}

// A lane's share (16 bytes of each 64) of the product of item x `r` and item y `l`: the walk leaves the
// label's class out, and has no use for its logit before the end.
template <int KS, int PL>
__device__ __forceinline__ float own_product(const WalkArgs &a, int r, int l, int lane) {
  float z = 0.f;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    f16x8 x[PL], y[PL];
#pragma unroll
    for (int p = 0; p < PL; ++p) {
      x[p] = *reinterpret_cast<const f16x8 *>(a.x + p * a.x_plane + static_cast<int64_t>(r) * (KS * 64) + k * 64 + lane / 16 * 16);
      y[p] = *reinterpret_cast<const f16x8 *>(a.y + p * a.y_plane + static_cast<int64_t>(l) * (KS * 64) + k * 64 + lane / 16 * 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float xh = static_cast<float>(x[0][i]), yh = static_cast<float>(y[0][i]);
      z = __builtin_fmaf(xh, yh, z);
      if constexpr (PL == 2) {
        z = __builtin_fmaf(xh, static_cast<float>(y[1][i]), z);
        z = __builtin_fmaf(static_cast<float>(x[1][i]), yh, z);
      }
    }
  }
  return z;
}

// What is left to do once a row's sums are whole: loss, stats, and what d_features is made of.
struct RowEnd {
  float loss, big, total, missing, scale;  // scale: of the sums over the other classes
};

__device__ __forceinline__ RowEnd end_row(float m, float s, float z, int label, int classes, float w, float c,
                                          float inv_t) {
  RowEnd e{0.f, m, s, 1.f, 0.f};
  if (label >= 0) {
    z = own_logit(z, label, classes);
    e.big = fmaxf(m, z);
    e.scale = __builtin_amdgcn_exp2f((m - e.big) * c);
    s *= e.scale;
    e.total = s + __builtin_amdgcn_exp2f((z - e.big) * c);
    e.missing = s / e.total;
    e.loss = z >= m ? log1pf(s) : logf(e.total) + (m - z) * inv_t;
    e.loss = w == 0.f ? 0.f : e.loss * w;
    e.scale /= e.total;
  }
  return e;
}

// The walk over the table: rows are the items x.
struct RowsShared {
  const Exponents *exps;
  RowInfo row;
  float c, inv_t;
  float *loss;            // nullable
  float4 *stats;          // nullable
  // in parts: [part][rows] (max, sum), the label's logits, [part][rows][DP] sums of the table
  float2 *part_sum;       // nullable: one part
  float *own;             // [rows]
  float *part_out;
};

// d_features of four dims, of a row that is used.
template <class T>
__device__ __forceinline__ void put_features(const RowsShared &g, const RowEnd &e, float w, int label, int r, int dim,
                                             f32x4t sum, float back, const T *table, int64_t table_ld, T *out,
                                             int64_t out_ld, int dims) {
  const bool used = label >= 0 && w != 0.f;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = dim + i;
    const float mine = used && label < g.row.classes && d < dims ? to_f32(table[label * table_ld + d]) : 0.f;
    v[i] = used ? (sum[i] * back * e.scale - e.missing * mine) * (w * g.inv_t) : 0.f;
  }
  if (dim < dims) store_four<T>(out + r * out_ld + dim, v, dims - dim);
}

template <class T, bool GRADIENT>
struct RowsWalk : RowsShared {
  static constexpr int RJ = 1;  // 16 rows of a wave
  static constexpr bool kGradient = GRADIENT, kInfo = false;
  const T *table;
  int64_t table_ld;
  T *out;
  int64_t out_ld;
  int32_t dims;

  struct Held {
    int label[RJ];
    float top[RJ], m[RJ], s[RJ], lost[RJ], inv;  // top: the largest product; m: what the sums are relative to
  } held;

  __device__ __forceinline__ void begin(int r0, int nx, int lane) {
    held.inv = logit_scale(exps);
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      const int r = r0 + j * 16 + lane % 16;
      held.label[j] = r < nx ? row.label(r) : -1;
      held.top[j] = held.m[j] = kLowest;
      held.s[j] = held.lost[j] = 0.f;
    }
  }

  __device__ __forceinline__ float exponent_of_one() const { return fminf(held.inv * c, 3e38f); }
  // The sums relative to another m.
  template <int FD>
  __device__ __forceinline__ void rescale(f32x4t (&o)[FD][RJ], int j, float m, float k) {
    const float f = __builtin_amdgcn_exp2f((held.m[j] - m) * k);
    held.s[j] *= f;
    held.lost[j] *= f;
    if constexpr (GRADIENT)
#pragma unroll
      for (int d = 0; d < FD; ++d) o[d][j] *= f;
    held.m[j] = m;
  }

  template <bool EDGE, int FD>
  __device__ __forceinline__ void transform(f32x4t (&z)[4][RJ], f32x4t (&o)[FD][RJ], const char *, int first, int ny,
                                            int lane) {
    // (m and z of the products as they are, scaled; probabilities times 2^14)
    const float k = exponent_of_one();
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      float top = held.top[j];
      const int mine = held.label[j] - first - 4 * (lane / 16);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (__any(static_cast<uint32_t>(mine - i * 16) < 4u))  // (most blocks of 16 classes hold none of the labels)
#pragma unroll
          for (int e = 0; e < 4; ++e) z[i][j][e] = mine == i * 16 + e ? -__builtin_inff() : z[i][j][e];
      if constexpr (EDGE)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            z[i][j][e] = first + i * 16 + 4 * (lane / 16) + e < ny ? z[i][j][e] : -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, z[i][j][e]);
      top = held.top[j] = max_of_four(top);
      // m follows when a term would pass 2^15, not at every new largest logit: with logits that rise from tile to tile
      // each would cost the sums two roundings.
      const bool follow = (top - held.m[j]) * k > 1.f;
      if (__any(follow)) {
        const float m = follow ? top : held.m[j];
        rescale<FD>(o, j, m, k);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i][j][e] - held.m[j], k, static_cast<float>(kDTerm)));
          z[i][j][e] = p;
        }
      // The tile's terms first, four sums of four, then what an addition to a long sum loses is kept for the next: a lane's
      // sum has a quarter of all the classes' terms, and equal ones are all rounded in one direction (2^20 classes of
      // equal logits but one: the loss 400 times as far off as all other roundings allow; 4096 x 128 x 131072 bf16
      // 322 and 339 us without it, 328 and 336 with it).
      f32x4t four = (z[0][j] + z[1][j]) + (z[2][j] + z[3][j]);
      const float term = ((four[0] + four[1]) + (four[2] + four[3])) - held.lost[j], sum = held.s[j] + term;
      held.lost[j] = (sum - held.s[j]) - term;
      held.s[j] = sum;
    }
  }

  template <int FD>
  __device__ __forceinline__ void finish(f32x4t (&o)[FD][RJ], const WalkArgs &a, int r0, int part, int lane) {
    const int nx = a.nx;
    const float back = ldexpf(1.f, -kDTerm - (exps ? exps->y : 0));
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      const int r = r0 + j * 16 + lane % 16;
      rescale<FD>(o, j, held.top[j], exponent_of_one());
      float s = held.s[j] * (1.f / (1 << kDTerm)), z = 0.f;
      // the label's logit, by one part
      const int label = held.label[j];
      if (part == 0 && label >= 0 && label < row.classes)
        z = own_product<FD / 2, sizeof(T) == 4 ? 2 : 1>(a, r, label, lane) * held.inv;
      const float m = held.m[j] == kLowest ? kLowest : held.m[j] * held.inv;
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      z += __shfl_xor(z, 16);
      z += __shfl_xor(z, 32);
      if (r >= nx) continue;
      if (part_sum) {
        if (lane < 16) {
          part_sum[static_cast<int64_t>(part) * nx + r] = float2{m, s};
          if (part == 0) own[r] = z;
        }
        if constexpr (GRADIENT)
#pragma unroll
          for (int f = 0; f < FD; ++f)
            *reinterpret_cast<f32x4t *>(part_out + (static_cast<int64_t>(part) * nx + r) * (FD * 16) + f * 16 +
                                        4 * (lane / 16)) = o[f][j];
        continue;
      }
      const float w = row.weight(r);
      const RowEnd e = end_row(m, s, z, label, row.classes, w, c, inv_t);
      if (lane < 16) {
        if (loss) loss[r] = e.loss;
        if (stats) stats[r] = float4{e.big, e.total, e.missing, 0.f};
      }
      if constexpr (GRADIENT)
#pragma unroll
        for (int f = 0; f < FD; ++f)
          put_features<T>(*this, e, w, label, r, f * 16 + 4 * (lane / 16), o[f][j], back, table, table_ld, out,
                          out_ld, dims);
    }
  }
};

// What a row's joined sums give: loss, stats, and four dims of d_features.
template <class T>
__device__ __forceinline__ void put_row(const RowsShared &g, int r, int dim, float m, float s, f32x4t sum, const T *table,
                                        int64_t table_ld, T *out, int64_t out_ld, int32_t dims) {
  const int label = g.row.label(r);
  const float w = g.row.weight(r);
  const RowEnd e = end_row(m, s, g.own[r], label, g.row.classes, w, g.c, g.inv_t);
  if (dim == 0) {
    if (g.loss) g.loss[r] = e.loss;
    if (g.stats) g.stats[r] = float4{e.big, e.total, e.missing, 0.f};
  }
  if (out)
    put_features<T>(g, e, w, label, r, dim, sum, ldexpf(1.f, -kDTerm - (g.exps ? g.exps->y : 0)), table, table_ld, out,
                    out_ld, dims);
}

// Joins the parts of a row. Few of them: DP / 4 threads a row take them one after another, four dims a thread. (So
// and by a block a row, us: 2 parts of 30000 rows of 32 dims 7.7 and 46, 8 of 8000 of 64 dims 10.4 and 15.2, 16 of
// 4096 14.8 and 9.8, 32 of 2000 25.8 and 7.6.)
constexpr int kFewParts = 8;

template <class T, int DP>
__global__ __launch_bounds__(256) void walk_join_few_kernel(RowsShared g, int32_t rows, int32_t parts, const T *table,
                                                           int64_t table_ld, T *out, int64_t out_ld, int32_t dims) {
  constexpr int lanes = DP / 4, per = 256 / lanes;
  const int r = static_cast<int>(blockIdx.x) * per + threadIdx.x / lanes, at = threadIdx.x % lanes;
  if (r >= rows) return;
  float m = kLowest;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, g.part_sum[p * static_cast<int64_t>(rows) + r].x);
  float s = 0.f;
  f32x4t sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const int64_t row = p * static_cast<int64_t>(rows) + r;
    const float2 v = g.part_sum[row];
    const float f = __builtin_amdgcn_exp2f((v.x - m) * g.c);
    s += v.y * f;
    if (out) sum += *reinterpret_cast<const f32x4t *>(g.part_out + row * DP + at * 4) * f;
  }
  put_row<T>(g, r, at * 4, m, s, sum, table, table_ld, out, out_ld, dims);
}

// More of them: a block a row, whose threads take parts side by side (one after another, 340 parts of
// three rows took 47 us), four dims a thread.
template <class T, int DP>
__global__ __launch_bounds__(256) void walk_join_kernel(RowsShared g, int32_t rows, int32_t parts, const T *table,
                                                       int64_t table_ld, T *out, int64_t out_ld, int32_t dims) {
  constexpr int lanes = DP / 4, slices = 256 / lanes;
  __shared__ float room[8];
  __shared__ f32x4t shares[slices][lanes];
  const int64_t r = blockIdx.x;
  const int at = threadIdx.x % lanes, slice = threadIdx.x / lanes;
  float m = kLowest;
  for (int p = threadIdx.x; p < parts; p += 256) m = fmaxf(m, g.part_sum[p * static_cast<int64_t>(rows) + r].x);
#pragma unroll
  for (int x = 1; x < 64; x *= 2) m = fmaxf(m, __shfl_xor(m, x));
  if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = m;
  __syncthreads();
  m = fmaxf(fmaxf(room[0], room[1]), fmaxf(room[2], room[3]));
  float s = 0.f;
  for (int p = threadIdx.x; p < parts; p += 256) {
    const float2 v = g.part_sum[p * static_cast<int64_t>(rows) + r];
    s += v.y * __builtin_amdgcn_exp2f((v.x - m) * g.c);
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) s += __shfl_xor(s, x);
  if (threadIdx.x % 64 == 0) room[4 + threadIdx.x / 64] = s;
  if (out) {
    f32x4t sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = slice; p < parts; p += slices) {
      const int64_t row = p * static_cast<int64_t>(rows) + r;
      const float f = __builtin_amdgcn_exp2f((g.part_sum[row].x - m) * g.c);
      sum += *reinterpret_cast<const f32x4t *>(g.part_out + row * DP + at * 4) * f;
    }
    shares[slice][at] = sum;
  }
  __syncthreads();
  if (slice != 0) return;
  s = (room[4] + room[5]) + (room[6] + room[7]);
  f32x4t sum{0.f, 0.f, 0.f, 0.f};
  if (out)
    for (int k = 0; k < slices; ++k) sum += shares[k][at];
  put_row<T>(g, static_cast<int>(r), at * 4, m, s, sum, table, table_ld, out, out_ld, dims);
}

// The walk over the rows: classes are the items x. d is held times 2^14 T w / 2^top, top being the
// largest weight's exponent.
template <class T, int RJ>
struct TableWalk {
  static constexpr bool kGradient = true, kInfo = true;
  const Exponents *exps;
  RowInfo row;
  float c;
  const float4 *stats;
  GradScale scale;
  T *out;
  int64_t out_ld;
  int32_t dims;
  float *slabs;    // [part][classes][slab_ld], nullable
  int32_t slab_ld;

  float inv, raw;  // inv: of a product, times log2(e) / T
  int top, c0;

  __device__ __forceinline__ void begin(int r0, int, int) {
    c0 = r0;
    raw = 1.f / logit_scale(exps);
    inv = fminf(logit_scale(exps) * c, 3e38f);
    top = exps ? exps->w : 0;
  }
  // Of each row of a tile: m, what its probabilities are multiplied with (0: the row does not count), the
  // label's d, the label.
  __device__ __forceinline__ void put_info(char *info, int first, int n) const {
    if (threadIdx.x >= kWalkItems) return;
    const int r = first + threadIdx.x;
    float4 v{0.f, 0.f, 0.f, __builtin_bit_cast(float, -1)};
    if (r < n) {
      const float w = row.weight(r);
      const int label = row.label(r);
      if (label >= 0 && w != 0.f) {
        const float4 st = stats[r];
        float f = __builtin_isfinite(w) ? ldexpf(w, kDTerm - top) : w;
        if (label >= row.classes) f = __builtin_nanf("");
        v = float4{st.x * raw, f / st.y, -f * st.z, __builtin_bit_cast(float, label)};
      }
    }
    *reinterpret_cast<float4 *>(info + threadIdx.x * 16) = v;
  }

  template <bool, int FD>
  __device__ __forceinline__ void transform(f32x4t (&z)[4][RJ], f32x4t (&)[FD][RJ], const char *info, int, int, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 v = *reinterpret_cast<const float4 *>(info + (i * 16 + 4 * (lane / 16) + e) * 16);
        const int label = __builtin_bit_cast(int, v.w);
#pragma unroll
        for (int j = 0; j < RJ; ++j) {
          float d = __builtin_amdgcn_exp2f((z[i][j][e] - v.x) * inv) * v.y;
          d = label == c0 + j * 16 + lane % 16 ? v.z : d;
          z[i][j][e] = v.y == 0.f ? 0.f : d;
        }
      }
  }

  template <int FD>
  __device__ __forceinline__ void finish(f32x4t (&o)[FD][RJ], const WalkArgs &a, int r0, int part, int lane) const {
    const int nx = a.nx;
    const Exponents e = exps ? *exps : Exponents{};
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      const int r = r0 + j * 16 + lane % 16;
      if (r >= nx) continue;
#pragma unroll
      for (int f = 0; f < FD; ++f) {
        const int d = f * 16 + 4 * (lane / 16);
        if (d >= dims) continue;
        if (slabs) {
          *reinterpret_cast<f32x4t *>(slabs + (static_cast<int64_t>(part) * nx + r) * slab_ld + d) = o[f][j];
        } else {
          float v[4];
          bool none;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = scale(o[f][j][k], r, e, none);
          store_four<T>(out + r * out_ld + d, v, dims - d);
        }
      }
    }
  }
};

}  // namespace tmnn_hip
