// tile_product.hpp -- matrix products out[r][c] = sum_k x[r][k] y[c][k] on the
// matrix cores, one tile of the output a block, with what happens to a finished tile
// left to an epilogue. 16-bit floating point or e4m3, sums in fp32.
//
// The tile's steps of k (128 bytes of each row: 64 16-bit elements, 128 8-bit ones) pass through
// LDS in a ring of stages, loaded straight from memory without registers in between. One
// barrier a step: when it is passed, the step's stage has arrived and the stage before
// it is free for the next load. An operand whose k is contiguous lies in LDS as
// rows of 128 bytes; one whose k goes from row to row (a transposed operand) as 64 rows of the
// tile's width, read with the transposing LDS loads, so that no transposed copy of
// it is ever made. Both lie swizzled, so that neither reading wave meets a bank twice.
//
// Layout of a result: lane l of a 16 x 16 block holds row r = l % 16, columns
// c = 4 (l / 16) .. + 3: y is the matrix instruction's first operand.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tmnn_hip {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4t __attribute__((ext_vector_type(4)));
typedef int32_t i32x4t __attribute__((ext_vector_type(4)));
typedef int32_t i32x8t __attribute__((ext_vector_type(8)));

constexpr int kStepBytes = 128;  // of k, in a row of a stage

// One operand. Rows of it are the output's rows (x) or columns (y), or, of a transposed
// one, the values of k. Everything of it that a tile reads starts at multiples of 16 bytes.
struct Operand {
  const char *base;
  int64_t ld;      // bytes from row to row: below 2^23
  int64_t plane;   // bytes from plane to plane (operands in two terms)
  int32_t rows;    // rows that exist
  int32_t bytes;   // bytes of a row that exist, a multiple of 16; what lies beyond counts as 0
};

struct TileArgs {
  Operand x, y;
  int32_t rows, cols;          // of the output
  int32_t tiles_r, tiles_c, parts;
  int32_t steps;               // of k, in one pair of planes
  int32_t pairs;               // 1: one plane each; 3: high x high, high x low, low x high
  int32_t part_steps;          // steps of one part, counted over all pairs
};

// A block's tile and part. Blocks go to the chip's eight dies in turn, each with an L2 of
// its own: every die takes a contiguous eighth, in columns of four tiles.
struct TilePlace {
  int32_t r, c, part;
};

__device__ __forceinline__ TilePlace tile_place(const TileArgs &a) {
  const uint32_t n = static_cast<uint32_t>(a.tiles_r) * a.tiles_c * a.parts;
  const uint32_t die = blockIdx.x % 8, at = blockIdx.x / 8, share = n / 8, rest = n % 8;
  uint32_t id = die * share + (die < rest ? die : rest) + at;
  TilePlace p;
  const uint32_t tiles = static_cast<uint32_t>(a.tiles_r) * a.tiles_c;
  p.part = id / tiles;
  id -= p.part * tiles;
  const uint32_t per = 4u * a.tiles_c, group = id / per;
  const uint32_t first = group * 4, high = min(4u, a.tiles_r - first);
  id -= group * per;
  p.c = id / high;
  p.r = first + (id - p.c * high);
  return p;
}

struct F16 {
  static constexpr int bytes = 2;
};
struct BF16 {
  static constexpr int bytes = 2;
};
struct F8 {
  static constexpr int bytes = 1;
};

// WC x WR waves of FC x FR blocks of 16 x 16; NS stages; XT, YT: transposed operands.
template <class E_, int WC_, int WR_, int FC_, int FR_, int NS_, bool XT_, bool YT_>
struct TileShape {
  typedef E_ E;
  static constexpr int WC = WC_, WR = WR_, FC = FC_, FR = FR_, NS = NS_;
  static constexpr bool XT = XT_, YT = YT_;
  static constexpr int kWaves = WC * WR, kThreads = kWaves * 64;
  static constexpr int BC = WC * FC * 16, BR = WR * FR * 16;
  // (8-bit operands: and 64 words a wave, the scales of its rows)
  static constexpr int kStage = (BC + BR) * kStepBytes + (E::bytes == 1 ? kWaves * 256 : 0);
  static constexpr int kLds = NS * kStage;
  static constexpr int QY = BC / 8 / kWaves, QX = BR / 8 / kWaves;  // loads of a thread in a stage
  static_assert(BC / 8 % kWaves == 0 && BR / 8 % kWaves == 0, "every wave loads as much");
  static constexpr int kLoads = QX + QY + (E::bytes == 1 ? 1 : 0);
  static_assert(NS >= 2 && (NS - 2) * kLoads < 64 && kLds <= 160 * 1024, "");
  static_assert(!(XT || YT) || E::bytes == 2, "the transposing loads take 16-bit elements");
};

extern __shared__ __align__(1024) char tile_lds[];

__device__ __forceinline__ uint32_t lds_address(const char *p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char *)p));
}

// Which 16 bytes of a row of 128 lie at a place in LDS: rows r and r + 1 fill the 64 banks, the
// pairs of rows beside them have their chunks elsewhere.
__device__ __forceinline__ int swizzle_row(int row) { return (row >> 1) & 7; }
// The same for a transposed operand, in pairs of chunks: a transposing read takes 32 bytes of
// rows k .. k + 3 and k + 8 .. k + 11 at a time.
__device__ __forceinline__ int swizzle_k(int k, int chunks) {
  return 2 * (((k & 3) | ((k >> 1) & 4)) & (chunks / 2 - 1));
}

constexpr uint32_t kOutside = 0x80000000u;  // an offset past the end of every buffer: loads give 0

// One thread's loads of one operand's part of a stage: B rows (columns) of the tile.
template <class S, int B, bool T, int Q>
struct TileLoad {
  uint32_t at[Q];  // byte offsets from the step's base
  uint32_t chunk;  // of k, in a row (contiguous k): bytes from the step's first
  const char *base;
  int64_t advance, plane;
  int64_t left;    // bytes of k (contiguous), or rows of k, that exist

  __device__ __forceinline__ void begin(const Operand &o, int first, int wave, int lane) {
    plane = o.plane;
    if constexpr (!T) {
      const int row = wave * 8 + lane / 8;
      chunk = 16 * ((lane % 8) ^ swizzle_row(row));
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int r = q * S::kWaves * 8 + row;
        at[q] = first + r < o.rows ? static_cast<uint32_t>(r * o.ld) + chunk : kOutside;
      }
      base = o.base + first * o.ld;
      advance = kStepBytes;
      left = o.bytes;
    } else {
      constexpr int chunks = B / 8, rows = 64 / chunks;  // of a row; rows that one load takes
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int k = (q * S::kWaves + wave) * rows + lane / chunks;
        const int c = 16 * ((lane % chunks) ^ swizzle_k(k, chunks));
        at[q] = first * 2 + c < o.bytes ? static_cast<uint32_t>(k * o.ld) + c : kOutside;
      }
      chunk = 0;
      base = o.base + first * 2;
      advance = 64 * o.ld;
      left = o.rows;
    }
  }

  // Loads step `st` of plane `pl` into LDS at `to` (the wave's first place of the operand's part).
  __device__ __forceinline__ void step(int pl, int st, bool exists, uint32_t to, int64_t ld) const {
    const char *b = base + pl * plane + st * advance;
    i32x4t rsrc;
    rsrc[0] = static_cast<int32_t>(reinterpret_cast<uintptr_t>(b));
    rsrc[1] = static_cast<int32_t>((reinterpret_cast<uintptr_t>(b) >> 32) & 0xffff);
    rsrc[3] = 0x00020000;
    uint32_t most = 0;
    if constexpr (!T) {
      const int64_t l = exists ? left - static_cast<int64_t>(st) * kStepBytes : 0;
      most = static_cast<uint32_t>(l < 0 ? 0 : l < kStepBytes ? l : kStepBytes);
      rsrc[2] = 0x7fffffff;
    } else {
      const int64_t l = exists ? (left - static_cast<int64_t>(st) * 64) * ld : 0;
      rsrc[2] = static_cast<int32_t>(l < 0 ? 0 : l < 0x7fffffff ? l : 0x7fffffff);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const uint32_t off = T || chunk < most ? at[q] : kOutside;
      // (nothing here is an output: the data goes to LDS, and the main loop waits for it)
      asm volatile(
          "s_mov_b32 m0, %0\n\t"
          "s_nop 0\n\t"
          "buffer_load_dwordx4 %1, %2, 0 offen lds"
          :
          : "s"(to + q * S::kWaves * 1024), "v"(off), "s"(rsrc)
          : "memory", "m0");
    }
  }
};

// What a lane holds of 16 rows x 32 values of k.
template <class E>
struct Fragment;
template <>
struct Fragment<F16> {
  typedef f16x8 V;
  static __device__ __forceinline__ f32x4t mul(V y, V x, f32x4t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(y, x, c, 0, 0, 0);
  }
};
template <>
struct Fragment<BF16> {
  typedef bf16x8 V;
  static __device__ __forceinline__ f32x4t mul(V y, V x, f32x4t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, x, c, 0, 0, 0);
  }
};

// A transposed operand's fragment: k = 8 (lane / 16) + 0 .. 7 of ks * 32, column `col` + lane % 16.
template <class V>
__device__ __forceinline__ V read_transposed(const char *tile, int width, int col, int ks, int lane) {
  const int chunks = width / 8, t = lane % 16;
  union {
    s16x4 half[2];
    V v;
  } u;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = ks * 32 + 8 * (lane / 16) + 4 * h + t / 4;
    const int slot = (col / 8 + (t % 4) / 2) ^ swizzle_k(k, chunks);
    const char *p = tile + k * (2 * width) + slot * 16 + (t % 2) * 8;
    u.half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4 *)(__attribute__((address_space(3))) char *)p);
  }
  return u.v;
}

template <class V>
__device__ __forceinline__ V read_row(const char *tile, int row, int chunk, int lane) {
  return *reinterpret_cast<const V *>(tile + row * kStepBytes + ((chunk + lane / 16) ^ swizzle_row(row)) * 16);
}

// What a step multiplies: 16-bit operands.
template <class S>
struct PlainSteps {
  template <class A>
  __device__ __forceinline__ PlainSteps(const A &, const TileArgs &, int, int, int, int) {}
  __device__ __forceinline__ void load(int, bool, uint32_t) const {}
  __device__ __forceinline__ void before(int) {}
  __device__ __forceinline__ void step(f32x4t (&acc)[S::FC][S::FR], const char *y, const char *x, int, int wc,
                                       int wr, int lane) {
    typedef Fragment<typename S::E> M;
    typedef typename M::V V;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      V fy[S::FC], fx[S::FR];
#pragma unroll
      for (int j = 0; j < S::FR; ++j) {
        const int at = (wr * S::FR + j) * 16;
        if constexpr (S::XT)
          fx[j] = read_transposed<V>(x, S::BR, at, ks, lane);
        else
          fx[j] = read_row<V>(x, at + lane % 16, ks * 4, lane);
      }
#pragma unroll
      for (int i = 0; i < S::FC; ++i) {
        const int at = (wc * S::FC + i) * 16;
        if constexpr (S::YT)
          fy[i] = read_transposed<V>(y, S::BC, at, ks, lane);
        else
          fy[i] = read_row<V>(y, at + lane % 16, ks * 4, lane);
      }
#pragma unroll
      for (int i = 0; i < S::FC; ++i)
#pragma unroll
        for (int j = 0; j < S::FR; ++j) acc[i][j] = M::mul(fy[i], fx[j], acc[i][j]);
    }
  }
};

// Steps: how a step is multiplied (with scales that it loads). Epi: what becomes of the tile,
// called with the accumulators by all threads, LDS being free.
template <class S, class Steps, class Epi, class StepArgs>
__global__ __launch_bounds__(S::kThreads, S::kWaves == 8 ? 2 : 1) void tile_kernel(TileArgs a, StepArgs sa,
                                                                                  Epi epi) {
  const int lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wc = wave % S::WC, wr = wave / S::WC;
  const TilePlace p = tile_place(a);
  const int first_c = p.c * S::BC, first_r = p.r * S::BR;

  TileLoad<S, S::BC, S::YT, S::QY> ly;
  TileLoad<S, S::BR, S::XT, S::QX> lx;
  ly.begin(a.y, first_c, wave, lane);
  lx.begin(a.x, first_r, wave, lane);
  const uint32_t lds_first = __builtin_amdgcn_readfirstlane(lds_address(tile_lds));
  const uint32_t lds = lds_first + wave * 1024;
  Steps steps(sa, a, first_c + wc * S::FC * 16, first_r + wr * S::FR * 16, wave, lane);

  const int total = a.steps * a.pairs;
  const int from = p.part * a.part_steps, to = min(total, from + a.part_steps);
  int next = from, pair = from / a.steps, st = from - pair * a.steps;
  auto load = [&](int stage) {
    const bool exists = next < to;
    const uint32_t at = lds + stage * S::kStage;
    ly.step(pair == 1, st, exists, at, a.y.ld);
    lx.step(pair == 2, st, exists, at + S::BC * kStepBytes, a.x.ld);
    steps.load(next, exists, lds_first + stage * S::kStage + (S::BC + S::BR) * kStepBytes + wave * 256);
    ++next;
    if (++st == a.steps) {
      st = 0;
      ++pair;
    }
  };

  f32x4t acc[S::FC][S::FR];
#pragma unroll
  for (int i = 0; i < S::FC; ++i)
#pragma unroll
    for (int j = 0; j < S::FR; ++j) acc[i][j] = f32x4t{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int s = 0; s < S::NS - 1; ++s) load(s);
  int now = 0, free = S::NS - 1;
  for (int k = from; k < to; ++k) {
    // this step's stage has arrived (later ones may be on their way), and this wave's
    // reads of the stage before it are done
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S::NS - 2) * S::kLoads) : "memory");
    steps.before(k);
    load(free);
    const char *y = tile_lds + now * S::kStage;
    steps.step(acc, y, y + S::BC * kStepBytes, k, wc, wr, lane);
    free = now;
    now = now + 1 == S::NS ? 0 : now + 1;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  epi.template finish<S>(a, p, acc, first_c + wc * S::FC * 16, first_r + wr * S::FR * 16, wc, wr, lane);
}

}  // namespace tmnn_hip
