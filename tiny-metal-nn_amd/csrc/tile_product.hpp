// tile_product.hpp -- matrix products out[r][c] = sum_k x[r][k] y[c][k] on the
// matrix cores, one tile of the output a block, with what happens to a finished tile
// left to an epilogue. 16-bit floating point or e4m3, sums in fp32.
//
// The tile's steps of k (128 bytes of each row) pass through LDS in a ring of stages, loaded
// straight from memory without registers in between. One barrier a step: when it is passed, a
// stage has arrived and another is free for the next load. An operand whose k is contiguous lies in
// LDS as rows of a step's bytes; one whose k goes from row to row (a transposed operand) as rows of the
// tile's width, read with the transposing LDS loads, so that no transposed copy of
// it is ever made. Both lie swizzled: by the counters no two lanes of a read meet in a bank.
//
// 16-bit products reach 1.2 to 1.3 PFLOP/s, 8-bit ones with scales 1.7 to 1.9. A tile of 256 x 256 takes 64 KB for 8.4
// MFLOP of 16-bit products, so 9 to 10 TB/s pass from the L2 into LDS over the chip, 1.7 us a step; with the loads
// left out (and with them the data, which lowers the power too) the loop runs at 1.56 to 1.86 PFLOP/s. It is not their
// latency: with a ring of five half stages, which gives a load one to two steps to arrive, the times were the same
// (4096 x 2048 x 131072 bf16, all products 7.37 and 7.46 ms). Half steps of 64 bytes in five stages were slower: half a
// cache line a row, and a barrier for half the products.
//
// Layout of a result: lane l of a 16 x 16 block holds row r = l % 16, columns
// c = 4 (l / 16) .. + 3: y is the matrix instruction's first operand.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tile_args.hpp"

namespace tmnn_hip {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4t __attribute__((ext_vector_type(4)));
typedef int32_t i32x4t __attribute__((ext_vector_type(4)));
typedef int32_t i32x8t __attribute__((ext_vector_type(8)));

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
  static constexpr int KB = 128, KN = KB / E::bytes;  // of a step: bytes, elements
  static constexpr int WC = WC_, WR = WR_, FC = FC_, FR = FR_, NS = NS_;
  static constexpr bool XT = XT_, YT = YT_;
  static constexpr int kWaves = WC * WR, kThreads = kWaves * 64;
  static constexpr int BC = WC * FC * 16, BR = WR * FR * 16;
  // (8-bit operands: and 64 words a wave, the scales of its rows)
  static constexpr int kStage = (BC + BR) * KB + (E::bytes == 1 ? kWaves * 256 : 0);
  static constexpr int kLds = NS * kStage;
  static constexpr int QY = BC * KB / 1024 / kWaves, QX = BR * KB / 1024 / kWaves;  // loads of a thread in a stage
  static_assert(BC * KB / 1024 % kWaves == 0 && BR * KB / 1024 % kWaves == 0, "every wave loads as much");
  static constexpr int kLoads = QX + QY + (E::bytes == 1 ? 1 : 0);
  static_assert(NS >= 2 && (NS - 1) * kLoads < 64 && kLds <= 160 * 1024, "");
  static_assert(!(XT || YT) || E::bytes == 2, "the transposing loads take 16-bit elements");
};

extern __shared__ __align__(1024) char tile_lds[];

__device__ __forceinline__ uint32_t lds_address(const char *p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char *)p));
}

// Which 16 bytes of a row lie at a place in LDS: two rows of 128 bytes fill the 64 banks, and the ones
// beside them have their chunks elsewhere.
__device__ __forceinline__ int swizzle_row(int row) { return (row >> 1) & 7; }
// The same for a transposed operand, in pairs of chunks: a transposing read takes 32 bytes of
// rows k .. k + 3 and k + 8 .. k + 11 at a time.
__device__ __forceinline__ int swizzle_k(int k, int chunks) {
  return 2 * (((k & 3) | ((k >> 1) & 4)) & (chunks / 2 - 1));
}

// One thread's loads of one operand's part of a stage: B rows (columns) of the tile. What changes from
// step to step is in scalar registers: the base and how much of k is left.
template <class S, int B, bool T, int Q>
struct TileLoad {
  static constexpr int kChunks = T ? B / 8 : S::KB / 16, kRows = 64 / kChunks;  // of a row; rows of a load
  static constexpr int kEach = S::kWaves * kRows;  // rows from one load of a thread to its next
  static_assert(kEach % 16 == 0, "its places are swizzled alike");
  uint32_t at;      // byte offset of its first load from the step's base
  uint32_t each;    // bytes from one load to the next
  int32_t place;    // of the thread in k: bytes (contiguous k) or rows of its first load
  i32x4t rsrc;
  int64_t advance;
  int32_t left;     // of k, bytes or rows, from the step on

  __device__ __forceinline__ void begin(const Operand &o, int first, int wave, int lane) {
    const int row = wave * kRows + lane / kChunks;
    if constexpr (T) {
      const int c = 16 * ((lane % kChunks) ^ swizzle_k(row, kChunks));
      place = row;
      at = first * 2 + c < o.bytes ? row_offset(o, row) + c : kOutside;
      rsrc[2] = 0x7fffffff;
    } else {
      place = 16 * ((lane % kChunks) ^ swizzle_row(row));
      at = row_offset(o, row) + place;
      // (rows past the last one lie past the buffer's end)
      rsrc[2] = tile_bytes(o, first, B);
    }
    each = load_step(o, kEach);
    advance = T ? S::KN * o.ld : S::KB;
    rsrc[3] = 0x00020000;
  }
  // To step `st` of a plane.
  __device__ __forceinline__ void seek(const Operand &o, int first, int pl, int st) {
    const char *b = o.base + (T ? first * 2 : first * o.ld) + pl * o.plane + st * advance;
    rsrc[0] = static_cast<int32_t>(reinterpret_cast<uintptr_t>(b));
    rsrc[1] = static_cast<int32_t>((reinterpret_cast<uintptr_t>(b) >> 32) & 0xffff);
    left = (T ? o.rows : o.bytes) - st * (T ? S::KN : S::KB);
  }
  __device__ __forceinline__ void next() {
    const uint64_t b = (static_cast<uint64_t>(static_cast<uint32_t>(rsrc[1])) << 32 | static_cast<uint32_t>(rsrc[0])) + advance;
    rsrc[0] = static_cast<int32_t>(b);
    rsrc[1] = static_cast<int32_t>(b >> 32);
    left -= T ? S::KN : S::KB;
  }
  // Load q of the step to LDS, from `to` on (the wave's first place of the operand).
  __device__ __forceinline__ void load(int q, uint32_t to) const {
    const uint32_t off = place + (T ? q * kEach : 0) < left ? at + q * each : kOutside;
    // (nothing here is an output: the data goes to LDS, and the main loop waits for it)
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :
        : "s"(to + q * S::kWaves * 1024), "v"(off), "s"(rsrc)
        : "memory");
  }
};

// All of a wave's own loads from LDS, and of its loads into it all but the last `n`, are done; then
// all waves'. (The builtin, unlike inline assembly, is seen by the compiler, which
// then needs no wait of its own before the fragments are used.)
template <int n>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((n & 15) | 7 << 4 | 0 << 8 | (n >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

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
  return *reinterpret_cast<const V *>(tile + row * 128 + ((chunk + lane / 16) ^ swizzle_row(row)) * 16);
}

// What a step multiplies: 16-bit operands. The fragments of the next 64 bytes are on their
// way from LDS while these are multiplied.
template <class S>
struct PlainSteps {
  static constexpr bool kAhead = S::FC * S::FR >= 16;  // (small tiles wait for memory)
  static constexpr bool kStream = false;
  typedef Fragment<typename S::E> M;
  typedef typename M::V V;
  struct Held {
    V y[S::FC], x[S::FR];
  };
  template <class A>
  __device__ __forceinline__ PlainSteps(const A &, const TileArgs &, int, int, int, int) {}
  __device__ __forceinline__ void load(int, bool, uint32_t) const {}
  __device__ __forceinline__ void before(int) {}
  __device__ __forceinline__ void arrived(int, int) const {}
  __device__ __forceinline__ void read_x(Held &f, const char *y, int ks, int j, int wr, int lane) const {
    const char *x = y + S::BC * S::KB;
    const int at = (wr * S::FR + j) * 16;
    if constexpr (S::XT)
      f.x[j] = read_transposed<V>(x, S::BR, at, ks, lane);
    else
      f.x[j] = read_row<V>(x, at + lane % 16, ks * 4, lane);
  }
  __device__ __forceinline__ void read_y(Held &f, const char *y, int ks, int i, int wc, int lane) const {
    const int at = (wc * S::FC + i) * 16;
    if constexpr (S::YT)
      f.y[i] = read_transposed<V>(y, S::BC, at, ks, lane);
    else
      f.y[i] = read_row<V>(y, at + lane % 16, ks * 4, lane);
  }
  // Part g of `of` of a fragment set, and of the products.
  __device__ __forceinline__ void read(Held &f, const char *y, int ks, int g, int of, int wc, int wr, int lane) const {
#pragma unroll
    for (int j = 0; j < S::FR; ++j)
      if (j * of / S::FR == g) read_x(f, y, ks, j, wr, lane);
#pragma unroll
    for (int i = 0; i < S::FC; ++i)
      if (i * of / S::FC == g) read_y(f, y, ks, i, wc, lane);
  }
  __device__ __forceinline__ void multiply(f32x4t (&acc)[S::FC][S::FR], const Held &f, int g, int of) const {
#pragma unroll
    for (int i = 0; i < S::FC; ++i)
      if (i * of / S::FC == g)
#pragma unroll
        for (int j = 0; j < S::FR; ++j) acc[i][j] = M::mul(f.y[i], f.x[j], acc[i][j]);
  }
  __device__ __forceinline__ void step(f32x4t (&acc)[S::FC][S::FR], const char *y, int, int wc, int wr, int lane) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      Held f;
      read(f, y, ks, 0, 1, wc, wr, lane);
      multiply(acc, f, 0, 1);
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

  const uint32_t lds_first = __builtin_amdgcn_readfirstlane(lds_address(tile_lds));
  const uint32_t lds = lds_first + wave * 1024;
  Steps steps(sa, a, first_c + wc * S::FC * 16, first_r + wr * S::FR * 16, wave, lane);

  const int total = a.steps * a.pairs;
  const int from = p.part * a.part_steps, to = min(total, from + a.part_steps);
  int next = from, pair = from / a.steps, st = from - pair * a.steps;
  TileLoad<S, S::BC, S::YT, S::QY> ly;
  TileLoad<S, S::BR, S::XT, S::QX> lx;
  ly.begin(a.y, first_c, wave, lane);
  lx.begin(a.x, first_r, wave, lane);
  auto seek = [&] {
    ly.seek(a.y, first_c, a.pairs == 3 && pair == 1, st);
    lx.seek(a.x, first_r, pair > 0 && pair == a.pairs - 1, st);
  };
  seek();
  // Loads the next step into a stage (zeros, without touching memory, after the last one), with
  // `between` after each load.
  auto load = [&](int stage, auto between) {
    const uint32_t at = lds + stage * S::kStage;
    if (next >= to) ly.left = lx.left = 0;
    steps.load(next, next < to, lds_first + stage * S::kStage + (S::BC + S::BR) * S::KB + wave * 256);
#pragma unroll
    for (int q = 0; q < S::QY + S::QX; ++q) {
      if (q < S::QY)
        ly.load(q, at);
      else
        lx.load(q - S::QY, at + S::BC * S::KB);
      between(q);
    }
    ++next;
    ly.next();
    lx.next();
    if (++st == a.steps && next < to) {
      st = 0;
      ++pair;
      seek();
    }
  };
  auto nothing = [](int) {};

  f32x4t acc[S::FC][S::FR];
#pragma unroll
  for (int i = 0; i < S::FC; ++i)
#pragma unroll
    for (int j = 0; j < S::FR; ++j) acc[i][j] = f32x4t{0.f, 0.f, 0.f, 0.f};

  int now = 0;
  auto next_stage = [](int s) { return s + 1 == S::NS ? 0 : s + 1; };
  if constexpr (Steps::kAhead) {
    // All stages on their way. Fragments are read 64 bytes of k ahead of their products; when the barrier
    // in a step's last half is passed, all waves hold that half in registers, so its stage is
    // free, and the next step has arrived.
    typename Steps::Held f[2];
#pragma unroll
    for (int s = 0; s < S::NS; ++s) load(s, nothing);
    wait_and_meet<(S::NS - 1) * S::kLoads>();
    steps.read(f[0], tile_lds, 0, 0, 1, wc, wr, lane);
    auto first = [&](typename Steps::Held &held, typename Steps::Held &coming) {
      const char *y = tile_lds + now * S::kStage;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        steps.read(coming, y, 1, g, 4, wc, wr, lane);
        steps.multiply(acc, held, g, 4);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto last = [&](typename Steps::Held &held, typename Steps::Held &coming) {
      wait_and_meet<(S::NS - 2) * S::kLoads>();
      const int free = now;
      now = next_stage(now);
      const char *y = tile_lds + now * S::kStage;
      // Loads, reads and products take turns: a wave that issues its loads in a row waits for the
      // memory pipeline with the matrix cores idle.
      load(free, [&](int q) {
        steps.read(coming, y, 0, q, S::kLoads, wc, wr, lane);
        steps.multiply(acc, held, q, S::kLoads);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    for (int k = from; k < to; ++k) {
      first(f[0], f[1]);
      last(f[1], f[0]);
    }
  } else if constexpr (Steps::kStream) {
    // The classes' fragments go one by one, one ahead; the barrier is before the last one's products, when
    // all of the step is in registers.
    // Each of the rows' is read anew behind its last product.
    typename Steps::Rows x;
    i32x8t c[2];
#pragma unroll
    for (int s = 0; s < S::NS; ++s) load(s, nothing);
    steps.before(from);
    wait_and_meet<(S::NS - 1) * S::kLoads>();
    steps.arrived(0, from);
#pragma unroll
    for (int j = 0; j < S::FR; ++j) steps.read(x, tile_lds, from, j, wr, lane);
    c[0] = steps.classes(tile_lds, 0, wc, lane);
    for (int k = from; k < to; ++k) {
      const char *y = tile_lds + now * S::kStage;
      steps.ready(x);
#pragma unroll
      for (int i = 0; i < S::FC - 1; ++i) {
        c[(i + 1) % 2] = steps.classes(y, i + 1, wc, lane);
#pragma unroll
        for (int j = 0; j < S::FR; ++j) steps.multiply(acc, x, c[i % 2], i, j);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_and_meet<(S::NS - 2) * S::kLoads>();
      load(now, nothing);
      now = next_stage(now);
      steps.arrived(now, k + 1);
      y = tile_lds + now * S::kStage;
      static_assert(S::FC % 2 == 0, "");
      c[0] = steps.classes(y, 0, wc, lane);
#pragma unroll
      for (int j = 0; j < S::FR; ++j) {
        steps.multiply(acc, x, c[1], S::FC - 1, j);
        steps.read(x, y, k + 1, j, wr, lane);
        __builtin_amdgcn_sched_barrier(0);
      }
      steps.before(min(k + 1, to - 1));
    }
  } else {
#pragma unroll
    for (int s = 0; s < S::NS - 1; ++s) load(s, nothing);
    int free = S::NS - 1;
    for (int k = from; k < to; ++k) {
      // this step's stage has arrived (later ones may be on their way), and this wave's
      // reads of the stage before it are done
      wait_and_meet<(S::NS - 2) * S::kLoads>();
      steps.before(k);
      steps.arrived(now, k);
      load(free, nothing);
      const char *y = tile_lds + now * S::kStage;
      steps.step(acc, y, k, wc, wr, lane);
      free = now;
      now = next_stage(now);
    }
  }
  wait_and_meet<0>();
  epi.template finish<S>(a, p, acc, first_c + wc * S::FC * 16, first_r + wr * S::FR * 16, wc, wr, lane);
}

}  // namespace tmnn_hip
