// head_plan.hpp -- what a call of the class head launches, as plain numbers: tiles, parts and pieces, which
// operand lies where, and the workspace. Plain C++: tests without a GPU read it too.
#pragma once

#include <stdint.h>

#include <algorithm>

#include "arg_types.hpp"
#include "tile_args.hpp"
#include "tmnn_hip.h"

namespace tmnn_hip {

constexpr int kScaleParts = 1024;  // most blocks that look for one operand's largest magnitude
constexpr int kExponentBytes = 16;
constexpr int kScaleBlock = 128;   // values of a scale of 8-bit operands
constexpr int kWalkItems = 64;     // items of a walk's tile in LDS
constexpr int kWalkWaves = 4;

inline int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
inline int64_t parts_of(int64_t n, int64_t of) { return (n + of - 1) / of; }

// ---- tiles --------------------------------------------------------------------------

enum Shape { kLarge, kWide, kMiddle, kFlat, kSmall };

struct Tiles {
  Shape shape;
  int32_t bc, br, r, c, parts, steps, part_steps;  // steps: of one pair of planes
};

constexpr int kUnits = 256;  // compute units

// What a tile's step of 128 bytes of k takes, in us, with one block on a unit and with two, and what a tile
// takes besides. All shapes of 16 bits are bound by the way from the L2 into LDS, 9 to 12 TB/s over the chip, so
// the larger the tile the less a product takes, and the smaller the less is left over at the edges. Measured
// (us): 515 x 1000 x 50021 fp16, logits and sums, Large 84 (588 tiles, 3 rounds), Wide 98 (980, 4), Middle 102
// (1955, 4), Flat 116 (3519, 7), Small 176 (6647, 13); 64 x 1024 x 32768 Wide 20, Middle 22, Flat 15, Small 15;
// 1 x 4096 x 131072 Wide 190, Middle 183, Flat 179, Small 176. 8-bit, 64 x 2048 x 65536 to fp32 Wide 45, Middle 44, Flat
// 32, Small 52; 777 x 1000 x 10007 to fp16 Large 30, Wide 35, Middle 29, Flat 41, Small 64; 256 x 2048 x 32768 to bf16
// Wide 36, Middle 37, Flat 64, Small 108.
struct StepTime {
  double one, two, besides;
};
constexpr StepTime kTimes[] = {{1.75, 0, 10}, {1.5, 0, 6}, {1.0, 1.6, 3}, {0.75, 1.04, 2}, {0.6, 0.85, 1.5}};
constexpr StepTime kTimes8[] = {{2.1, 0, 11}, {1.9, 0, 6}, {1.3, 1.7, 3}, {1.5, 1.9, 2}, {1.2, 1.6, 1.5}};
constexpr StepTime kTimes8Wide[] = {{0, 0, 0}, {2.5, 0, 6}, {1.9, 2.6, 3}, {1.5, 1.9, 2}, {1.2, 1.6, 1.5}};  // widened

// The shape, and parts of k where the epilogue allows them (sums in fp32 that a second kernel ends), that
// take the least time by these.
inline Tiles choose(int64_t rows, int64_t cols, int64_t k_bytes, int pairs, bool f8, bool large, bool small, bool split) {
  Tiles best{};
  double least = 1e300;
  for (const Shape s : {kLarge, kWide, kMiddle, kFlat, kSmall}) {
    if ((s >= kFlat && !small) || (s == kLarge && !large)) continue;
    Tiles t{};
    t.shape = s;
    t.bc = s <= kWide ? 256 : 128;
    t.br = s == kLarge ? 256 : s <= kMiddle ? 128 : s == kFlat ? 64 : 32;
    t.r = static_cast<int32_t>(parts_of(rows, t.br));
    t.c = static_cast<int32_t>(parts_of(cols, t.bc));
    t.steps = static_cast<int32_t>(parts_of(k_bytes, 128));
    const int64_t steps = static_cast<int64_t>(t.steps) * pairs, tiles = static_cast<int64_t>(t.r) * t.c;
    const StepTime &m = (!f8 ? kTimes : large ? kTimes8 : kTimes8Wide)[s];
    for (int64_t parts = 1; parts <= 64 && parts <= steps; ++parts) {
      if (parts > 1 && (!split || tiles * parts > 4 * kUnits || steps / parts < 4)) break;
      const int64_t part_steps = parts_of(steps, parts), blocks = tiles * parts;
      const bool two = m.two > 0 && blocks > kUnits;
      double time = static_cast<double>(parts_of(blocks, two ? 2 * kUnits : kUnits)) *
                    (static_cast<double>(part_steps) * (two ? m.two : m.one) + m.besides);
      if (parts > 1)  // parts are written and read again, by one more kernel
        time += 3 + static_cast<double>(parts) * static_cast<double>(rows) * static_cast<double>(cols) * 8 / 5e6;
      if (time < least) {
        least = time;
        t.part_steps = static_cast<int32_t>(part_steps);
        t.parts = static_cast<int32_t>(parts_of(steps, part_steps));
        best = t;
      }
    }
  }
  return best;
}

inline TileArgs tile_args(const Operand &x, const Operand &y, int64_t rows, int64_t cols, const Tiles &t,
                   int pairs) {
  TileArgs a{};
  a.x = x;
  a.y = y;
  a.rows = static_cast<int32_t>(rows);
  a.cols = static_cast<int32_t>(cols);
  a.tiles_r = t.r;
  a.tiles_c = t.c;
  a.parts = t.parts;
  a.steps = t.steps;
  a.pairs = pairs;
  a.part_steps = t.part_steps;
  return a;
}

// ---- class loss ---------------------------------------------------------------------------

// Bytes of the piece's d up to which more classes go into one piece: larger pieces mean fewer
// launches and fewer passes over the sums of d_features (4096 x 2048 x 131072 bf16: 8.16 ms with 64 MiB, 7.86 with
// 256, 7.82 with 1 GiB).
constexpr int64_t kPieceBytes = int64_t{256} << 20;

// What a call lays out, in which tiles it goes, and where in the workspace things are.
struct LossPlan {
  bool grad, sums, f32, scaled;      // scaled: operands in fp16 terms
  bool lay_x, lay_y, weighted;       // copies that are made
  int planes, pairs;                 // terms of the operands, products of them
  int planes_d, pairs_d;             // of d, and of the gradients' products
  int64_t k, ld;                     // elements of a laid-out row, and from row to row
  int64_t piece, k_d, ld_d;          // classes of a piece; elements of a row of d, and from row to row
  Tiles t_sums, t_d, t_x, t_y;       // logits for sums, for d; d_features, d_table
  int64_t slab_ld;
  bool slabs_x, slabs_y;
  // features of up to 128 dims: parts of the walks
  bool keep;                         // the logits, between the sums and d
  bool narrow, wide_t;
  int32_t blocks_r, tiles_r, parts_r, blocks_t, tiles_t, parts_t;
  int64_t at_part_sum, at_part_own, at_part_out;
  int64_t at_exps, at_most, at_x, at_w, at_y, at_sums, at_own, at_stats, at_z, at_d, at_slab_x, at_slab_y, bytes;
};

// Rows up to which d of fp16 inputs goes in two terms. (rows x 1000 x 50000, a call with one term and with two, us:
// 64 rows 166 and 190, 128 rows 182 and 219, 256 rows 225 and 299, 512 rows 358 and 476: few rows wait for memory.)
constexpr int64_t kFewRows = 128;

// Dims up to which the walks of narrow_kernel.hpp take a call. (By them and by products of tiles, with both gradients:
// 65536 x 128 x 1000 bf16 172 and 275 us, 4096 x 128 x 131072 bf16 755 and 1838, fp32 1522 and 3148, 64 x 128 x
// 131072 bf16 77 and 128. Beyond 128 dims a wave's accumulators do not fit.)
constexpr int64_t kNarrow = 128;

// Parts of a walk's tiles, where the items of one side alone make too few blocks: four blocks a unit, and
// four tiles a part at least. (Kernels of a call with both gradients, us. With two, four and eight blocks a unit: 512 x
// 64 x 262144 fp16 191, 188 and 188. With two, four and eight tiles: 4096 x 16 x 64 fp32 27, 31 and 36, 64 x 128 x
// 131072 bf16 84, 77 and 70, 1000 x 100 x 5000 fp32 79, 75 and 86.)
inline int32_t walk_parts(int64_t blocks, int64_t tiles) {
  int64_t parts = std::max<int64_t>(1, std::min<int64_t>(4 * kUnits / blocks, tiles / 4));
  return static_cast<int32_t>(parts_of(tiles, parts_of(tiles, parts)));
}

inline LossPlan plan_loss(const tmnn_class_loss_args &a, bool back) {
  LossPlan p{};
  const int64_t n = a.rows, v = a.classes, size = static_cast<int64_t>(dtype_size(a.dtype));
  p.grad = a.d_features || a.d_table;
  p.sums = !back;
  p.f32 = a.dtype == TMNN_DTYPE_F32;
  p.planes = p.f32 ? 2 : 1;
  p.pairs = p.f32 ? 3 : 1;
  // fp16 gradients hold as many bits as d in one term: over many rows its rounding adds as much error as theirs
  // (1.4 times it together), over few a row's largest d alone can add twice as much
  p.planes_d = p.f32 || (a.dtype == TMNN_DTYPE_F16 && n <= kFewRows) ? 2 : 1;
  p.pairs_d = p.f32 ? 3 : p.planes_d;
  p.narrow = a.dims <= kNarrow;
  p.k = up(a.dims, 64);
  p.ld = !p.narrow ? p.k : a.dims <= 32 ? 32 : a.dims <= 64 ? 64 : 128;
  // operands that lie well are read in place
  auto lies_well = [&](const void *ptr, int64_t stride, int64_t rows) {
    return size == 2 && aligned(ptr, 16) && (stride % 8 == 0 || rows <= 1) && a.dims % 8 == 0 &&
           stride * size < (1 << 23);
  };
  const bool x_well = lies_well(a.features, a.feature_stride, n), y_well = lies_well(a.table, a.table_stride, v);
  p.scaled = p.f32 || p.grad;
  const bool convert = p.narrow || p.f32 || (p.grad && a.dtype == TMNN_DTYPE_BF16);
  if (p.narrow) p.scaled = true;
  p.lay_x = convert || !x_well;
  p.lay_y = convert || !y_well;
  p.weighted = a.d_table != nullptr;
  int64_t at = 0;
  auto room = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  p.at_exps = room(kExponentBytes);
  p.at_most = room(3 * kScaleParts * 4);
  const int64_t x_bytes = n * p.ld * 2 * p.planes;
  if (p.lay_x) p.at_x = room(x_bytes);
  if (p.weighted) p.at_w = room(x_bytes);
  if (p.lay_y) p.at_y = room(v * p.ld * 2 * p.planes);
  if (p.narrow) {
    auto blocks = [](int64_t items, bool wide) {
      return static_cast<int32_t>(parts_of(items, kWalkWaves * (wide ? 32 : 16)));
    };
    p.blocks_r = blocks(n, false);
    p.tiles_r = static_cast<int32_t>(parts_of(v, kWalkItems));
    p.parts_r = walk_parts(p.blocks_r, p.tiles_r);
    if (p.sums && p.grad && !a.stats) p.at_stats = room(n * 16);
    if (p.parts_r > 1) {
      p.at_part_sum = room(n * p.parts_r * 8);
      p.at_part_own = room(n * 4);
      if (a.d_features) p.at_part_out = room(n * p.parts_r * p.ld * 4);
    }
    if (a.d_table) {
      // 32 classes a wave where that still makes four blocks a unit, and the walk is long enough (16 a wave and 32,
      // us: 4096 x 128 x 131072 bf16 415 and 352, fp32 838 and 730, 512 x 64 x 262144 fp16 91 and 83, 64 x 128 x
      // 1000000 bf16 169 and 182). Rows go 16 a wave: 262144 x 128 x 1000 fp16 261 and 280, 1048576 x 64 x 150
      // bf16 219 and 240.
      p.wide_t = v >= 4 * kUnits * kWalkWaves * 32 && n >= 512;
      p.blocks_t = blocks(v, p.wide_t);
      p.tiles_t = static_cast<int32_t>(parts_of(n, kWalkItems));
      p.parts_t = walk_parts(p.blocks_t, p.tiles_t);
      p.slab_ld = up(a.dims, 4);
      p.slabs_y = p.parts_t > 1;
      if (p.slabs_y) p.at_slab_y = room(v * p.slab_ld * 4 * p.parts_t);
    }
    p.bytes = std::max<int64_t>(at, 256);
    return p;
  }
  if (p.sums) {
    p.t_sums = choose(n, v, p.k * 2, p.pairs, false, true, true, false);
    p.at_sums = room(n * p.t_sums.c * 8);
    p.at_own = room(n * 4);
    if (p.grad && !a.stats) p.at_stats = room(n * 16);
  }
  if (p.grad) {
    int64_t piece = kPieceBytes / (std::max<int64_t>(n, 1) * 2 * p.planes_d) / 256 * 256;
    piece = std::max<int64_t>(piece, 256);
    if (piece >= v)
      piece = v;
    else
      piece = up(parts_of(v, parts_of(v, piece)), 256);
    p.piece = piece;
    p.k_d = up(piece, 64);
    // (an odd number of 128-byte lines from row to row: tiles that read rows of d side by side meet in fewer
    // channels of the caches: 2048 x 768 x 32768 fp32's d_features 285 -> 264 us, 4096 x 2048 x 131072 bf16's 440 -> 430)
    p.ld_d = p.k_d / 64 % 2 ? p.k_d : p.k_d + 64;
    p.t_d = choose(n, piece, p.k * 2, p.pairs, false, true, true, false);
    // Logits of a call whose d is one piece are kept between the two, in fp32, rather than computed again (all
    // kernels of a call, computed again and kept, us: 515 x 1000 x 50021 fp16 418 and 373, 2048 x 768 x 32768 fp32 1433
    // and 1212, 512 x 4096 x 100000 bf16 2420 and 2070, 100 x 200 x 50 fp32 58 and 53).
    p.keep = p.sums && piece == v && n * p.k_d * 4 <= 2 * kPieceBytes;
    if (p.keep) p.at_z = room(n * p.k_d * 4);
    p.at_d = room(n * p.ld_d * 2 * p.planes_d);
    p.slab_ld = up(a.dims, 4);
    if (a.d_features) {
      p.t_x = choose(n, a.dims, p.k_d * 2, p.pairs_d, false, true, false, true);
      p.slabs_x = p.t_x.parts > 1 || piece < v;
      if (p.slabs_x) p.at_slab_x = room(n * p.slab_ld * 4 * p.t_x.parts);
    }
    if (a.d_table) {
      p.t_y = choose(piece, a.dims, n * 2, p.pairs_d, false, true, false, true);
      p.slabs_y = p.t_y.parts > 1;
      if (p.slabs_y) p.at_slab_y = room(piece * p.slab_ld * 4 * p.t_y.parts);
    }
  }
  p.bytes = std::max<int64_t>(at, 256);
  return p;
}

// One piece of the classes: which, the columns of d that are written and multiplied (its classes, up to a whole
// 128 bytes, those past its classes being 0), and the tiles of its products. The last piece may be shorter than
// the others: its tiles are its own, so that none begins past its classes.
struct LossPiece {
  int64_t first, count, width;
  Tiles d, x, y;
};

inline LossPiece piece_of(const LossPlan &p, int64_t classes, int64_t first) {
  const int64_t count = std::min(p.piece, classes - first);
  LossPiece q{first, count, up(count, 64), p.t_d, p.t_x, p.t_y};
  q.d.c = static_cast<int32_t>(parts_of(count, q.d.bc));  // (a tile is a multiple of 64 wide: it writes all of `width`)
  if (q.y.br > 0) q.y.r = static_cast<int32_t>(parts_of(q.count, q.y.br));  // (planned where d_table is wanted)
  return q;
}

// The operands of a call's products: laid out in the workspace or in place; w: the weighted features.
struct LossOperands {
  Operand x, y, w;
};

inline LossOperands loss_operands(const tmnn_class_loss_args &a, const LossPlan &p) {
  const char *ws = static_cast<const char *>(a.workspace);
  const int64_t size = static_cast<int64_t>(dtype_size(a.dtype));
  auto laid = [&](int64_t at, int64_t rows) {
    return Operand{ws + at, p.ld * 2, rows * p.ld * 2, static_cast<int32_t>(rows), static_cast<int32_t>(p.k * 2)};
  };
  auto in_place = [&](const void *ptr, int64_t stride, int64_t rows) {  // rows of dims values
    return Operand{static_cast<const char *>(ptr), stride * size, 0, static_cast<int32_t>(rows),
                   static_cast<int32_t>(up(a.dims, 8) * 2)};
  };
  return {p.lay_x ? laid(p.at_x, a.rows) : in_place(a.features, a.feature_stride, a.rows),
          p.lay_y ? laid(p.at_y, a.classes) : in_place(a.table, a.table_stride, a.classes), laid(p.at_w, a.rows)};
}

// The products: the logits for the sums; of a piece the logits for d, d_features (d and the table, the latter
// transposed) and d_table (d and the weighted features, both transposed).
inline TileArgs sums_product(const tmnn_class_loss_args &a, const LossPlan &p, const LossOperands &o) {
  return tile_args(o.x, o.y, a.rows, a.classes, p.t_sums, p.pairs);
}
inline Operand piece_table(const LossOperands &o, const LossPiece &q) {
  Operand y = o.y;
  y.base += q.first * y.ld;
  y.rows = static_cast<int32_t>(q.count);
  return y;
}
inline Operand piece_d(const tmnn_class_loss_args &a, const LossPlan &p, const LossPiece &q) {
  return {static_cast<const char *>(a.workspace) + p.at_d, p.ld_d * 2, a.rows * p.ld_d * 2,
          static_cast<int32_t>(a.rows), static_cast<int32_t>(q.width * 2)};
}
inline TileArgs d_product(const tmnn_class_loss_args &a, const LossPlan &p, const LossOperands &o, const LossPiece &q) {
  return tile_args(o.x, piece_table(o, q), a.rows, q.count, q.d, p.pairs);
}
inline TileArgs features_product(const tmnn_class_loss_args &a, const LossPlan &p, const LossOperands &o, const LossPiece &q) {
  return tile_args(piece_d(a, p, q), piece_table(o, q), a.rows, a.dims, q.x, p.pairs_d);
}
inline TileArgs table_product(const tmnn_class_loss_args &a, const LossPlan &p, const LossOperands &o, const LossPiece &q) {
  return tile_args(piece_d(a, p, q), o.w, q.count, a.dims, q.y, p.pairs_d);
}

// ---- logits from 8-bit operands ------------------------------------------------------------

struct LogitsPlan {
  bool lay_x, lay_y;
  int64_t ld, steps;
  Tiles t;
  int64_t slab_ld, at_x, at_y, at_slabs, bytes;
};

inline LogitsPlan plan_logits(const tmnn_class_logits_f8_args &a) {
  LogitsPlan p{};
  auto lies_well = [&](const void *ptr, int64_t stride, int64_t rows) {
    return aligned(ptr, 16) && (stride % 16 == 0 || rows <= 1) && stride < (1 << 23);
  };
  p.lay_x = !lies_well(a.features, a.feature_stride, a.rows);
  p.lay_y = !lies_well(a.table, a.table_stride, a.classes);
  p.ld = up(a.dims, 16);
  p.steps = parts_of(a.dims, kScaleBlock);
  p.t = choose(a.rows, a.classes, a.dims, 1, true, a.dtype != TMNN_DTYPE_F32, true, true);
  p.slab_ld = up(a.classes, 4);
  int64_t at = 0;
  auto room = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  if (p.lay_x) p.at_x = room(a.rows * p.ld);
  if (p.lay_y) p.at_y = room(a.classes * p.ld);
  if (p.t.parts > 1) p.at_slabs = room(a.rows * p.slab_ld * 4 * p.t.parts);
  p.bytes = at;  // (0: most calls need none)
  return p;
}

inline TileArgs logits_product(const tmnn_class_logits_f8_args &a, const LogitsPlan &p) {
  auto operand = [&](const void *ptr, int64_t stride, bool lay, int64_t at, int64_t rows) {
    // (a row's end counts in whole 16 bytes, also that of a single row)
    return Operand{lay ? static_cast<const char *>(a.workspace) + at : static_cast<const char *>(ptr),
                   lay ? p.ld : std::max(stride, p.ld), 0, static_cast<int32_t>(rows), static_cast<int32_t>(p.ld)};
  };
  return tile_args(operand(a.features, a.feature_stride, p.lay_x, p.at_x, a.rows),
                   operand(a.table, a.table_stride, p.lay_y, p.at_y, a.classes), a.rows, a.classes, p.t, 1);
}

}  // namespace tmnn_hip
