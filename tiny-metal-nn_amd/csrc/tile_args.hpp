// tile_args.hpp -- what a tile product is given, and which bytes of an operand a tile's
// loads may touch. Plain C++: tests without a GPU read it too.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define TMNN_BOTH __host__ __device__ __forceinline__
#else
#define TMNN_BOTH inline
#endif

namespace tmnn_hip {

// One operand. Rows of it are the output's rows (x) or columns (y), or, of a transposed
// one, the values of k. Everything of it that a tile reads starts at multiples of 16 bytes.
struct Operand {
  const char *base;
  int64_t ld;      // bytes from row to row: below 2^23, or, of d of few rows, up to 2^25 and 256; the rows of a
                   // tile, those that do not exist too, lie within 32 bits (d's tiles of up to 128 rows are 128 high)
  int64_t plane;   // bytes from plane to plane (operands in two terms)
  int32_t rows;    // rows that exist
  int32_t bytes;   // bytes of a row that exist, a multiple of 16; what lies beyond counts as 0
};

struct TileArgs {
  Operand x, y;
  int32_t rows, cols;          // of the output
  int32_t tiles_r, tiles_c, parts;
  int32_t steps;               // of k, in one pair of planes
  int32_t pairs;               // 1: one plane each; 2: and x low; 3: x high, y low first, x low then
  int32_t part_steps;          // steps of one part, counted over all pairs
};

constexpr uint32_t kOutside = 0x80000000u;  // an offset past the end of every buffer: loads give 0

// Bytes of the buffer that a tile of `tile` rows from row `first` on loads from: its rows that exist. It lies below
// kOutside (the hardware takes it as an unsigned number), or loads there would be made.
TMNN_BOTH int32_t tile_bytes(const Operand &o, int32_t first, int32_t tile) {
  const int32_t left = o.rows - first;
  return left <= 0 ? 0 : static_cast<int32_t>((left < tile ? left : tile) * o.ld);
}

// Byte offset of a tile's row, and from one load of a thread to its next, `rows` rows on. (32 bits: a row that does
// not exist lies past the buffer's end, never back inside it.)
TMNN_BOTH uint32_t row_offset(const Operand &o, int32_t row) { return static_cast<uint32_t>(row * o.ld); }
TMNN_BOTH uint32_t load_step(const Operand &o, int32_t rows) { return static_cast<uint32_t>(rows * o.ld); }

}  // namespace tmnn_hip
