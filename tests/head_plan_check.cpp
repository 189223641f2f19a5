// Reads the class head's plans (csrc/head_plan.hpp) on the CPU: every tile that a call launches begins inside its
// operands, no buffer that a tile loads from has a size that a load meant to give zeros falls into, rows that exist
// are loaded from where they are and others from past the buffer's end, laid-out operands lie
// in the workspace, and a launch's threads fit 32 bits. Prints the first plans that break this; returns how
// many there are (up to 100).
#include <math.h>
#include <stdio.h>
#include <stdlib.h>

#include <random>

#include "head_plan.hpp"

using namespace tmnn_hip;

namespace {

int bad = 0;
long long plans = 0, several = 0, tiles = 0;
char now[256];

void fail(const char *what, const char *product, long long tile, long long value) {
  if (++bad <= 10) printf("%s: %s, %s from %lld on: %lld\n", now, what, product, tile, value);
}

// The rows that the tile from row `first` on loads, `each` rows from one load of a thread to its next.
void rows_of(const char *product, const Operand &o, bool transposed, int64_t first, int64_t edge, int64_t waves) {
  const int64_t each = waves * (transposed ? 64 / (edge / 8) : 8), rows = transposed ? 64 : edge;
  const int64_t exist = transposed ? std::min<int64_t>(o.rows, 64) : std::min<int64_t>(o.rows - first, edge);
  const uint32_t size = transposed ? 0x7fffffffu : static_cast<uint32_t>(tile_bytes(o, static_cast<int32_t>(first), static_cast<int32_t>(edge)));
  for (const int64_t r : {int64_t{0}, each - 1, each, exist - 1, exist, (exist / each + 1) * each, 128 - each % 128, rows - 1}) {
    if (r < 0 || r >= rows) continue;
    const uint64_t whole = static_cast<uint64_t>(row_offset(o, static_cast<int32_t>(r % each))) +
                           static_cast<uint64_t>(r / each) * load_step(o, static_cast<int32_t>(each));
    if (r < exist && (whole != static_cast<uint64_t>(r * o.ld) || whole + 16 > size)) fail("an offset", product, first + r, static_cast<long long>(whole));
    // (a transposed operand's rows that do not exist are left out by their number)
    if (r >= exist && !transposed && whole < size) fail("a row that does not exist lies inside", product, first + r, static_cast<long long>(whole));
    if (!transposed && whole + 128 >= 1ull << 32) fail("an offset past 32 bits", product, first + r, static_cast<long long>(whole));
    if (transposed && r < exist && kOutside + static_cast<uint64_t>(r / each) * load_step(o, static_cast<int32_t>(each)) >= 1ull << 32)
      fail("an offset past 32 bits", product, first + r, o.ld);
  }
}

// One side of a product: tiles of `edge` rows, `count` of them, over `rows` of the output.
void side(const char *product, const Operand &o, bool transposed, int64_t count, int64_t edge, int64_t rows, const char *ws,
          int64_t ws_bytes, int planes, int64_t waves) {
  if (count * edge < rows) fail("rows that no tile takes", product, count * edge, rows);
  if (count > 0 && (count - 1) * edge >= rows) fail("a tile past the output", product, (count - 1) * edge, rows);
  if (o.rows < 0 || o.bytes < 0 || o.bytes % 16) fail("rows or bytes", product, 0, o.bytes);
  for (int64_t t = 0; t < count; ++t) {
    const int64_t first = t * edge;
    ++tiles;
    if (t == 0 || t == count - 1) rows_of(product, o, transposed, first, edge, waves);
    if (transposed) {
      if (first * 2 >= o.bytes) fail("a tile past the operand", product, first, o.bytes);
      continue;
    }
    if (first >= o.rows) fail("a tile past the operand", product, first, o.rows);
    const int32_t size = tile_bytes(o, static_cast<int32_t>(first), static_cast<int32_t>(edge));
    // (as the buffer takes it: unsigned)
    if (static_cast<uint32_t>(size) >= kOutside) fail("a buffer's size", product, first, static_cast<uint32_t>(size));
    const int64_t left = std::min<int64_t>(o.rows - first, edge);
    if (first < o.rows && size != left * o.ld) fail("a buffer's size is not its rows'", product, first, size);
  }
  if (o.base >= ws && o.base < ws + ws_bytes) {
    const int64_t end = o.base - ws + (planes - 1) * o.plane + (static_cast<int64_t>(o.rows) - 1) * o.ld + o.bytes;
    if (end > ws_bytes) fail("an operand past the workspace", product, end, ws_bytes);
  }
}

void product(const char *name, const TileArgs &t, const Tiles &s, bool xt, bool yt, const char *ws, int64_t ws_bytes,
             int x_planes, int y_planes) {
  if (t.tiles_r != s.r || t.tiles_c != s.c) fail("tiles", name, t.tiles_r, s.r);
  const int64_t waves = s.shape <= kWide ? 8 : 4;
  side(name, t.x, xt, t.tiles_r, s.br, t.rows, ws, ws_bytes, x_planes, waves);
  side(name, t.y, yt, t.tiles_c, s.bc, t.cols, ws, ws_bytes, y_planes, waves);
  const long long threads = 64ll * waves * t.tiles_r * t.tiles_c * t.parts;
  if (threads >= 1ll << 32) fail("threads of a launch", name, 0, threads);
  if (t.parts < 1 || (t.parts - 1ll) * t.part_steps >= 1ll * t.steps * t.pairs ||
      1ll * t.parts * t.part_steps < 1ll * t.steps * t.pairs)
    fail("parts", name, t.parts, t.part_steps);
}

char *at(int64_t place) { return reinterpret_cast<char *>(static_cast<uintptr_t>(place)); }

void loss(int32_t dtype, int64_t n, int64_t v, int64_t d, int64_t pad, int gradient, bool back) {
  tmnn_class_loss_args a{};
  a.dtype = dtype;
  a.temperature = 1.f;
  a.rows = n, a.classes = v, a.dims = d;
  a.feature_stride = a.table_stride = a.d_feature_stride = a.d_table_stride = d + pad;
  a.features = at(1ll << 40);
  a.table = at(2ll << 40);
  a.labels = at(3ll << 40);
  a.loss = back ? nullptr : reinterpret_cast<float *>(at(4ll << 40));
  a.stats = reinterpret_cast<float *>(at(5ll << 40));
  if (gradient & 1) a.d_features = at(6ll << 40);
  if (gradient & 2) a.d_table = at(7ll << 40);
  a.workspace = at(8ll << 40);
  const LossPlan p = plan_loss(a, back);
  a.workspace_bytes = p.bytes;
  ++plans;
  if (p.narrow) return;
  snprintf(now, sizeof now, "class_loss%s %lld x %lld x %lld, dtype %d, pad %lld, gradients %d", back ? "_backward" : "",
           static_cast<long long>(n), static_cast<long long>(d), static_cast<long long>(v), dtype,
           static_cast<long long>(pad), gradient);
  const char *ws = static_cast<const char *>(a.workspace);
  const LossOperands o = loss_operands(a, p);
  if (p.sums) product("sums", sums_product(a, p, o), p.t_sums, false, false, ws, p.bytes, p.planes, p.planes);
  if (!p.grad) return;
  if (p.piece < v) ++several;
  for (int64_t first = 0; first < v; first += p.piece) {
    const LossPiece q = piece_of(p, v, first);
    if (!p.keep)
      product("d of a piece", d_product(a, p, o, q), q.d, false, false, ws, p.bytes, p.planes, 1);
    // what d's rows hold is written: by tiles, whole
    const int64_t written = p.keep ? q.width : static_cast<int64_t>(q.d.c) * q.d.bc;
    if (q.width < q.count || q.width > written || q.width > p.ld_d) fail("d's columns", "d", first, q.width);
    if (a.d_features)
      product("d_features", features_product(a, p, o, q), q.x, false, true, ws, p.bytes, p.planes_d, 1);
    if (a.d_table)
      product("d_table", table_product(a, p, o, q), q.y, true, true, ws, p.bytes, p.planes_d, p.planes);
  }
}

void logits(int32_t dtype, int64_t n, int64_t v, int64_t d, int64_t stride) {
  tmnn_class_logits_f8_args a{};
  a.dtype = dtype;
  a.rows = n, a.classes = v, a.dims = d;
  a.feature_stride = a.table_stride = stride;
  a.logit_stride = v;
  a.features = at(1ll << 40);
  a.table = at(2ll << 40);
  a.workspace = at(8ll << 40);
  const LogitsPlan p = plan_logits(a);
  ++plans;
  snprintf(now, sizeof now, "class_logits_f8 %lld x %lld x %lld, dtype %d, stride %lld", static_cast<long long>(n),
           static_cast<long long>(d), static_cast<long long>(v), dtype, static_cast<long long>(stride));
  product("logits", logits_product(a, p), p.t, false, false, static_cast<const char *>(a.workspace), p.bytes, 1, 1);
}

}  // namespace

int main(int argc, char **argv) {
  const int draws = argc > 1 ? atoi(argv[1]) : 2000;
  const int64_t rows[] = {1, 2, 63, 64, 65, 127, 128, 129, 515, 1024, 1100, 2048, 4096, 5000, 8192, 16384, 65536};
  const int64_t classes[] = {1, 2, 127, 128, 129, 255, 257, 1000, 10007, 32000, 50021, 50257, 65024, 70001, 128256, 130001, 131072, 151936, 262144};
  const int64_t dims[] = {129, 136, 200, 768, 1000, 2048, 4096};
  for (int32_t dtype = 0; dtype < 3; ++dtype)
    for (int64_t n : rows)
      for (int64_t v : classes)
        for (int64_t d : dims)
          for (int back = 0; back < 2; ++back)
            for (int gradient = back; gradient < 4; ++gradient) loss(dtype, n, v, d, d % 8 ? 3 : 0, gradient, back);
  for (int32_t dtype = 0; dtype < 3; ++dtype)  // few rows of very many classes: rows of d far apart
    for (int64_t n : {1, 2, 3, 7, 15, 16, 31, 33, 64})
      for (int64_t v : {1ll << 20, (1ll << 22) - 64, 1ll << 22, (1ll << 22) + 1, 5000001ll, 1ll << 23, (1ll << 24) - 1, 1ll << 24})
        for (int gradient = 0; gradient < 4; ++gradient) loss(dtype, n, v, 136, 0, gradient, false);
  std::mt19937_64 g(1);
  auto between = [&](double low, double high) {  // over the logarithm
    return static_cast<int64_t>(exp2(std::uniform_real_distribution<double>(log2(low), log2(high))(g)));
  };
  for (int i = 0; i < draws; ++i) {
    const int64_t n = between(1, 1 << 24), v = std::min<int64_t>(between(1, 1 << 24), (1ll << 38) / n);
    const int64_t d = between(1, 1 << 16);
    if (static_cast<double>(n + v) * static_cast<double>(d) > 1e11) continue;
    const bool back = g() % 2;
    loss(static_cast<int32_t>(g() % 3), n, v, d, g() % 3 ? 0 : g() % 9, back ? 1 + g() % 3 : g() % 4, back);
    if (static_cast<double>(n) * static_cast<double>(v) < 1.4e11)  // (288 GB of logits)
      logits(static_cast<int32_t>(g() % 3), n, v, d, g() % 2 ? up(d, 16) : d);
  }
  printf("%lld plans, %lld in several pieces, %lld tiles, %d bad\n", plans, several, tiles, bad);
  return bad < 100 ? bad : 100;
}
