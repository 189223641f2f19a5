// distill_kernel.hpp -- distillation of rows of logits from a teacher's listed
// values: loss and gradient.
//
//   loss = w T^2 [ sum_j q_j (ln q_j - ln p_j) + q_r (ln q_r - ln p_r) ]
//   d z_v = w T [ Q p_v - q_v [v listed] - q_r p_v / p_r [v not listed] ],  Q = sum_j q_j + q_r
//
// with p = softmax(z / T). Kind 0 (teacher logits): q = softmax(t / T) over the
// listed classes, q_r = 0. Kind 1 (teacher log-probabilities): q = exp(t), and
// the classes that are not listed form one class of mass q_r = 1 - sum q.
//
// Kind 1 sums up the classes that are not listed by themselves, relative to their
// own maximum m_d, and lets the listed ones join: ln p_r and p_v / p_r keep their
// precision however little the rest weighs. Either way the gradient of the
// classes that are not listed is one exponential,
//   w T a_d 2^(c (z_v - m_d)),
// and that of listed class j is w T (a_a 2^(c (z_j - m_a)) - q_j); (m_d, a_d, m_a,
// a_a) are the row's statistics. m_a = -inf marks a row whose classes are all
// masked: loss and gradient 0.
//
// Bound: reading the logits once and writing the gradient, and, for rows that do not stay in
// registers, reading them again from the caches: 8192 x 65536 bf16, 32 values with the tail
// 454 us (4.7 TB/s of the 2.1 GB that have to move; a pass that reads and writes each once takes
// 345 at the card's best); 16384 x 8192 bf16, in
// registers, 111 us (4.8 TB/s). Short rows are bound by their instructions: 30011 x 1000 fp16
// 42 us, 2^18 x 16 fp32 14 us.
#pragma once

#include "logprob_kernel.hpp"

namespace tmnn_hip {

constexpr int kMaxTeacher = 256;
constexpr int kMaxPartLen = 1 << 17;  // classes of a block: its bits of listed classes in LDS

struct DistillArgs {
  const void *logits;
  int64_t row_stride;
  const void *ids;
  const float *teacher;
  const float *weights;  // null: 1; backward: the loss's gradient
  int32_t wide_index, kind;
  int32_t rows, classes, k;
  int32_t parts, part_len;
  float c, t, inv_t;  // log2(e) / T, T, 1 / T
  double inv_t64;
  float *loss;
  float *stats;  // [rows][4]
  void *d_logits;
  int64_t d_row_stride;
  float2 *part_sum;  // [rows][parts]: m, r
  float *list_z;     // [rows][k]: logits of the listed classes
};

// What the loss and the gradient need of a row beyond its listed classes.
struct DistillRow {
  float m_d, a_d, m_a, a_a;
};

// A listed class's ln q - ln p, the differences of its logits in 64 bits: the loss is
// small against both.
template <bool TAIL>
__device__ __forceinline__ float log_ratio(const DistillArgs &a, float t, float top, float log_z,
                                           float z, float m, float log_s) {
  const double lq = TAIL ? t : (static_cast<double>(t) - top) * a.inv_t64 - log_z;
  return static_cast<float>(lq - (static_cast<double>(z) - m) * a.inv_t64 + log_s);
}
// q of a teacher value: relative to `top` over 1 / inv_z (kind 0), or itself.
template <bool TAIL>
__device__ __forceinline__ float teacher_mass(const DistillArgs &a, float t, float top, float inv_z) {
  return TAIL ? exp_of(t) : exp2_raw((t - top) * a.c) * inv_z;
}

// sum q over G lanes' listed classes, each lane's by `each(f)`: (sum q, 1 - sum q).
// Kind 1 takes the mass that the teacher left out from 64-bit sums: 1 - sum q in 32 bits
// is off by 2^-24 of the whole, which is all of a small rest.
struct TeacherMass {
  float all, left;
  float poison;  // 0, or NaN where one of the lanes' is
};
template <bool TAIL, int G, class Each>
__device__ __forceinline__ TeacherMass teacher_total(const DistillArgs &a, float top, float poison,
                                                     Each each) {
  TeacherMass m{0.0f, 0.0f, lanes_any<G>(poison != 0.0f) ? __builtin_nanf("") : 0.0f};
  if (!TAIL) {
    each([&](float t) { m.all += exp2_raw((t - top) * a.c); });
    m.all = lanes_sum<G>(m.all);
    return m;
  }
  double total = 0.0;
  each([&](float t) { total += exp(static_cast<double>(t)); });
  total = lanes_sum<G>(total);
  m.all = static_cast<float>(total);
  m.left = fmaxf(static_cast<float>(1.0 - total), 0.0f);
  return m;
}

// The row's statistics and the part of its loss that the listed classes do not
// bring: dense = settled sums of all classes (kind 0) or of the unlisted ones
// (kind 1); all = of all classes; listed = the sum of the listed ones in the shift of
// all.m (kind 1); mass = sum q, left = 1 - mass (kind 1).
template <bool TAIL>
__device__ __forceinline__ DistillRow distill_row(const DistillArgs &a, const Soft &dense,
                                                  const Soft &all, float listed, float mass,
                                                  float left, float *rest_loss) {
  DistillRow r;
  r.m_a = all.m;
  *rest_loss = 0.0f;
  if (!TAIL) {
    r.a_a = quotient(mass, all.S);
    r.m_d = r.m_a;
    r.a_d = r.a_a;
    return r;
  }
  const bool rest = dense.S != 0.0f;
  const float qr = rest ? left : 0.0f;
  const float q = mass + qr;
  r.a_a = quotient(q, all.S);
  r.m_d = rest ? dense.m : 0.0f;
  // (no rest: 0, or the NaN of the listed classes)
  r.a_d = rest ? exp2_raw((dense.m - all.m) * a.c) * r.a_a - quotient(qr, dense.S) : 0.0f * r.a_a;
  if (qr > 0.0f) {
    // Where the rest is most of both, its two logarithms are small, and are taken from what
    // is missing to 1: rounded logarithms of the sums would be off by half an ulp of ln
    // of the class count, which the loss of a flat teacher is not large against.
    const float over = quotient(listed, dense.S * exp2_raw((dense.m - all.m) * a.c));
    const float log_pr = over < 1.0f ? -log1p_of(over)
                                     : ((dense.m - all.m) * a.inv_t + log1p_of(dense.r)) - log1p_of(all.r);
    const float log_qr = mass < 0.5f ? log1p_of(-mass) : logf(qr);
    *rest_loss = qr * (log_qr - log_pr);
  }
  return r;
}

// ---- short rows -----------------------------------------------------------------

// TAIL: kind 1. BACK: statistics are given and only the gradient is written. Else, with TAIL,
// the listed classes are left out of the sums over the lanes' classes, and join them one
// by one.
template <class T, int G, int NV, bool TAIL, bool BACK>
__global__ __launch_bounds__(kGroupThreads) void distill_group_kernel(DistillArgs a) {
  constexpr int N = Row<T>::n, E = N * NV;
  __shared__ GroupWords<T, G, NV> words;  // the first entry that lists a class, then its gradient
  const float inf = __builtin_inff();
  const Group<T, G, NV> g;
  const int64_t row = g.row;
  const float w = row < a.rows ? (a.weights ? a.weights[row] : 1.0f) : 0.0f;
  const bool live = row < a.rows && w != 0.0f;
  const T *z = static_cast<const T *>(a.logits) + (live ? row : 0) * a.row_stride;
  const int k = live ? a.k : 0;
  // The lane's entries lane, lane + G, ...: the first kKept in registers. NaN values
  // and ids beyond the classes make `poison` NaN.
  constexpr int kKept = G <= 4 ? 8 / G : 1;
  int id[kKept];
  float value[kKept], logit[kKept], poison = 0.0f;
  auto entry = [&](int j, int &i, float &t) {
    const int64_t at = load_index(a.ids, row * a.k + j, a.wide_index);
    i = at >= 0 && at < a.classes ? static_cast<int>(at) : -1;
    t = a.teacher[row * a.k + j];
    if (at >= a.classes || (at >= 0 && t != t)) poison = __builtin_nanf("");
  };
#pragma unroll
  for (int e = 0; e < kKept; ++e) {
    id[e] = -1;
    value[e] = 0.0f;
    if (g.lane + e * G < k) entry(g.lane + e * G, id[e], value[e]);
  }
  float v[E];
  g.load_rows(a.logits, a.row_stride, a.rows, a.classes, live, words.word, v);
  int *mine = words.lane();
#pragma unroll
  for (int e = 0; e < E; ++e) mine[e] = kUnlisted;
  wave_fence();
#pragma unroll
  for (int e = 0; e < kKept; ++e)
    if (id[e] >= 0) {
      atomicMin(&words.of(id[e]), g.lane + e * G);
      logit[e] = Row<T>::up(z[id[e]]);
    }
  for (int j = g.lane + kKept * G; j < k; j += G) {
    int i;
    float t;
    entry(j, i, t);
    if (i >= 0) atomicMin(&words.of(i), j);
  }
  wave_fence();
#pragma unroll
  for (int e = 0; e < kKept; ++e)
    if (id[e] >= 0 && words.of(id[e]) != g.lane + e * G) id[e] = -1;
  // f(class, value, logit) for the lane's entries that count: first the others, which may
  // find a class's word taken by another's gradient, whose bits are no entry's number
  auto entries = [&](auto f) {
    for (int j = g.lane + kKept * G; j < k; j += G) {
      int i;
      float t;
      entry(j, i, t);
      if (i >= 0 && words.of(i) == j) f(i, t, Row<T>::up(z[i]));
    }
#pragma unroll
    for (int e = 0; e < kKept; ++e)
      if (id[e] >= 0) f(id[e], value[e], logit[e]);
  };
  float top = -inf;
  if (!TAIL) {
    entries([&](int, float t, float) { top = fmaxf(top, t); });
    top = lanes_max<G>(top);
  }
  const TeacherMass tm = teacher_total<TAIL, G>(
      a, top, poison, [&](auto f) { entries([&](int, float t, float) { f(t); }); });
  const float total = tm.all;
  // no mass at all: nothing is listed, or only values of -inf
  const bool none = !TAIL && top == -inf && tm.poison == 0.0f;
  const float inv_z = TAIL ? 1.0f : quotient(1.0f, total), log_z = TAIL ? 0.0f : log_of(total);
  const float mass = (TAIL ? total : none ? 0.0f : total * inv_z) + tm.poison;

  DistillRow r{};
  float loss = 0.0f, rest_loss = 0.0f, listed = 0.0f;
  Soft all;
  if (BACK) {
    if (live) {
      const float4 s = reinterpret_cast<const float4 *>(a.stats)[row];
      r = DistillRow{s.x, s.y, s.z, s.w};
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = exp2_raw((v[e] - r.m_d) * a.c);
  } else {
    Soft dense;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (TAIL && mine[e] != kUnlisted) v[e] = -inf;
      dense.m = fmaxf(dense.m, v[e]);
    }
    dense.m = lanes_max<G>(dense.m);
    const float shift = dense.m == -inf ? 0.0f : dense.m;
    int best_n = 0;  // classes of the largest logit, whose terms are 1
    dense.r = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool best = v[e] == dense.m;
      v[e] = exp2_raw((v[e] - shift) * a.c);
      dense.r += best ? 0.0f : v[e];
      best_n += best;
    }
    best_n = lanes_isum<G>(best_n);
    dense.r = lanes_sum<G>(dense.r) + static_cast<float>((dense.m == -inf ? 0 : best_n) - 1);
    if (dense.m == inf) dense.r = __builtin_nanf("");
    dense.S = 1.0f + dense.r;
    all = dense;
    if (TAIL) {
      entries([&](int, float, float y) { all.m = fmaxf(all.m, y); });
      all.m = lanes_max<G>(all.m);
      const float up = all.m == -inf ? 0.0f : all.m;
      float p = 0.0f;
      int n = 0;  // listed classes of the largest logit
      entries([&](int, float, float y) {
        p += y == all.m ? 0.0f : exp2_raw((y - up) * a.c);
        n += y == all.m;
      });
      n = lanes_isum<G>(n);
      const bool one = dense.m == all.m;  // the 1 that r leaves out is the rest's, or a listed class's
      all.r = 0.0f;
      soft_join(all, dense, a.c, one && dense.m != -inf);
      p = lanes_sum<G>(p);
      listed = p + static_cast<float>(n);
      all.r += p + static_cast<float>(all.m == -inf ? -1 : one ? n : n - 1);
      if (all.m == inf) all.r = __builtin_nanf("");
      all.S = 1.0f + all.r;
    }
    r = distill_row<TAIL>(a, dense, all, listed, mass, tm.left, &rest_loss);
    if (all.m == -inf && all.S == 0.0f) r = DistillRow{0.0f, 0.0f, -inf, 0.0f};  // every class is masked
  }
  const bool zero = !live || (r.m_a == -inf && r.a_a == r.a_a);
  const float scale = w * a.t, log_s = log1p_of(all.r);
  entries([&](int i, float t, float y) {
    const float q = none ? 0.0f : teacher_mass<TAIL>(a, t, top, inv_z);
    if (!BACK && q != 0.0f) loss += q * log_ratio<TAIL>(a, t, top, log_z, y, all.m, log_s);
    const float d = scale * (r.a_a * exp2_raw((y - r.m_a) * a.c) - q);
    words.of(i) = fabsf(d) < 1.2e-38f ? 0 : __float_as_int(d);
  });
  if (!BACK) {
    loss = lanes_sum<G>(loss) + rest_loss + tm.poison;
    const bool empty = all.m == -inf && all.S == 0.0f;
    if (g.lane == 0 && row < a.rows) {
      if (a.loss) a.loss[row] = !live || empty ? 0.0f : loss * a.t * a.t * w;
      if (a.stats)
        reinterpret_cast<float4 *>(a.stats)[row] =
            live ? make_float4(r.m_d, r.a_d, r.m_a, r.a_a) : make_float4(0.0f, 0.0f, -inf, 0.0f);
    }
    if (!a.d_logits) return;
  }
  wave_fence();
  const float dense_scale = scale * r.a_d;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = mine[e] == kUnlisted ? dense_scale * v[e] : __int_as_float(mine[e]);
    v[e] = zero ? 0.0f : d;
  }
  g.store_rows(a.d_logits, a.d_row_stride, a.rows, a.classes, words.word, v);
}

// ---- long rows ---------------------------------------------------------------------

struct ListLds {
  __attribute__((aligned(16))) int id[kMaxTeacher];
  float z[kMaxTeacher], t[kMaxTeacher], q[kMaxTeacher];
  float wrong;
  DistillRow row;
};

// The thread's entry: its class, or -1 for an unused entry. An entry beyond the classes
// makes the row NaN. NT >= k.
__device__ __forceinline__ int list_entry(const DistillArgs &a, int64_t row, bool *wrong) {
  const int tid = threadIdx.x;
  if (tid >= a.k) return -1;
  const int64_t i = load_index(a.ids, row * a.k + tid, a.wide_index);
  if (i >= a.classes) *wrong = true;
  return i >= 0 && i < a.classes ? static_cast<int>(i) : -1;
}

// Puts the entries into LDS; a class counts by its first entry (the others: -1). Returns
// the thread's.
__device__ __forceinline__ int put_list(const DistillArgs &a, ListLds &l, int64_t row, int id,
                                        float z, bool wrong) {
  const int tid = threadIdx.x;
  if (tid == 0) l.wrong = 0.0f;
  if (tid < ((a.k + 3) & ~3)) {
    l.id[tid] = id;
    if (tid < a.k) {
      l.t[tid] = a.teacher[row * a.k + tid];
      l.z[tid] = z;
    }
  }
  __syncthreads();
  const bool again = tid < a.k && id >= 0 && listed_before(l.id, a.k, tid, id);
  if (wrong) l.wrong = __builtin_nanf("");  // every writer writes the same
  __syncthreads();
  if (again) l.id[tid] = id = -1;
  __syncthreads();
  return id;
}

// One wave: q of the listed classes into l.q; returns their mass. `top` and `log_z`
// as log_ratio takes them.
template <bool TAIL>
__device__ __forceinline__ TeacherMass teacher_sums(const DistillArgs &a, ListLds &l, float *top,
                                                    float *log_z) {
  const int lane = threadIdx.x & (kWave - 1);
  const float inf = __builtin_inff();
  float t_max = -inf, poison = l.wrong;
  for (int j = lane; j < a.k; j += kWave)
    if (l.id[j] >= 0) {
      t_max = fmaxf(t_max, l.t[j]);
      if (l.t[j] != l.t[j]) poison = __builtin_nanf("");
    }
  if (!TAIL) t_max = lanes_max<kWave>(t_max);
  TeacherMass m = teacher_total<TAIL, kWave>(a, t_max, poison, [&](auto f) {
    for (int j = lane; j < a.k; j += kWave)
      if (l.id[j] >= 0) f(l.t[j]);
  });
  const float total = m.all;
  const bool none = !TAIL && t_max == -inf && m.poison == 0.0f;
  const float inv_z = TAIL ? 1.0f : quotient(1.0f, total);
  for (int j = lane; j < a.k; j += kWave)
    l.q[j] = l.id[j] >= 0 && !none ? teacher_mass<TAIL>(a, l.t[j], t_max, inv_z) : 0.0f;
  *top = t_max;
  *log_z = TAIL ? 0.0f : log_of(total);
  // sum q is 1 for kind 0 (a sum of NaN stays one)
  m.all = (TAIL ? total : none ? 0.0f : total * inv_z) + m.poison;
  return m;
}

// Writes the gradient of a part: all classes as unlisted ones, then the listed; between
// the two listed() returns the thread's class (-1: none) and its q. The thread's logit
// zj has been read.
template <class T, int NT, class Map, class Listed>
__device__ __forceinline__ void distill_gradient(const DistillArgs &a, const Part<T, NT> &p, T *out,
                                                 const DistillRow &r, float scale, float zj,
                                                 Map map, Listed listed) {
  if (r.m_a == -__builtin_inff() && r.a_a == r.a_a) {  // every class is masked
    p.zero(out);
    return;
  }
  const ExpAt e(r.m_d, a.c);
  const float f = scale * r.a_d * e.fix;
  if (e.huge)
    map([&](float v) { return f * exp2_raw(e.x_huge(v)); });
  else
    map([&](float v) { return f * exp2_raw(e.x_plain(v)); });
  float q;
  const int id = listed(&q);
  __syncthreads();
  if (id >= p.begin && id < p.end)
    out[id] = Row<T>::down(scale * (r.a_a * exp2_raw((zj - r.m_a) * a.c) - q));
}

// From the sums of a row: its loss, statistics and gradient (of one part).
template <bool TAIL, class T, int NT, class Map>
__device__ __forceinline__ void distill_finish(const DistillArgs &a, ListLds &l, int64_t row,
                                               int part, const Part<T, NT> &p, const Soft &dense,
                                               int id, float zj, float w, Map map) {
  const int tid = threadIdx.x;
  if (tid < kWave) {
    float top, log_z, rest_loss, loss = 0.0f;
    const TeacherMass mass = teacher_sums<TAIL>(a, l, &top, &log_z);
    float listed = 0.0f;
    Soft all = dense;
    if (TAIL) {
      for (int j = tid; j < a.k; j += kWave)
        if (l.id[j] >= 0) all.m = fmaxf(all.m, l.z[j]);
      all.m = lanes_max<kWave>(all.m);
      const float shift = all.m == -__builtin_inff() ? 0.0f : all.m;
      // the 1 that r leaves out is the rest's, or of the first listed class that has it
      const bool first = dense.m != all.m || dense.m == -__builtin_inff();
      all.r = 0.0f;
      soft_join(all, dense, a.c, !first);
      int one = -1;
      for (int j = 0; first && one < 0 && j < a.k; j += kWave) {
        const uint64_t at = __ballot(j + tid < a.k && l.id[j + tid] >= 0 && l.z[j + tid] == all.m);
        if (at) one = j + __builtin_ctzll(at);
      }
      float s = 0.0f;
      for (int j = tid; j < a.k; j += kWave)
        if (l.id[j] >= 0 && j != one) s += exp2_raw((l.z[j] - shift) * a.c);
      s = lanes_sum<kWave>(s);
      listed = one >= 0 ? s + 1.0f : s;
      all.r += s;
      if (all.m == -__builtin_inff()) all.r -= 1.0f;  // no class: S = 0 (or NaN)
      if (all.m == __builtin_inff()) all.r = __builtin_nanf("");
      all.S = 1.0f + all.r;
    }
    const DistillRow r = distill_row<TAIL>(a, dense, all, listed, mass.all, mass.left, &rest_loss);
    const float log_s = log1p_of(all.r);
    for (int j = tid; j < a.k; j += kWave) {
      const float q = l.q[j];
      if (l.id[j] >= 0 && q != 0.0f)
        loss += q * log_ratio<TAIL>(a, l.t[j], top, log_z, l.z[j], all.m, log_s);
    }
    loss = lanes_sum<kWave>(loss) + rest_loss;
    loss += mass.poison;
    if (tid == 0) {
      const bool empty = all.m == -__builtin_inff() && all.S == 0.0f;
      DistillRow o = r;
      if (empty) o = DistillRow{0.0f, 0.0f, -__builtin_inff(), 0.0f};
      l.row = o;
      if (part == 0) {
        if (a.loss) a.loss[row] = empty ? 0.0f : loss * a.t * a.t * w;
        if (a.stats)
          reinterpret_cast<float4 *>(a.stats)[row] = make_float4(o.m_d, o.a_d, o.m_a, o.a_a);
      }
    }
  }
  __syncthreads();
  if (!a.d_logits) return;
  T *out = static_cast<T *>(a.d_logits) + row * a.d_row_stride;
  distill_gradient<T, NT>(a, p, out, l.row, w * a.t, zj, [&](auto f) { map(out, f); }, [&](float *q) {
    *q = tid < a.k ? l.q[tid] : 0.0f;
    return id;
  });
}

// A row of weight 0 is not read.
template <class T, int NT>
__device__ __forceinline__ void distill_no_weight(const DistillArgs &a, int64_t row, int part,
                                                  const Part<T, NT> &p) {
  if (part == 0 && threadIdx.x == 0) {
    if (a.loss) a.loss[row] = 0.0f;
    if (a.stats)
      reinterpret_cast<float4 *>(a.stats)[row] =
          make_float4(0.0f, 0.0f, -__builtin_inff(), 0.0f);
  }
  if (a.d_logits) p.zero(static_cast<T *>(a.d_logits) + row * a.d_row_stride);
}

// KEEP: the row's vectors stay in registers for the gradient, KEEP a thread (0: they are read
// again).
template <class T, int NT, bool TAIL, int KEEP>
__global__ __launch_bounds__(NT) void distill_block_kernel(DistillArgs a) {
  constexpr int N = Row<T>::n;
  extern __shared__ uint32_t listed[];  // TAIL: a bit for each class of the part
  __shared__ BlockLds<NT> lds;
  __shared__ ListLds list;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  const Part<T, NT> p(z, part, a.part_len, a.classes);
  const float w = a.weights ? a.weights[row] : 1.0f;
  if (w == 0.0f) {
    if (a.parts == 1) distill_no_weight<T, NT>(a, row, part, p);
    return;
  }
  if (TAIL)
    for (int i = tid; i * 32 < p.end - p.begin; i += NT) listed[i] = 0u;
  if (TAIL) __syncthreads();
  bool wrong = false;
  int id = list_entry(a, row, &wrong);
  float zj = 0.0f;
  if (id >= p.begin && id < p.end) {
    zj = Row<T>::up(z[id]);
    if (TAIL) atomicOr(&listed[(id - p.begin) >> 5], 1u << ((id - p.begin) & 31));
  }
  if (TAIL) __syncthreads();
  // a listed class counts apart from the rest
  auto hide = [&](int i, float *v) {
    if (!TAIL) return;
    const int o = i - p.begin;
    if (i >= p.end) return;
    const uint32_t bits = (listed[o >> 5] >> (o & 31)) & ((1u << N) - 1u);
    if (bits == 0) return;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (bits >> j & 1u) v[j] = -__builtin_inff();
  };
  typename Part<T, NT>::template Kept<KEEP ? KEEP : 4> kept;
  if (KEEP) p.load(kept);
  Soft s;
  auto take = [&](int at, auto &v) {
    constexpr int W = sizeof(v) / sizeof(v[0]);
    float cm = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < W; ++u) {
      hide(at + tid * N + u * NT * N, v[u]);
#pragma unroll
      for (int j = 0; j < N; ++j) cm = fmaxf(cm, v[u][j]);
    }
    soft_add<W * N, false>(s, &v[0][0], cm, a.c);
  };
  if (KEEP)
    p.scan(kept, take);
  else
    p.scan(take);
  int n = 0;
  s = soft_finish<T, NT, false>(lds, s, p, a.c, n, hide);
  if (a.parts > 1) {
    if (tid == 0) a.part_sum[blockIdx.x] = make_float2(s.m, s.r);
    if (id >= p.begin && id < p.end) a.list_z[row * a.k + tid] = zj;
    return;
  }
  id = put_list(a, list, row, id, zj, wrong);
  distill_finish<TAIL>(a, list, row, 0, p, s, id, zj, w, [&](T *out, auto f) {
    if (KEEP)
      p.map(kept, out, f);
    else
      p.map(out, f);
  });
}

// Joins the sums of a row's parts (in their order), and finishes one part.
template <class T, int NT, bool TAIL>
__global__ __launch_bounds__(NT) void distill_join_kernel(DistillArgs a) {
  __shared__ ListLds list;
  const int tid = threadIdx.x;
  const int blocks = a.d_logits ? a.parts : 1;
  const int64_t row = blockIdx.x / blocks;
  const int part = blockIdx.x % blocks;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  const Part<T, NT> p(z, part, a.part_len, a.classes);
  const float w = a.weights ? a.weights[row] : 1.0f;
  if (w == 0.0f) {
    distill_no_weight<T, NT>(a, row, part, p);
    return;
  }
  bool wrong = false;
  int id = list_entry(a, row, &wrong);
  const float zj = id >= 0 ? a.list_z[row * a.k + tid] : 0.0f;
  int n = 0;
  const Soft s = soft_join_parts(a.parts, a.c, n, [&](int p, int &) {
    const float2 q = a.part_sum[row * a.parts + p];
    Soft b;
    b.m = q.x;
    b.r = q.y;
    return b;
  });
  id = put_list(a, list, row, id, zj, wrong);
  distill_finish<TAIL>(a, list, row, part, p, s, id, zj, w, [&](T *out, auto f) { p.map(out, f); });
}

// The gradient alone, from the statistics.
template <class T, int NT, bool TAIL>
__global__ __launch_bounds__(NT) void distill_grad_block_kernel(DistillArgs a) {
  __shared__ ListLds list;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  T *out = static_cast<T *>(a.d_logits) + row * a.d_row_stride;
  const Part<T, NT> p(z, part, a.part_len, a.classes);
  const float w = a.weights ? a.weights[row] : 1.0f;
  if (w == 0.0f) {
    p.zero(out);
    return;
  }
  bool wrong = false;
  const int entry = list_entry(a, row, &wrong);
  const float zj = entry >= p.begin && entry < p.end ? Row<T>::up(z[entry]) : 0.0f;
  const float4 s = reinterpret_cast<const float4 *>(a.stats)[row];
  if (a.d_logits == a.logits) __syncthreads();
  distill_gradient<T, NT>(
      a, p, out, DistillRow{s.x, s.y, s.z, s.w}, w * a.t, zj,
      [&](auto f) { p.map(out, f); }, [&](float *q) {
        const int id = put_list(a, list, row, entry, zj, wrong);
        if (tid < kWave) {
          float top, log_z;
          (void)teacher_sums<TAIL>(a, list, &top, &log_z);
        }
        __syncthreads();
        *q = tid < a.k ? list.q[tid] : 0.0f;
        return id;
      });
}

}  // namespace tmnn_hip
