// logprob_kernel.hpp -- log-probabilities of given classes, their rank, the
// entropy and the best alternatives of rows of logits, and the gradient of all
// of these.
//
//   log p_v = (z_v - m) / T - ln S           H = ln S - ln2 E / S
//   d z_v = 1/T [ p_v (A + B log p_v) + g_token [v = token] + sum_j g_j [v = top_j] ],
//   A = -(g_token + sum_j g_j + g_H H),  B = -g_H
//
// Short rows (one vector a lane on up to 64 lanes) stay in registers, several
// rows to a wave. Longer rows are read once by a block, or by several blocks
// whose sums and best classes a second kernel joins (few rows).
#pragma once

#include "logits_common.hpp"

namespace tmnn_hip {

struct LogprobArgs {
  const void *logits;
  int64_t row_stride;
  const void *tokens;  // null: no class is given
  int32_t wide_index;
  int32_t rows, classes, top_k;
  int32_t parts, part_len;  // blocks of a row and the classes of each
  float c;                  // log2(e) / T
  float inv_t;
  float *logprob, *entropy;
  int32_t *rank;
  float *stats;  // [rows][2]: m, S
  int32_t *top_ids;
  float *top_logprobs;
  // sums of a row's parts, [rows][parts]: m, r, E, rank; [rows][parts][top_k] keys
  float4 *part_sum;
  uint64_t *part_key;
  // backward
  const float *d_logprob, *d_entropy, *d_top;
  const float *entropy_in, *stats_in;
  const int32_t *top_in;
  void *d_logits;
  int64_t d_row_stride;
};

constexpr int kMaxTop = 128;
constexpr int kLogitVecs = 4;  // vectors a thread has in flight

// The outputs of a row that do not come from its selection. S == 0: every class
// is masked. S not finite: the row holds a NaN or +inf.
__device__ __forceinline__ void put_row(const LogprobArgs &a, int64_t row, const Soft &s,
                                        int64_t token, float zt, int rank) {
  const float nan = __builtin_nanf(""), inf = __builtin_inff();
  const float m = s.m, S = s.S, E = s.E;
  const bool empty = S == 0.0f, bad = !(S < inf) || m == inf;
  const float log_s = log1pf(s.r);
  if (a.entropy) a.entropy[row] = bad ? nan : empty ? 0.0f : log_s - kLn2 * (E / S);
  if (a.stats) {
    a.stats[2 * row] = m;
    a.stats[2 * row + 1] = bad ? nan : S;
  }
  const bool known = token >= 0 && token < a.classes;
  if (a.logprob) {
    float lp = 0.0f;
    if (token >= a.classes)
      lp = nan;
    else if (token >= 0)
      lp = bad ? nan : empty ? -inf : (zt - m) * a.inv_t - log_s;
    a.logprob[row] = lp;
  }
  if (a.rank) a.rank[row] = known && !bad && !empty ? rank : -1;
}

__device__ __forceinline__ void put_top(const LogprobArgs &a, int64_t row, int j, float z, int id,
                                        float m, float log_s) {
  a.top_ids[row * a.top_k + j] = id;
  a.top_logprobs[row * a.top_k + j] = (z - m) * a.inv_t - log_s;
}
__device__ __forceinline__ void put_no_top(const LogprobArgs &a, int64_t row, int j, bool bad) {
  a.top_ids[row * a.top_k + j] = -1;
  a.top_logprobs[row * a.top_k + j] = bad ? __builtin_nanf("") : -__builtin_inff();
}

// ---- short rows -----------------------------------------------------------------

constexpr int kGroupThreads = 256;

template <class T, int G>
__global__ __launch_bounds__(kGroupThreads) void logprob_group_kernel(LogprobArgs a) {
  constexpr int N = Row<T>::n;
  const int lane = threadIdx.x & (G - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kGroupThreads / G) + threadIdx.x / G;
  const bool live = row < a.rows;
  const T *z = static_cast<const T *>(a.logits) + (live ? row : 0) * a.row_stride;
  float v[N];
  load_vec<T>(z, lane * N, live ? a.classes : 0, v);
  int64_t token = -1;
  if (live && a.tokens) token = load_index(a.tokens, row, a.wide_index);
  const bool known = token >= 0 && token < a.classes;
  const float zt = known ? Row<T>::up(z[token]) : 0.0f;
  float m = v[0];
#pragma unroll
  for (int j = 1; j < N; ++j) m = fmaxf(m, v[j]);
  m = lanes_max<G>(m);
  const float shift = m == -__builtin_inff() ? 0.0f : m;
  Soft s;
  s.m = m;
  s.r = 0.0f;
  int rank = 0, best_n = 0;  // best_n: classes of the largest logit, whose terms are 1
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float x = (v[j] - shift) * a.c, e = exp2_raw(x);
    s.r += v[j] == m ? 0.0f : e;
    best_n += v[j] == m;
    s.E = __builtin_fmaf(e, fmaxf(x, -200.0f), s.E);
    rank += v[j] > zt || (v[j] == zt && lane * N + j < token);
  }
  s.r = lanes_sum<G>(s.r);
  s.E = lanes_sum<G>(s.E);
  rank = lanes_isum<G>(rank);
  best_n = lanes_isum<G>(best_n);
  if (m == -__builtin_inff()) best_n = 0;
  if (m == __builtin_inff()) s.r = __builtin_nanf("");
  s.r += static_cast<float>(best_n - 1);
  s.S = 1.0f + s.r;
  if (live && lane == 0) put_row(a, row, s, token, zt, rank);
  if (a.top_k == 0) return;
  const bool bad = !(s.S < __builtin_inff());
  const float log_s = log1pf(s.r);
  uint64_t key[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    key[j] = v[j] > -__builtin_inff() && !bad ? key_of(v[j], lane * N + j) : 0;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t best = key[0];
#pragma unroll
    for (int j = 1; j < N; ++j) best = key[j] > best ? key[j] : best;
    best = lanes_key_max<G>(best);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (key[j] == best) key[j] = 0;
    if (live && lane == (k & (G - 1))) {
      if (best != 0)
        put_top(a, row, k, value_of(static_cast<uint32_t>(best >> 32)), key_index(best), m, log_s);
      else
        put_no_top(a, row, k, bad);
    }
  }
}

// ---- long rows ---------------------------------------------------------------------

template <int NT>
struct BlockLds {
  float m[NT / kWave], R[NT / kWave], S[NT / kWave], E[NT / kWave];
  int n[NT / kWave];
};

// The block's sum from its threads', in every thread, and the total of `n`.
template <int NT, bool ENT>
__device__ __forceinline__ Soft soft_block(BlockLds<NT> &l, Soft s, float c, int &n) {
  constexpr int W = NT / kWave;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  soft_lanes<kWave, ENT>(s, c);
  n = lanes_isum<kWave>(n);
  if (W == 1) return s;
  if (lane == 0) {
    l.m[wave] = s.m;
    l.R[wave] = s.R;
    l.S[wave] = s.S;
    l.E[wave] = s.E;
    l.n[wave] = n;
  }
  __syncthreads();
  const int i = lane & (W - 1);
  Soft o;
  o.m = l.m[i];
  o.R = l.R[i];
  o.S = l.S[i];
  o.E = l.E[i];
  n = lanes_isum<W>(l.n[i]);
  soft_lanes<W, ENT>(o, c);
  return o;
}

// Calls take(at, v) for the classes begin .. end of a row: v[W][N] are W vectors of
// the thread, NT N classes apart, the block's first at `at`. U vectors are in flight;
// what does not fill them is loaded at once too, and taken one by one.
template <class T, int NT, class Take>
__device__ __forceinline__ void scan_part(const T *z, int begin, int end, Take take) {
  constexpr int N = Row<T>::n, U = kLogitVecs;
  const int mine = static_cast<int>(threadIdx.x) * N;
  int at = begin;
  for (; at + NT * N * U <= end; at += NT * N * U) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) widen<T>(load_raw(z + at + mine + u * NT * N), v[u]);
    take(at, v);
  }
  if (at >= end) return;
  float v[U][1][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (at + u * NT * N < end) load_vec<T>(z, at + mine + u * NT * N, end, v[u][0]);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (at + u * NT * N < end) take(at + u * NT * N, v[u]);
}

// The block's sum of x, in every thread.
template <int NT>
__device__ __forceinline__ float block_sum(BlockLds<NT> &l, float x) {
  x = lanes_sum<kWave>(x);
  if (NT == kWave) return x;
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) l.S[threadIdx.x / kWave] = x;
  __syncthreads();
  return lanes_sum<NT / kWave>(l.S[threadIdx.x & (NT / kWave - 1)]);
}

// Sums of huge logits (|m c| above kPlainShift) again, differences first.
template <class T, int NT, bool ENT, class Hide>
__device__ __forceinline__ Soft soft_huge(BlockLds<NT> &l, const T *z, int begin, int end, float m,
                                          float c, Hide hide) {
  constexpr int N = Row<T>::n;
  Soft s;
  for (int i = begin + static_cast<int>(threadIdx.x) * N; i < end; i += NT * N) {
    float v[N];
    load_vec<T>(z, i, end, v);
    hide(i, v);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = (v[j] - m) * c, e = exp2_raw(x);
      s.S += e;
      if (ENT) s.E = __builtin_fmaf(e, fmaxf(x, -200.0f), s.E);
    }
  }
  s.m = m;
  s.S = m == __builtin_inff() ? __builtin_nanf("") : block_sum<NT>(l, s.S);
  s.E = ENT ? block_sum<NT>(l, s.E) : 0.0f;
  s.r = s.S - 1.0f;
  return s;
}

// The block's finished sum from its threads' (`n`: see soft_block). `hide(i, v)`
// masks classes of the vector v at i that do not count.
template <class T, int NT, bool ENT, class Hide>
__device__ __forceinline__ Soft soft_finish(BlockLds<NT> &l, const Soft &mine, const T *z,
                                            int begin, int end, float c, int &n, Hide hide) {
  constexpr int N = Row<T>::n;
  Soft s = soft_block<NT, ENT>(l, mine, c, n);
  if (soft_is_huge(s.m, c)) return soft_huge<T, NT, ENT>(l, z, begin, end, s.m, c, hide);
  const float R = s.R;
  soft_settle(s, c);
  if (!(s.S < kPeaked) || s.S == 0.0f) return s;
  // One class outweighs all others: its thread sums up its others again without it.
  float r = 0.0f;
  if (mine.m == s.m) {
    for (int i = begin + static_cast<int>(threadIdx.x) * N; i < end; i += NT * N) {
      float v[N];
      load_vec<T>(z, i, end, v);
      hide(i, v);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (v[j] != s.m) r += exp2_raw((v[j] - s.m) * c);
    }
  } else {
    r = mine.S * exp2_raw(mine.R - R) * exp2f(-__builtin_fmaf(s.m, c, -R));
  }
  r = block_sum<NT>(l, r);
  s.r = r;
  s.S = 1.0f + r;
  return s;
}

// One part of a row: its sums, the count of its classes before the token, and
// its best classes. `parts` == 1: the row's outputs; else to the workspace.
template <class T, int NT>
__global__ __launch_bounds__(NT) void logprob_block_kernel(LogprobArgs a) {
  constexpr int N = Row<T>::n;
  __shared__ BlockLds<NT> lds;
  __shared__ SelectLds<NT> sel;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  const int begin = part * a.part_len;
  const int end = begin + a.part_len < a.classes ? begin + a.part_len : a.classes;
  const int64_t token = a.tokens ? load_index(a.tokens, row, a.wide_index) : -1;
  const bool known = token >= 0 && token < a.classes;
  const float zt = known ? Row<T>::up(z[token]) : __builtin_inff();
  // classes of this part come before the token's only below `tok` (the fill past
  // the end, -inf, must not count where the token itself is masked)
  const int tok = known ? (token < end ? static_cast<int>(token) : end) : 0;
  const float above = next_above(zt);

  Soft s;
  int rank = 0, first = begin;  // `first`: the vector of the first maximum
  // W vectors of the thread, the first at i, NT N classes apart. Classes that come
  // before the token's: at least its logit up to its own place, above it from there
  // on (`at`: the first class of the block's W vectors).
  auto take = [&](int at, auto &v) {
    constexpr int W = sizeof(v) / sizeof(v[0]);
    const int i = at + tid * N;
    float vm[W], cm;
#pragma unroll
    for (int u = 0; u < W; ++u) {
      vm[u] = v[u][0];
#pragma unroll
      for (int j = 1; j < N; ++j) vm[u] = fmaxf(vm[u], v[u][j]);
    }
    cm = vm[0];
#pragma unroll
    for (int u = 1; u < W; ++u) cm = fmaxf(cm, vm[u]);
    if (cm > s.m) {
#pragma unroll
      for (int u = W - 1; u >= 0; --u)
        if (vm[u] == cm) first = i + u * NT * N;
    }
    soft_add<W * N, true>(s, &v[0][0], cm, a.c);
    if (cm >= zt) {
      if (at + W * NT * N <= tok || at > tok) {
        const float t = at > tok ? above : zt;
#pragma unroll
        for (int u = 0; u < W; ++u)
#pragma unroll
          for (int j = 0; j < N; ++j) rank += v[u][j] >= t;
      } else {
#pragma unroll
        for (int u = 0; u < W; ++u) {
          const int before = tok - i - u * NT * N;
#pragma unroll
          for (int j = 0; j < N; ++j) rank += v[u][j] >= (j < before ? zt : above);
        }
      }
    }
  };
  scan_part<T, NT>(z, begin, end, take);
  const float mine = s.m;
  s = soft_finish<T, NT, true>(lds, s, z, begin, end, a.c, rank, [](int, float *) {});

  const bool whole = a.parts == 1;
  if (tid == 0) {
    if (whole)
      put_row(a, row, s, token, zt, rank);
    else
      a.part_sum[blockIdx.x] = make_float4(s.m, s.r, s.E, __int_as_float(rank));
  }
  if (a.top_k == 0) return;
  const bool bad = !(s.S < __builtin_inff()) || s.m == __builtin_inff();
  const float log_s = log1pf(s.r);
  int got = 0;
  if (!bad && s.S != 0.0f) {
    const uint64_t key =
        mine > -__builtin_inff()
            ? static_cast<uint64_t>(order_of(mine)) << 32 | (0xffffffffu - static_cast<uint32_t>(first + N - 1))
            : 0;
    const int vectors = (end - begin + NT * N - 1) / (NT * N);
    auto visit = [&](int thread, int it, auto f) {
      const int i = begin + (it * NT + thread) * N;
      float v[N];
      load_vec<T>(z, i, end, v);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (v[j] > -__builtin_inff()) f(key_of(v[j], i + j));
    };
    got = block_select<NT>(sel, key, a.top_k, vectors, visit, [&](int j, uint64_t q) {
      if (whole)
        put_top(a, row, j, value_of(static_cast<uint32_t>(q >> 32)), key_index(q), s.m, log_s);
      else
        a.part_key[static_cast<int64_t>(blockIdx.x) * a.top_k + j] = q;
    });
  }
  for (int j = got + tid; j < a.top_k; j += NT) {
    if (whole)
      put_no_top(a, row, j, bad);
    else
      a.part_key[static_cast<int64_t>(blockIdx.x) * a.top_k + j] = 0;
  }
}

// Joins the parts of a row.
constexpr int kJoinThreads = 512;
constexpr int kMaxParts = 128;

template <class T>
__global__ __launch_bounds__(kJoinThreads) void logprob_join_kernel(LogprobArgs a) {
  __shared__ SelectLds<kJoinThreads> sel;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  int rank = 0;
  const Soft s = soft_join_parts(a.parts, a.c, rank, [&](int p, int &n) {
    const float4 q = a.part_sum[row * a.parts + p];
    Soft b;
    b.m = q.x;
    b.r = q.y;
    b.E = q.z;
    n = __float_as_int(q.w);
    return b;
  });
  const bool bad = !(s.S < __builtin_inff()) || s.m == __builtin_inff();
  if (tid == 0) {
    const int64_t token = a.tokens ? load_index(a.tokens, row, a.wide_index) : -1;
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const float zt = token >= 0 && token < a.classes ? Row<T>::up(z[token]) : 0.0f;
    put_row(a, row, s, token, zt, rank);
  }
  if (a.top_k == 0) return;
  const float m = s.m, log_s = log1pf(s.r);
  int got = 0;
  if (!bad && s.S != 0.0f) {
    const uint64_t *keys = a.part_key + row * a.parts * a.top_k;
    const int n = a.parts * a.top_k;
    uint64_t best = 0;
    for (int i = tid; i < n; i += kJoinThreads) best = keys[i] > best ? keys[i] : best;
    auto visit = [&](int thread, int it, auto f) {
      const int i = it * kJoinThreads + thread;
      if (i < n && keys[i] != 0) f(keys[i]);
    };
    const int vectors = (n + kJoinThreads - 1) / kJoinThreads;
    got = block_select<kJoinThreads>(sel, best, a.top_k, vectors, visit, [&](int j, uint64_t q) {
      put_top(a, row, j, value_of(static_cast<uint32_t>(q >> 32)), key_index(q), m, log_s);
    });
  }
  for (int j = got + tid; j < a.top_k; j += kJoinThreads) put_no_top(a, row, j, bad);
}

// ---- gradient ---------------------------------------------------------------------

// A row's gradient: class v gets 2^x (a + b x) with x = c (z_v - m), plus its
// listed terms.
struct LogprobRow {
  float m, a, b;
  int token;       // -1: none, or without a term
  float g_token;   // times 1 / T
  bool skip;       // 0 everywhere
};

// top_sum: the sum of the listed terms; top_any: one of them is not 0; spread(S):
// H - ln S.
template <class Spread>
__device__ __forceinline__ LogprobRow logprob_row(const LogprobArgs &a, int64_t row, float top_sum,
                                                  bool top_any, Spread spread) {
  LogprobRow r;
  const int64_t token = a.tokens && a.d_logprob ? load_index(a.tokens, row, a.wide_index) : -1;
  r.m = a.stats_in[2 * row];
  const float S = a.stats_in[2 * row + 1];
  const float g = token >= 0 ? a.d_logprob[row] : 0.0f;
  const float gh = a.d_entropy ? a.d_entropy[row] : 0.0f;
  r.token = token < a.classes ? static_cast<int>(token) : -1;
  const float h = gh != 0.0f ? spread(S) : 0.0f;
  const float scale = a.inv_t / S;
  r.a = -(g + top_sum + gh * h) * scale;
  r.b = -gh * kLn2 * scale;
  r.g_token = g * a.inv_t;
  if (token >= a.classes && g != 0.0f) r.a = __builtin_nanf("");
  r.skip = S == 0.0f || (g == 0.0f && gh == 0.0f && !top_any);
  return r;
}

template <class T, int G>
__global__ __launch_bounds__(kGroupThreads) void logprob_grad_group_kernel(LogprobArgs a) {
  constexpr int N = Row<T>::n;
  __shared__ int owner[kGroupThreads * N];    // the first entry that lists a class
  __shared__ float extra[kGroupThreads * N];  // its term
  const int lane = threadIdx.x & (G - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kGroupThreads / G) + threadIdx.x / G;
  const bool live = row < a.rows;
  const T *z = static_cast<const T *>(a.logits) + (live ? row : 0) * a.row_stride;
  float v[N];
  load_vec<T>(z, lane * N, live ? a.classes : 0, v);
  int *own = owner + (threadIdx.x - lane) * N;
  float *ext = extra + (threadIdx.x - lane) * N;
  const int k = live && a.d_top ? a.top_k : 0;
  float top_sum = 0.0f, any = 0.0f;
  if (a.d_top) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      own[lane * N + j] = 0x7fffffff;
      ext[lane * N + j] = 0.0f;
    }
    wave_fence();
    for (int j = lane; j < k; j += G) {
      const int id = a.top_in[row * a.top_k + j];
      if (id >= 0 && id < a.classes) atomicMin(&own[id], j);
    }
    wave_fence();
    for (int j = lane; j < k; j += G) {
      const int id = a.top_in[row * a.top_k + j];
      if (id >= 0 && id < a.classes && own[id] == j) {
        const float g = a.d_top[row * a.top_k + j];
        ext[id] = g * a.inv_t;
        top_sum += g;
        if (g != 0.0f) any = 1.0f;
      }
    }
    wave_fence();
    top_sum = lanes_sum<G>(top_sum);
    any = lanes_max<G>(any);
  }
  const float m = live ? a.stats_in[2 * row] : 0.0f;
  float x[N], e[N], E = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    x[j] = (v[j] - m) * a.c;
    e[j] = exp2_raw(x[j]);
    x[j] = fmaxf(x[j], -200.0f);
    E = __builtin_fmaf(e[j], x[j], E);
  }
  // H - ln S from the row itself: the entropy's own rounding does not enter
  E = lanes_sum<G>(E);
  if (!live) return;
  const LogprobRow r =
      logprob_row(a, row, top_sum, any != 0.0f, [&](float S) { return -kLn2 * (E / S); });
  float d[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float t = e[j] * __builtin_fmaf(r.b, x[j], r.a);
    if (a.d_top) t += ext[lane * N + j];
    if (lane * N + j == r.token) t += r.g_token;
    d[j] = r.skip ? 0.0f : t;
  }
  store_vec<T>(static_cast<T *>(a.d_logits) + row * a.d_row_stride, lane * N, a.classes, d);
}

// Writes f(z) for the classes begin .. end of a row, all of a block's threads.
template <class T, int NT, class F>
__device__ __forceinline__ void map_part(const T *z, T *out, int begin, int end, F f) {
  constexpr int N = Row<T>::n, U = kLogitVecs;
  const int tid = threadIdx.x;
  int at = begin;
  for (; at + NT * N * U <= end; at += NT * N * U) {
    const int i = at + tid * N;
    typename Row<T>::V raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw(z + i + u * NT * N);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[N];
      widen<T>(raw[u], v);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = f(v[j]);
      store_vec<T>(out, i + u * NT * N, end, v);
    }
  }
  for (int i = at + tid * N; i < end; i += NT * N) {
    float v[N];
    load_vec<T>(z, i, end, v);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = f(v[j]);
    store_vec<T>(out, i, end, v);
  }
}

template <class T, int NT>
__device__ __forceinline__ void zero_part(T *out, int begin, int end) {
  constexpr int N = Row<T>::n;
  const float v[N] = {};
  for (int i = begin + static_cast<int>(threadIdx.x) * N; i < end; i += NT * N)
    store_vec<T>(out, i, end, v);
}

// One part of a row. The listed classes and the token are written after all
// others; their logits are read before the block writes anything, so that the
// gradient may take the place of the logits. NT > top_k: a thread for each listed class
// and one for the token.
template <class T, int NT>
__global__ __launch_bounds__(NT) void logprob_grad_block_kernel(LogprobArgs a) {
  __shared__ int list[kMaxTop];
  __shared__ float term[kMaxTop];
  __shared__ float sums[2];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  T *out = static_cast<T *>(a.d_logits) + row * a.d_row_stride;
  const int begin = part * a.part_len;
  const int end = begin + a.part_len < a.classes ? begin + a.part_len : a.classes;
  const int k = a.d_top ? a.top_k : 0;
  float top_sum = 0.0f;
  bool top_any = false;
  int mine = -1;
  float g = 0.0f;
  if (k > 0) {
    if (tid < k) {
      const int id = a.top_in[row * a.top_k + tid];
      list[tid] = id >= 0 && id < a.classes ? id : -1;
    }
    __syncthreads();
    if (tid < k) {
      mine = list[tid];
      for (int j = 0; j < tid; ++j)
        if (list[j] == mine) mine = -1;  // a class counts by its first entry
      g = mine >= 0 ? a.d_top[row * a.top_k + tid] : 0.0f;
      term[tid] = g;
    }
    __syncthreads();
    if (tid < kWave) {
      float s = 0.0f, any = 0.0f;
      for (int j = tid; j < k; j += kWave) {
        s += term[j];
        if (term[j] != 0.0f) any = 1.0f;
      }
      s = lanes_sum<kWave>(s);
      any = lanes_max<kWave>(any);
      if (tid == 0) {
        sums[0] = s;
        sums[1] = any;
      }
    }
    __syncthreads();
    top_sum = sums[0];
    top_any = sums[1] != 0.0f;
  }
  const LogprobRow r = logprob_row(a, row, top_sum, top_any,
                                   [&](float S) { return a.entropy_in[row] - logf(S); });
  if (r.skip) {
    zero_part<T, NT>(out, begin, end);
    return;
  }
  g *= a.inv_t;
  if (tid == k) {
    mine = r.token;
    for (int j = 0; j < k; ++j)
      if (list[j] == mine) mine = -1;  // its entry's thread writes it
    g = r.g_token;
  } else if (mine >= 0 && mine == r.token) {
    g += r.g_token;
  }
  if (mine < begin || mine >= end) mine = -1;
  const float zm = mine >= 0 ? Row<T>::up(z[mine]) : 0.0f;
  __syncthreads();
  const ExpAt e(r.m, a.c);
  // 2^x of the fma form carries `fix`, and its x the same correction
  const float rho = e.huge ? 0.0f : __builtin_fmaf(r.m, a.c, -e.R);
  const float fa = __builtin_fmaf(-r.b, rho, r.a) * e.fix, fb = r.b * e.fix;
  if (e.huge) {
    map_part<T, NT>(z, out, begin, end, [&](float v) {
      const float x = e.x_huge(v);
      return exp2_raw(x) * __builtin_fmaf(fb, fmaxf(x, -200.0f), fa);
    });
  } else {
    map_part<T, NT>(z, out, begin, end, [&](float v) {
      const float x = e.x_plain(v);
      return exp2_raw(x) * __builtin_fmaf(fb, fmaxf(x, -200.0f), fa);
    });
  }
  __syncthreads();
  if (mine >= 0) {
    const float x = e.x(zm);
    out[mine] = Row<T>::down(exp2_raw(x) * __builtin_fmaf(r.b, fmaxf(x, -200.0f), r.a) + g);
  }
}

}  // namespace tmnn_hip
