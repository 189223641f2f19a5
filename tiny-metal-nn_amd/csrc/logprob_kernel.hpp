// logprob_kernel.hpp -- log-probabilities of given classes, their rank, the
// entropy and the best alternatives of rows of logits, and the gradient of all
// of these.
//
//   log p_v = (z_v - m) / T - ln S           H = ln S - ln2 E / S
//   d z_v = 1/T [ p_v (A + B log p_v) + g_token [v = token] + sum_j g_j [v = top_j] ],
//   A = -(g_token + sum_j g_j + g_H H),  B = -g_H
//
// Short rows (up to 16 classes a lane on up to 64 lanes) stay in registers, several
// rows to a wave. Longer rows are read once by a block, or by several blocks
// whose sums and best classes a second kernel joins (few rows).
//
// Bound: the forward pass by reading the logits (4096 x 131072 bf16 with 20 alternatives
// 195 us, 5.5 TB/s; without alternatives 184 us, the rest is the selection at each block's
// end; the vector units issue in 88% of the time, yet counting the ranks with scalar
// instructions, two vector ones a class less, did not change it), the gradient by reading
// and writing them (8192 x 65536 bf16 380 us, 5.6 TB/s). Few rows are bound by latency:
// one block's loads, sums and selection (one row of 32768 bf16: 8.1 us; in parts and a join 4.8 +
// 6.5), or two dependent kernels for rows of more than 4096 vectors.
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
  int32_t part_threads;     // threads of a block (a power of two)
  float c;                  // log2(e) / T
  float inv_t;
  float *logprob, *entropy;
  int32_t *rank;
  float *stats;  // [rows][2]: m, S
  int32_t *top_ids;
  float *top_logprobs;
  // sums of a row's parts, [rows][parts]: m, r, E, rank; [rows][parts][part_threads] keys
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
  const float log_s = log1p_of(s.r);
  if (a.entropy) a.entropy[row] = bad ? nan : empty ? 0.0f : log_s - kLn2 * quotient(E, S);
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

// A row in the registers of G lanes, NV vectors each: vector u of a lane holds the
// classes from (u G + lane) N on. 16 classes a lane keep what a row costs beyond them (sums
// over lanes, logarithms, entries) in few instructions, which are what bounds short
// rows: 2^20 rows of 16 bf16 classes take 17 us for their gradient (4.0 TB/s), of 16 fp32
// classes 33 us. One lane a row takes its wave's rows, where they are adjacent, through LDS: its
// own 16-byte accesses would lie 64 bytes apart (fp32, direct: 42 us).
template <class T, int G, int NV>
struct Group {
  static constexpr int N = Row<T>::n, E = N * NV;
  static constexpr int rows = kGroupThreads / G;
  // LDS words a lane, so that 16 lanes' 16-byte accesses meet different banks
  static constexpr int pitch = E % 8 == 0 ? E + 4 : E;
  static constexpr int words = kGroupThreads * pitch;
  int lane;
  int64_t row;
  __device__ __forceinline__ Group()
      : lane(threadIdx.x & (G - 1)),
        row(static_cast<int64_t>(blockIdx.x) * rows + threadIdx.x / G) {}
  __device__ __forceinline__ int at(int u) const { return (u * G + lane) * N; }
  __device__ __forceinline__ int index(int e) const { return at(e / N) + e % N; }

  // The rows of the wave as one run of elements in LDS; a free vector after every
  // fourth keeps rows of four from meeting in the same banks.
  static __device__ __forceinline__ int slot(int element) {
    const int q = element / N;
    return (q + q / 4) * N + element % N;
  }
  struct Run {
    T *lds;
    int64_t first;  // element of the run's start
    int n, lane;
  };
  __device__ __forceinline__ Run run_of(int *word, int64_t all_rows, int classes) const {
    const int wave = threadIdx.x / kWave;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * rows + wave * kWave;
    const int64_t left = all_rows - first;
    Run r;
    r.lds = reinterpret_cast<T *>(word + wave * kWave * pitch);
    r.first = first * classes;
    r.n = left <= 0 ? 0 : static_cast<int>(left < kWave ? left : kWave) * classes;
    r.lane = threadIdx.x & (kWave - 1);
    return r;
  }
  static constexpr int kSteps = (E + N - 1) / N;  // vectors a lane moves of a full run

  // The row's classes (-inf where it is not `live` and past its end).
  __device__ __forceinline__ void load_rows(const void *logits, int64_t stride, int64_t all_rows,
                                            int classes, bool live, int *word, float *v) const {
    if (G == 1 && NV > 1 && stride == classes) {
      const Run r = run_of(word, all_rows, classes);
      const T *z = static_cast<const T *>(logits) + r.first;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int o = (i * kWave + r.lane) * N;
        if (o + N <= r.n)
          *reinterpret_cast<typename Row<T>::A *>(r.lds + slot(o)) = load_raw(z + o);
        else
          for (int j = o; j < r.n; ++j) r.lds[slot(j)] = z[j];
      }
      wave_fence();
      const int mine = r.lane * classes;
      if (classes % N == 0) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          if (live && u * N < classes) {
            const typename Row<T>::A raw = *reinterpret_cast<const typename Row<T>::A *>(r.lds + slot(mine + u * N));
#pragma unroll
            for (int j = 0; j < N; ++j) v[u * N + j] = Row<T>::up(raw[j]);
          } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[u * N + j] = -__builtin_inff();
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          v[e] = live && e < classes ? Row<T>::up(r.lds[slot(mine + e)]) : -__builtin_inff();
      }
      wave_fence();
      return;
    }
    const T *z = static_cast<const T *>(logits) + (live ? row : 0) * stride;
#pragma unroll
    for (int u = 0; u < NV; ++u) load_vec<T>(z, at(u), live ? classes : 0, v + u * N);
  }
  // Every lane of the wave calls it; what the LDS words held is gone.
  __device__ __forceinline__ void store_rows(void *out, int64_t stride, int64_t all_rows,
                                             int classes, int *word, const float *v) const {
    if (G == 1 && NV > 1 && stride == classes) {
      const Run r = run_of(word, all_rows, classes);
      T *z = static_cast<T *>(out) + r.first;
      const int mine = r.lane * classes;
      wave_fence();
      if (classes % N == 0) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
          if (u * N < classes) {
            typename Row<T>::A raw;
#pragma unroll
            for (int j = 0; j < N; ++j) raw[j] = Row<T>::down(v[u * N + j]);
            *reinterpret_cast<typename Row<T>::A *>(r.lds + slot(mine + u * N)) = raw;
          }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e < classes) r.lds[slot(mine + e)] = Row<T>::down(v[e]);
      }
      wave_fence();
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int o = (i * kWave + r.lane) * N;
        if (o + N <= r.n)
          *reinterpret_cast<typename Row<T>::V *>(z + o) =
              *reinterpret_cast<const typename Row<T>::A *>(r.lds + slot(o));
        else
          for (int j = o; j < r.n; ++j) z[j] = r.lds[slot(j)];
      }
      return;
    }
    if (row >= all_rows) return;
    T *z = static_cast<T *>(out) + row * stride;
#pragma unroll
    for (int u = 0; u < NV; ++u) store_vec<T>(z, at(u), classes, v + u * N);
  }
};

template <class T, int G, int NV>
__global__ __launch_bounds__(kGroupThreads) void logprob_group_kernel(LogprobArgs a) {
  constexpr int N = Row<T>::n, E = N * NV;
  __shared__ __attribute__((aligned(16))) int words[G == 1 ? Group<T, G, NV>::words : 1];
  const Group<T, G, NV> g;
  const int64_t row = g.row;
  const bool live = row < a.rows;
  int64_t token = -1;
  if (live && a.tokens) token = load_index(a.tokens, row, a.wide_index);
  float v[E];
  g.load_rows(a.logits, a.row_stride, a.rows, a.classes, live, words, v);
  float m = v[0];
#pragma unroll
  for (int e = 1; e < E; ++e) m = fmaxf(m, v[e]);
  m = lanes_max<G>(m);
  // the token's logit, from the lane that holds it
  float zt = 0.0f;
  const int tok = token >= 0 && token < a.classes ? static_cast<int>(token) : 0;
  if (a.tokens) {
    float mine = v[0];
    const int which = tok / (G * N) * N + (tok & (N - 1));
#pragma unroll
    for (int e = 1; e < E; ++e) mine = which == e ? v[e] : mine;
    zt = G == 1 ? mine : __shfl(mine, tok / N & (G - 1), G);
  }
  const float shift = m == -__builtin_inff() ? 0.0f : m;
  Soft s;
  s.m = m;
  s.r = 0.0f;
  int rank = 0, best_n = 0;  // best_n: classes of the largest logit, whose terms are 1
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float x = (v[e] - shift) * a.c, p = exp2_raw(x);
    s.r += v[e] == m ? 0.0f : p;
    best_n += v[e] == m;
    s.E = __builtin_fmaf(p, fmaxf(x, -200.0f), s.E);
    rank += v[e] > zt || (v[e] == zt && g.index(e) < tok);
  }
  s.r = lanes_sum<G>(s.r);
  s.E = lanes_sum<G>(s.E);
  if (a.tokens) rank = lanes_isum<G>(rank);
  best_n = lanes_isum<G>(best_n);
  if (m == -__builtin_inff()) best_n = 0;
  if (m == __builtin_inff()) s.r = __builtin_nanf("");
  s.r += static_cast<float>(best_n - 1);
  s.S = 1.0f + s.r;
  if (live && g.lane == 0) put_row(a, row, s, token, zt, rank);
  if (a.top_k == 0) return;
  const bool bad = !(s.S < __builtin_inff());
  const float log_s = log1p_of(s.r);
  // one round an alternative: the largest value, then the first class that has it
  uint32_t key[E];
#pragma unroll
  for (int e = 0; e < E; ++e)
    key[e] = v[e] > -__builtin_inff() && !bad ? order_of(v[e]) : 0;
  for (int k = 0; k < a.top_k; ++k) {
    uint32_t best = key[0];
#pragma unroll
    for (int e = 1; e < E; ++e) best = key[e] > best ? key[e] : best;
    uint64_t q = best;
    int mine = 0;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) mine = key[e] == best ? e : mine;
    const int at = (mine / N * G + g.lane) * N + (mine & (N - 1));
    q = lanes_key_max<G>(q << 32 | (0xffffffffu - static_cast<uint32_t>(at)));
    best = static_cast<uint32_t>(q >> 32);
    const bool ours = key_index(q) == at;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (ours && mine == e) key[e] = 0;
    if (live && g.lane == (k & (G - 1))) {
      if (best != 0)
        put_top(a, row, k, value_of(best), key_index(q), m, log_s);
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

// The block's sum from its threads', in every thread; with ENT also E and the total
// of `n`.
template <int NT, bool ENT>
__device__ __forceinline__ Soft soft_block(BlockLds<NT> &l, Soft s, float c, int &n) {
  constexpr int W = NT / kWave;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  soft_lanes<kWave, ENT>(s, c);
  if (ENT) n = lanes_isum<kWave>(n);
  if (W == 1) return s;
  if (lane == 0) {
    l.m[wave] = s.m;
    l.R[wave] = s.R;
    l.S[wave] = s.S;
    if (ENT) {
      l.E[wave] = s.E;
      l.n[wave] = n;
    }
  }
  __syncthreads();
  const int i = lane & (W - 1);
  Soft o;
  o.m = l.m[i];
  o.R = l.R[i];
  o.S = l.S[i];
  if (ENT) {
    o.E = l.E[i];
    n = lanes_isum<W>(l.n[i]);
  }
  soft_lanes<W, ENT>(o, c);
  return o;
}

// A part begin .. end of a row as a block's vectors: vector q belongs to thread q % NT.
template <class T, int NT>
struct Part {
  const T *z;
  int begin, end;
  __device__ __forceinline__ Part(const T *row, int part, int part_len, int classes) : z(row) {
    begin = part * part_len;
    end = begin + part_len < classes ? begin + part_len : classes;
  }
  __device__ __forceinline__ int vectors() const {  // of a thread
    return (end - begin + NT * Row<T>::n - 1) / (NT * Row<T>::n);
  }
  // f(i, v) for the thread's vectors, one after another
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = begin + static_cast<int>(threadIdx.x) * Row<T>::n; i < end; i += NT * Row<T>::n) {
      float v[Row<T>::n];
      load_vec<T>(z, i, end, v);
      f(i, v);
    }
  }
  // f(key) for the classes of a vector of a thread that are not masked
  template <class F>
  __device__ __forceinline__ void keys(int thread, int it, F f) const {
    const int i = begin + (it * NT + thread) * Row<T>::n;
    float v[Row<T>::n];
    load_vec<T>(z, i, end, v);
#pragma unroll
    for (int j = 0; j < Row<T>::n; ++j)
      if (v[j] > -__builtin_inff()) f(key_of(v[j], i + j));
  }
  // take(at, v): v[W][N] are W vectors of the thread, NT N classes apart, the block's
  // first at `at`. U vectors are in flight; where the part does not fill them, they are
  // loaded at once too, and taken one by one.
  template <class Take>
  __device__ __forceinline__ void scan(Take take) const {
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
  // out = f(z) for the part's classes, from its end: what a scan has just read is the
  // likeliest to be in a cache still (1030 x 100000 fp32 distilled: 224 us, 232 us from
  // its begin).
  template <class F>
  __device__ __forceinline__ void map(T *out, F f) const {
    constexpr int N = Row<T>::n, U = kLogitVecs;
    const int mine = static_cast<int>(threadIdx.x) * N;
    const int tiles = (end - begin) / (NT * N * U);
    for (int i = begin + tiles * NT * N * U + mine; i < end; i += NT * N) {
      float v[N];
      load_vec<T>(z, i, end, v);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = f(v[j]);
      store_vec<T>(out, i, end, v);
    }
    for (int t = tiles - 1; t >= 0; --t) {
      const int i = begin + t * NT * N * U + mine;
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
  }
  // The same with up to K vectors of the thread kept in between: load, then any number of
  // scans and one map. The part has at most K NT vectors.
  template <int K>
  struct Kept {
    typename Row<T>::V raw[K];
  };
  template <int K>
  __device__ __forceinline__ void load(Kept<K> &k) const {
    constexpr int N = Row<T>::n;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int i = begin + (u * NT + static_cast<int>(threadIdx.x)) * N;
      if (i + N <= end) {
        k.raw[u] = load_raw(z + i);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) k.raw[u][j] = i + j < end ? z[i + j] : Row<T>::down(-__builtin_inff());
      }
    }
  }
  template <int K, class Take>
  __device__ __forceinline__ void scan(const Kept<K> &k, Take take) const {
    constexpr int N = Row<T>::n, U = kLogitVecs;
    static_assert(K % U == 0, "");
#pragma unroll
    for (int g = 0; g < K; g += U) {
      const int at = begin + g * NT * N;
      if (at >= end) break;
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) widen<T>(k.raw[g + u], v[u]);
      take(at, v);
    }
  }
  template <int K, class F>
  __device__ __forceinline__ void map(const Kept<K> &k, T *out, F f) const {
    constexpr int N = Row<T>::n;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int i = begin + (u * NT + static_cast<int>(threadIdx.x)) * N;
      if (i < end) {
        float v[N];
        widen<T>(k.raw[u], v);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = f(v[j]);
        store_vec<T>(out, i, end, v);
      }
    }
  }
  __device__ __forceinline__ void zero(T *out) const {
    constexpr int N = Row<T>::n;
    const float v[N] = {};
    for (int i = begin + static_cast<int>(threadIdx.x) * N; i < end; i += NT * N)
      store_vec<T>(out, i, end, v);
  }
};

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
__device__ __forceinline__ Soft soft_huge(BlockLds<NT> &l, const Part<T, NT> &p, float m, float c,
                                          Hide hide) {
  Soft s;
  p.each([&](int i, float *v) {
    hide(i, v);
#pragma unroll
    for (int j = 0; j < Row<T>::n; ++j) {
      const float x = (v[j] - m) * c, e = exp2_raw(x);
      s.S += e;
      if (ENT) s.E = __builtin_fmaf(e, fmaxf(x, -200.0f), s.E);
    }
  });
  s.m = m;
  s.S = m == __builtin_inff() ? __builtin_nanf("") : block_sum<NT>(l, s.S);
  s.E = ENT ? block_sum<NT>(l, s.E) : 0.0f;
  s.r = s.S - 1.0f;
  return s;
}

// The block's finished sum from its threads' (`n`: see soft_block). `hide(i, v)`
// masks classes of the vector v at i that do not count.
template <class T, int NT, bool ENT, class Hide>
__device__ __forceinline__ Soft soft_finish(BlockLds<NT> &l, const Soft &mine,
                                            const Part<T, NT> &p, float c, int &n, Hide hide) {
  Soft s = soft_block<NT, ENT>(l, mine, c, n);
  if (soft_is_huge(s.m, c)) return soft_huge<T, NT, ENT>(l, p, s.m, c, hide);
  const float R = s.R;
  soft_settle(s, c);
  if (!(s.S < kPeaked) || s.S == 0.0f) return s;
  // One class outweighs all others: its thread sums up its others again without it.
  float r = 0.0f;
  if (mine.m == s.m) {
    p.each([&](int i, float *v) {
      hide(i, v);
#pragma unroll
      for (int j = 0; j < Row<T>::n; ++j)
        if (v[j] != s.m) r += exp2_raw((v[j] - s.m) * c);
    });
  } else {
    r = mine.S * exp2_raw(mine.R - R) * exp2f(-__builtin_fmaf(s.m, c, -R));
  }
  r = block_sum<NT>(l, r);
  s.r = r;
  s.S = 1.0f + r;
  return s;
}

// One part of a row: its sums, the count of its classes before the token, and
// its best classes. `parts` == 1: the row's outputs; else the sums and the threads' keys
// go to the workspace.
template <class T, int NT>
__global__ __launch_bounds__(NT) void logprob_block_kernel(LogprobArgs a) {
  constexpr int N = Row<T>::n;
  __shared__ BlockLds<NT> lds;
  __shared__ SelectLds<NT> sel;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  const Part<T, NT> p(z, part, a.part_len, a.classes);
  const int64_t token = a.tokens ? load_index(a.tokens, row, a.wide_index) : -1;
  const bool known = token >= 0 && token < a.classes;
  const float zt = known ? Row<T>::up(z[token]) : __builtin_inff();
  // classes of this part come before the token's only below `tok` (the fill past
  // the end, -inf, must not count where the token itself is masked)
  const int tok = known ? (token < p.end ? static_cast<int>(token) : p.end) : 0;
  const float above = next_above(zt);

  Soft s;
  int rank = 0, first = p.begin;  // `first`: the vector of the first maximum
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
  p.scan(take);
  const float mine = s.m;
  s = soft_finish<T, NT, true>(lds, s, p, a.c, rank, [](int, float *) {});

  const bool whole = a.parts == 1;
  if (tid == 0) {
    if (whole)
      put_row(a, row, s, token, zt, rank);
    else
      a.part_sum[blockIdx.x] = make_float4(s.m, s.r, s.E, __int_as_float(rank));
  }
  if (a.top_k == 0) return;
  const uint64_t key = mine > -__builtin_inff()
                           ? static_cast<uint64_t>(order_of(mine)) << 32 |
                                 (0xffffffffu - static_cast<uint32_t>(first + N - 1))
                           : 0;
  if (!whole) {
    a.part_key[static_cast<int64_t>(blockIdx.x) * NT + tid] = key;
    return;
  }
  const bool bad = !(s.S < __builtin_inff()) || s.m == __builtin_inff();
  const float log_s = log1p_of(s.r);
  int got = 0;
  if (!bad && s.S != 0.0f) {
    got = block_select(
        sel, key, a.top_k, p.vectors(), [&](auto f) { f(tid, key); },
        [&](int thread, int it, auto f) { p.keys(thread, it, f); },
        [&](int j, uint64_t q) {
          put_top(a, row, j, value_of(static_cast<uint32_t>(q >> 32)), key_index(q), s.m, log_s);
        });
  }
  for (int j = got + tid; j < a.top_k; j += NT) put_no_top(a, row, j, bad);
}

// Joins the parts of a row.
constexpr int kJoinThreads = 512;
constexpr int kMaxParts = 128;

template <class T>
__global__ __launch_bounds__(kJoinThreads) void logprob_join_kernel(LogprobArgs a) {
  __shared__ SelectLds<kJoinThreads, 1024> sel;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  const int64_t token = a.tokens ? load_index(a.tokens, row, a.wide_index) : -1;
  const float zt = token >= 0 && token < a.classes ? Row<T>::up(z[token]) : 0.0f;
  // the keys of the parts' threads: the first kKept of a thread in registers
  constexpr int kKept = 8;
  const int n = a.parts * a.part_threads;
  const uint64_t *keys = a.part_key + row * n;
  uint64_t kept[kKept], best = 0;
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    const int at = i * kJoinThreads + tid;
    kept[i] = a.top_k > 0 && at < n ? keys[at] : 0;
  }
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
  // (not the wave that searches)
  if (tid == kJoinThreads - kWave) put_row(a, row, s, token, zt, rank);
  if (a.top_k == 0) return;
  const float m = s.m, log_s = log1p_of(s.r);
  int got = 0;
  if (!bad && s.S != 0.0f) {
    // the sources are the parts' threads
    constexpr int N = Row<T>::n;
    const int stride = a.part_threads * N;
#pragma unroll
    for (int i = 0; i < kKept; ++i) best = kept[i] > best ? kept[i] : best;
    for (int i = kKept * kJoinThreads + tid; i < n; i += kJoinThreads)
      best = keys[i] > best ? keys[i] : best;
    auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (kept[i] != 0) f(i * kJoinThreads + tid, kept[i]);
      for (int i = kKept * kJoinThreads + tid; i < n; i += kJoinThreads) f(i, keys[i]);
    };
    auto visit = [&](int source, int it, auto f) {
      const int begin = source / a.part_threads * a.part_len;
      const int end = begin + a.part_len < a.classes ? begin + a.part_len : a.classes;
      const int i = begin + it * stride + (source & (a.part_threads - 1)) * N;
      float v[N];
      load_vec<T>(z, i, end, v);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (v[j] > -__builtin_inff()) f(key_of(v[j], i + j));
    };
    const int vectors = (a.part_len + stride - 1) / stride;
    got = block_select(
        sel, best, a.top_k, vectors, each, visit, [&](int j, uint64_t q) {
          put_top(a, row, j, value_of(static_cast<uint32_t>(q >> 32)), key_index(q), m, log_s);
        });
  }
  for (int j = got + tid; j < a.top_k; j += kJoinThreads) put_no_top(a, row, j, bad);
}

// ---- gradient ---------------------------------------------------------------------

// A row's gradient: class v gets 2^x (a + b x) with x = c (z_v - m), plus its
// listed terms.
//
// Where the best class outweighs all others (S = 1 + r, r < 1/8), its own terms cancel: with g
// listed and w = sum of all that are, T d z = (g - w) / S + g r / S - g_H (H - ln S) / S, the
// first difference 0 for a row with this one term. S holds r to 2^-24 only, 12% of it at
// 1 - p = 2e-7; so r and H - ln S = -ln2 E / S come from a sum over the other classes again.
struct LogprobRow {
  float m, S, a, b;
  int token;       // -1: none, or without a term
  float g_token;   // times 1 / T
  float all;       // w times 1 / T
  float g_entropy;
  float spread;    // g_H (H - ln S) / T
  bool skip;       // 0 everywhere
  bool peaked;
  // H - ln S (where the entropy has a gradient)
  __device__ __forceinline__ void finish(const LogprobArgs &args, float g, float top_sum, float h) {
    const float scale = quotient(args.inv_t, S);
    a = -(g + top_sum + g_entropy * h) * scale;
    b = -g_entropy * kLn2 * scale;
    spread = g_entropy * h * args.inv_t;
  }
  // of the best class of a peaked row, with `g` (times 1 / T) listed; `rest`: r
  __device__ __forceinline__ float best(float g, float rest) const {
    return quotient(__builtin_fmaf(g, rest, (g - all) - spread), S);
  }
};

// top_sum: the sum of the listed terms; top_any: one of them is not 0. `*token_g`: the token's
// term. finish() completes it.
__device__ __forceinline__ LogprobRow logprob_row(const LogprobArgs &a, int64_t row, float top_sum,
                                                  bool top_any, float *token_g) {
  LogprobRow r;
  const int64_t token = a.tokens && a.d_logprob ? load_index(a.tokens, row, a.wide_index) : -1;
  r.m = a.stats_in[2 * row];
  r.S = a.stats_in[2 * row + 1];
  float g = token >= 0 ? a.d_logprob[row] : 0.0f;
  r.g_entropy = a.d_entropy ? a.d_entropy[row] : 0.0f;
  r.token = token < a.classes ? static_cast<int>(token) : -1;
  r.skip = r.S == 0.0f || (g == 0.0f && r.g_entropy == 0.0f && !top_any);
  r.peaked = r.S < kPeaked && !r.skip;
  if (token >= a.classes && g != 0.0f) g = __builtin_nanf("");
  r.g_token = g * a.inv_t;
  r.all = r.g_token + top_sum * a.inv_t;
  *token_g = g;
  return r;
}

// LDS words of a group's rows: kUnlisted, or what a listed class brings.
constexpr int kUnlisted = 0x7fffffff;

// A word for each class of the block's rows, laid out as the lanes hold them.
template <class T, int G, int NV>
struct GroupWords {
  static constexpr int N = Row<T>::n, pitch = Group<T, G, NV>::pitch;
  __attribute__((aligned(16))) int word[kGroupThreads * pitch];
  // of this lane's classes, and of a class of this lane's row
  __device__ __forceinline__ int *lane() { return word + threadIdx.x * pitch; }
  __device__ __forceinline__ int &of(int id) {
    const int row = threadIdx.x & ~(G - 1);
    return word[(row + (id / N & (G - 1))) * pitch + id / (N * G) * N + (id & (N - 1))];
  }
};

template <class T, int G, int NV>
__global__ __launch_bounds__(kGroupThreads) void logprob_grad_group_kernel(LogprobArgs a) {
  constexpr int N = Row<T>::n, E = N * NV;
  __shared__ GroupWords<T, G, NV> words;  // the first entry that lists a class, then its term
  const Group<T, G, NV> g;
  const int64_t row = g.row;
  const bool live = row < a.rows;
  float v[E];
  g.load_rows(a.logits, a.row_stride, a.rows, a.classes, live, words.word, v);
  const int k = live && a.d_top ? a.top_k : 0;
  int *mine = words.lane();
  float top_sum = 0.0f;
  bool any = false;
  if (a.d_top) {
    constexpr int kKept = G <= 4 ? 4 / G : 1;
    int id[kKept];
    float term[kKept];
    auto entry = [&](int j, int &i, float &t) {
      i = a.top_in[row * a.top_k + j];
      t = a.d_top[row * a.top_k + j];
      if (i >= a.classes) i = -1;
    };
#pragma unroll
    for (int e = 0; e < kKept; ++e) {
      id[e] = -1;
      if (g.lane + e * G < k) entry(g.lane + e * G, id[e], term[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) mine[e] = kUnlisted;
    wave_fence();
#pragma unroll
    for (int e = 0; e < kKept; ++e)
      if (id[e] >= 0) atomicMin(&words.of(id[e]), g.lane + e * G);
    for (int j = g.lane + kKept * G; j < k; j += G) {
      int i;
      float t;
      entry(j, i, t);
      if (i >= 0) atomicMin(&words.of(i), j);
    }
    wave_fence();
    // Kept entries look before any term goes in; the others may meet a term, whose bits
    // are no entry's number (a term too small to be normal counts as 0).
    bool first[kKept];
#pragma unroll
    for (int e = 0; e < kKept; ++e)
      first[e] = id[e] >= 0 && words.of(id[e]) == g.lane + e * G;
    auto put = [&](int i, float t) {
      const float d = t * a.inv_t;
      words.of(i) = fabsf(d) < 1.2e-38f ? 0 : __float_as_int(d);
      top_sum += t;
      any |= t != 0.0f;
    };
    for (int j = g.lane + kKept * G; j < k; j += G) {
      int i;
      float t;
      entry(j, i, t);
      if (i >= 0 && words.of(i) == j) put(i, t);
    }
#pragma unroll
    for (int e = 0; e < kKept; ++e)
      if (first[e]) put(id[e], term[e]);
    wave_fence();
    top_sum = lanes_sum<G>(top_sum);
    any = lanes_any<G>(any);
  }
  const float m = live ? a.stats_in[2 * row] : 0.0f;
  float x[E], p[E], sum = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = (v[e] - m) * a.c;
    p[e] = exp2_raw(x[e]);
    x[e] = fmaxf(x[e], -200.0f);
    sum = __builtin_fmaf(p[e], x[e], sum);
  }
  // H - ln S from the row itself: the entropy's own rounding does not enter
  sum = lanes_sum<G>(sum);
  LogprobRow r{};
  r.token = -1;
  if (live) {
    float token_g;
    r = logprob_row(a, row, top_sum, any, &token_g);
    r.finish(a, token_g, top_sum, r.g_entropy != 0.0f ? -kLn2 * quotient(sum, r.S) : 0.0f);
  }
  // the best class of a peaked row, and what it gets (known before the others, in few registers)
  const bool some = __any(r.peaked);
  int best = -1;
  float best_d = 0.0f;
  if (some) {
    float rest = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      rest += __builtin_amdgcn_fractf(p[e]);  // the best class has 1, all others less
      best = x[e] == 0.0f ? e : best;
    }
    rest = lanes_sum<G>(rest);
    if (!r.peaked) best = -1;
    if (best >= 0) {
      float listed = a.d_top && mine[best] != kUnlisted ? __int_as_float(mine[best]) : 0.0f;
      if (g.index(best) == r.token) listed += r.g_token;
      best_d = r.best(listed, rest);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float t = p[e] * __builtin_fmaf(r.b, x[e], r.a);
    if (a.d_top && mine[e] != kUnlisted) t += __int_as_float(mine[e]);
    if (g.index(e) == r.token) t += r.g_token;
    v[e] = r.skip ? 0.0f : t;
  }
  if (some)
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e == best ? best_d : v[e];
  g.store_rows(a.d_logits, a.d_row_stride, a.rows, a.classes, words.word, v);
}

// What the long rows' gradient kernels have of a row's listed classes.
struct ListedLds {
  __attribute__((aligned(16))) int id[kMaxTop];
  float term[kMaxTop];
  float sum, any;
};

// The thread's listed class (-1: none, outside the classes or listed before) and its term, and
// the row's totals. NT > top_k.
struct Listed {
  int id = -1;
  float g = 0.0f, sum = 0.0f;
  bool any = false;
};
__device__ __forceinline__ Listed listed_terms(const LogprobArgs &a, ListedLds &l, int64_t row) {
  Listed o;
  const int tid = threadIdx.x, k = a.d_top ? a.top_k : 0;
  if (k == 0) return o;
  if (tid < ((k + 3) & ~3)) {
    const int id = tid < k ? a.top_in[row * a.top_k + tid] : -1;
    o.id = id >= 0 && id < a.classes ? id : -1;
    o.g = o.id >= 0 ? a.d_top[row * a.top_k + tid] : 0.0f;
    l.id[tid] = o.id;
  }
  __syncthreads();
  if (tid < k) {
    // a class counts by its first entry
    if (listed_before(l.id, k, tid, o.id)) o.id = -1;
    if (o.id < 0) o.g = 0.0f;
    l.term[tid] = o.g;
  }
  __syncthreads();
  if (tid < kWave) {
    float s = 0.0f;
    bool any = false;
    for (int j = tid; j < k; j += kWave) {
      s += l.term[j];
      any |= l.term[j] != 0.0f;
    }
    s = lanes_sum<kWave>(s);
    any = lanes_any<kWave>(any);
    if (tid == 0) {
      l.sum = s;
      l.any = any ? 1.0f : 0.0f;
    }
  }
  __syncthreads();
  o.sum = l.sum;
  o.any = l.any != 0.0f;
  return o;
}

// One part of a row. The listed classes and the token are written after all
// others; their logits are read before the block writes anything, so that the
// gradient may take the place of the logits. NT > top_k: a thread for each listed class
// and one for the token.
//
// A peaked row's r and E are summed up while it is written, with an H - ln S from the statistics
// that is right for all classes but the best, which is written once more at the end (by a
// second kernel where several blocks write the row: 64 x 131072 fp32 11.6 -> 13.2 us, peaked rows
// 15.5). 4096 x 32768 bf16, all rows peaked, 104 us (ordinary rows 98; summed up in a pass
// before it 117), 16384 x 5003 79 (71).
template <class T, int NT>
__global__ __launch_bounds__(NT) void logprob_grad_block_kernel(LogprobArgs a) {
  __shared__ ListedLds list;
  __shared__ BlockLds<NT> lds;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  T *out = static_cast<T *>(a.d_logits) + row * a.d_row_stride;
  const Part<T, NT> p(z, part, a.part_len, a.classes);
  const int k = a.d_top ? a.top_k : 0;
  const Listed listed = listed_terms(a, list, row);
  int mine = listed.id;
  float g = listed.g;
  float token_g;
  LogprobRow r = logprob_row(a, row, listed.sum, listed.any, &token_g);
  if (r.skip) {
    p.zero(out);
    return;
  }
  r.finish(a, token_g, listed.sum, r.g_entropy != 0.0f ? a.entropy_in[row] - log_of(r.S) : 0.0f);
  g *= a.inv_t;
  if (tid == k) {
    mine = r.token;
    if (listed_before(list.id, k, k, mine)) mine = -1;  // its entry's thread writes it
    g = r.g_token;
  } else if (mine >= 0 && mine == r.token) {
    g += r.g_token;
  }
  if (mine < p.begin || mine >= p.end) mine = -1;
  const float zm = mine >= 0 ? Row<T>::up(z[mine]) : 0.0f;
  if (a.d_logits == a.logits) __syncthreads();
  const ExpAt e(r.m, a.c);
  if (r.peaked) {
    float rest = 0.0f, sum = 0.0f;
    int best = -1;
    constexpr int N = Row<T>::n;
#pragma unroll 1  // (one vector in flight: registers for a class's index each cost the others)
    for (int i = p.begin + tid * N; i < p.end; i += NT * N) {
      float v[N];
      load_vec<T>(z, i, p.end, v);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float x = e.x(v[j]), t = exp2_raw(x), y = fmaxf(x, -200.0f);
        const bool top = v[j] == r.m;
        rest += top ? 0.0f : t;
        sum = __builtin_fmaf(t, y, sum);
        best = top ? i + j : best;
        v[j] = t * __builtin_fmaf(r.b, y, r.a);
      }
      store_vec<T>(out, i, p.end, v);
    }
    rest = block_sum<NT>(lds, rest);
    sum = block_sum<NT>(lds, sum);
    if (a.parts > 1) {
      // (a class and 1 more is a whole number that 32 bits hold; one thread has one)
      const float at = block_sum<NT>(lds, static_cast<float>(best + 1));
      if (tid == 0) a.part_sum[blockIdx.x] = make_float4(rest, sum, at, 0.0f);
    } else {
      // (read again rather than kept in registers through the row)
      const float top_sum = k > 0 ? list.sum : 0.0f;
      r = logprob_row(a, row, top_sum, true, &token_g);
      r.finish(a, token_g, top_sum, -kLn2 * quotient(sum, r.S));
      if (best >= 0) out[best] = Row<T>::down(r.best(0.0f, rest));
      __syncthreads();
      if (mine >= 0 && zm == r.m) {
        out[mine] = Row<T>::down(r.best(g, rest));
        mine = -1;
      }
    }
  } else {
    // 2^x of the fma form carries `fix`, and its x the same correction
    const float rho = e.huge ? 0.0f : __builtin_fmaf(r.m, a.c, -e.R);
    const float fa = __builtin_fmaf(-r.b, rho, r.a) * e.fix, fb = r.b * e.fix;
    if (e.huge) {
      p.map(out, [&](float v) {
        const float x = e.x_huge(v);
        return exp2_raw(x) * __builtin_fmaf(fb, fmaxf(x, -200.0f), fa);
      });
    } else {
      p.map(out, [&](float v) {
        const float x = e.x_plain(v);
        return exp2_raw(x) * __builtin_fmaf(fb, fmaxf(x, -200.0f), fa);
      });
    }
  }
  __syncthreads();
  if (mine >= 0) {
    const float x = e.x(zm);
    out[mine] = Row<T>::down(exp2_raw(x) * __builtin_fmaf(r.b, fmaxf(x, -200.0f), r.a) + g);
  }
}

// The best class of the peaked rows that several blocks have written (the others' blocks
// end at once).
constexpr int kBestThreads = 256;
static_assert(kBestThreads > kMaxTop, "");

template <class T>
__global__ __launch_bounds__(kBestThreads) void logprob_grad_best_kernel(LogprobArgs a) {
  __shared__ ListedLds list;
  __shared__ float term;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  if (!(a.stats_in[2 * row + 1] < kPeaked)) return;
  const Listed listed = listed_terms(a, list, row);
  float token_g;
  LogprobRow r = logprob_row(a, row, listed.sum, listed.any, &token_g);
  if (r.skip) return;
  // the parts' sums, in every lane: a fixed tree
  float rest = 0.0f, sum = 0.0f, at = 0.0f;
  for (int i = tid & (kWave - 1); i < a.parts; i += kWave) {
    const float4 q = a.part_sum[row * a.parts + i];
    rest += q.x;
    sum += q.y;
    at += q.z;
  }
  rest = lanes_sum<kWave>(rest);
  sum = lanes_sum<kWave>(sum);
  const int best = static_cast<int>(lanes_sum<kWave>(at)) - 1;
  if (best < 0 || best >= a.classes) return;  // statistics of other logits
  r.finish(a, token_g, listed.sum, -kLn2 * quotient(sum, r.S));
  if (tid == 0) term = 0.0f;
  __syncthreads();
  if (listed.id == best) term = listed.g * a.inv_t;
  __syncthreads();
  if (tid == 0)
    static_cast<T *>(a.d_logits)[row * a.d_row_stride + best] =
        Row<T>::down(r.best(best == r.token ? term + r.g_token : term, rest));
}

}  // namespace tmnn_hip
