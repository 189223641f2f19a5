// logits_common.hpp -- what the class-logit kernels share: typed vector
// access to rows of any alignment, sums over lanes, the online softmax and the
// selection of the k largest keys of a block.
//
// A row of logits z with scale c = log2(e) / T is summed up as (m, S, E):
//   m = max z,  S = sum 2^(c (z - m)),  E = sum 2^(c (z - m)) c (z - m)
// in one pass. Inside the pass the exponent is one fma, x = z c - R with
// R = fl(m c); at its end rho = m c - R (exact) takes the rounding of R out
// again, so that S belongs to m itself and not to R. A finished sum also has
// r = S - 1, the sum without the maximum's own term, to the precision of a sum that
// never met that 1: the logarithm of a probability near 1 is -ln(1 + r).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tmnn_hip {

constexpr float kLn2 = 0.6931471805599453f;
// |m c| up to which the fma form is used: R is off by at most 4 there, so no term passes 2^4,
// and logits of up to 93 have it at the lowest temperature (1e-6).
constexpr float kPlainShift = 134217728.0f;  // 2^27
// The lowest R, that of a sum without terms too. A thread whose classes all lie below (a finite
// mask fill) adds 0 with it, as every class does that is so far below its row's maximum; where
// the row's maximum is below itself, |m c| is above kPlainShift.
constexpr float kNoShift = -kPlainShift;
constexpr int kWave = 64;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));

// 16 bytes of a row at a time, at the alignment of one element: the hardware
// takes unaligned global vectors, so rows of odd strides need no other path.
template <class T>
struct Row;

template <>
struct Row<float> {
  static constexpr int n = 4;
  typedef f32x4v A;  // aligned to itself, as in LDS
  typedef f32x4v V __attribute__((aligned(4)));
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct Row<_Float16> {
  static constexpr int n = 8;
  typedef f16x8v A;
  typedef f16x8v V __attribute__((aligned(2)));
  static __device__ __forceinline__ float up(_Float16 x) { return static_cast<float>(x); }
  static __device__ __forceinline__ _Float16 down(float x) { return static_cast<_Float16>(x); }
};
template <>
struct Row<__bf16> {
  static constexpr int n = 8;
  typedef bf16x8v A;
  typedef bf16x8v V __attribute__((aligned(2)));
  static __device__ __forceinline__ float up(__bf16 x) { return static_cast<float>(x); }
  static __device__ __forceinline__ __bf16 down(float x) { return static_cast<__bf16>(x); }
};

template <class T>
__device__ __forceinline__ typename Row<T>::V load_raw(const T *p) {
  return *reinterpret_cast<const typename Row<T>::V *>(p);
}

template <class T>
__device__ __forceinline__ void widen(const typename Row<T>::V &v, float *out) {
#pragma unroll
  for (int j = 0; j < Row<T>::n; ++j) out[j] = Row<T>::up(v[j]);
}

// Elements i .. i + n of a row that ends at `end`; -inf past the end.
template <class T>
__device__ __forceinline__ void load_vec(const T *row, int i, int end, float *out) {
  if (i + Row<T>::n <= end) {
    widen<T>(load_raw(row + i), out);
  } else {
#pragma unroll
    for (int j = 0; j < Row<T>::n; ++j)
      out[j] = i + j < end ? Row<T>::up(row[i + j]) : -__builtin_inff();
  }
}

template <class T>
__device__ __forceinline__ void store_vec(T *row, int i, int end, const float *v) {
  if (i + Row<T>::n <= end) {
    typename Row<T>::V o;
#pragma unroll
    for (int j = 0; j < Row<T>::n; ++j) o[j] = Row<T>::down(v[j]);
    *reinterpret_cast<typename Row<T>::V *>(row + i) = o;
  } else {
#pragma unroll
    for (int j = 0; j < Row<T>::n; ++j)
      if (i + j < end) row[i + j] = Row<T>::down(v[j]);
  }
}

__device__ __forceinline__ int64_t load_index(const void *p, int64_t i, bool wide) {
  return wide ? static_cast<const int64_t *>(p)[i]
              : static_cast<int64_t>(static_cast<const int32_t *>(p)[i]);
}

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// a / b and ln x to an ulp or two, without the steps that make them exact.
__device__ __forceinline__ float quotient(float a, float b) { return a * __builtin_amdgcn_rcpf(b); }
__device__ __forceinline__ float log_of(float x) { return __builtin_amdgcn_logf(x) * kLn2; }

// e^t: the product t log2(e) in two parts, so that its rounding does not grow with t.
__device__ __forceinline__ float exp_of(float t) {
  constexpr float l = 1.44269504f, l_rest = 1.925963033e-8f;  // log2(e)
  const float x = t * l;
  const float rest = __builtin_fmaf(t, l_rest, __builtin_fmaf(t, l, -x));
  return x > -150.0f ? exp2_raw(x) * __builtin_fmaf(rest, kLn2, 1.0f) : 0.0f;
}

// ln(1 + r), r >= -1, by what rounding 1 + r leaves out: ln u + (r - (u - 1)) / u.
__device__ __forceinline__ float log1p_of(float r) {
  const float u = 1.0f + r, l = logf(u);
  const float rest = (r - (u - 1.0f)) * __builtin_amdgcn_rcpf(u);
  // u = 0, inf and NaN leave no rest
  return u > 0.0f && u < __builtin_inff() ? l + rest : l;
}

// ---- sums over G consecutive lanes (all lanes get the result) ----------------

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  // (every lane's source lane exists: no old value, so that the step is part of the
  // instruction that takes it)
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Lanes 1, 2, 4, 8 apart by DPP (quad permutations, then the mirror of 8 and of
// 16 lanes, whose quads already agree), 16 and 32 apart by swapping rows and halves
// of two copies. Both partners combine the same two numbers: every lane ends with
// the same bits.
template <int G, class Op>
__device__ __forceinline__ float over_lanes(float x, Op op) {
  if (G >= 2) x = op(x, dpp<0xB1>(x));
  if (G >= 4) x = op(x, dpp<0x4E>(x));
  if (G >= 8) x = op(x, dpp<0x141>(x));
  if (G >= 16) x = op(x, dpp<0x140>(x));
  if (G >= 32) {
    const uint32_t v = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (G >= 64) {
    const uint32_t v = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return x;
}
template <int G>
__device__ __forceinline__ float lanes_max(float x) {
  return over_lanes<G>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int G>
__device__ __forceinline__ float lanes_sum(float x) {
  return over_lanes<G>(x, [](float a, float b) { return a + b; });
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t v = __double_as_longlong(x);
  const uint32_t lo = static_cast<uint32_t>(v), hi = static_cast<uint32_t>(v >> 32);
  const uint32_t l = __builtin_amdgcn_update_dpp(0, lo, CTRL, 0xf, 0xf, true);
  const uint32_t h = __builtin_amdgcn_update_dpp(0, hi, CTRL, 0xf, 0xf, true);
  return __longlong_as_double(static_cast<uint64_t>(h) << 32 | l);
}
template <int G>
__device__ __forceinline__ double lanes_sum(double x) {
  if (G >= 2) x += dpp<0xB1>(x);
  if (G >= 4) x += dpp<0x4E>(x);
  if (G >= 8) x += dpp<0x141>(x);
  if (G >= 16) x += dpp<0x140>(x);
  if (G >= 32) x += __shfl_xor(x, 16);
  if (G >= 64) x += __shfl_xor(x, 32);
  return x;
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
template <int G, class Op>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, Op op) {
  if (G >= 2) v = op(v, dpp<0xB1>(v));
  if (G >= 4) v = op(v, dpp<0x4E>(v));
  if (G >= 8) v = op(v, dpp<0x141>(v));
  if (G >= 16) v = op(v, dpp<0x140>(v));
  if (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  if (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  return v;
}
template <int G>
__device__ __forceinline__ int lanes_isum(int x) {
  return static_cast<int>(over_lanes<G>(static_cast<uint32_t>(x), [](uint32_t a, uint32_t b) { return a + b; }));
}
template <int G>
__device__ __forceinline__ uint32_t lanes_or(uint32_t v) {
  return over_lanes<G>(v, [](uint32_t a, uint32_t b) { return a | b; });
}
template <int G>
__device__ __forceinline__ uint32_t lanes_and(uint32_t v) {
  return over_lanes<G>(v, [](uint32_t a, uint32_t b) { return a & b; });
}
template <int G>
__device__ __forceinline__ uint64_t lanes_key_max(uint64_t k) {
  uint32_t hi = static_cast<uint32_t>(k >> 32), lo = static_cast<uint32_t>(k);
  auto take = [&](uint32_t h, uint32_t l) {
    const bool more = h > hi || (h == hi && l > lo);
    hi = more ? h : hi;
    lo = more ? l : lo;
  };
  if (G >= 2) take(dpp<0xB1>(hi), dpp<0xB1>(lo));
  if (G >= 4) take(dpp<0x4E>(hi), dpp<0x4E>(lo));
  if (G >= 8) take(dpp<0x141>(hi), dpp<0x141>(lo));
  if (G >= 16) take(dpp<0x140>(hi), dpp<0x140>(lo));
  if (G >= 32) take(__shfl_xor(hi, 16), __shfl_xor(lo, 16));
  if (G >= 64) take(__shfl_xor(hi, 32), __shfl_xor(lo, 32));
  return static_cast<uint64_t>(hi) << 32 | lo;
}
// Whether `c` holds in one of the G lanes.
template <int G>
__device__ __forceinline__ bool lanes_any(bool c) {
  const uint64_t all = __ballot(c);
  if (G == kWave) return all != 0;
  const int lane = threadIdx.x & (kWave - 1) & ~(G - 1);
  return (all >> lane & ((1ull << (G & 63)) - 1ull)) != 0;
}

// Orders the LDS accesses of one wave's lanes (lockstep: a compiler fence).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- the online softmax -------------------------------------------------------

struct Soft {
  float m = -__builtin_inff();
  float R = kNoShift;
  float S = 0.0f;
  float E = 0.0f;
  float r = -1.0f;  // of a finished sum: S - 1
};

// Below this, S - 1 of an fp32 sum has lost too many bits.
constexpr float kPeaked = 1.125f;

// Takes the terms z[0..N) into a running sum. A new maximum rescales the sum,
// which happens about ln(length) times a thread. Masked terms (-inf) add 0: their
// exponent is held at -200 where it is multiplied. NaN terms make S NaN.
template <int N, bool ENT>
__device__ __forceinline__ void soft_add(Soft &s, const float *z, float zmax, float c) {
  if (zmax > s.m) {
    const float R = fmaxf(zmax * c, kNoShift);
    const float d = s.R - R, r = exp2_raw(d);
    if (ENT) s.E = r * __builtin_fmaf(s.S, d, s.E);
    s.S *= r;
    s.m = zmax;
    s.R = R;
  }
  float e[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float x = __builtin_fmaf(z[j], c, -s.R);
    e[j] = exp2_raw(x);
    if (ENT) s.E = __builtin_fmaf(e[j], fmaxf(x, -200.0f), s.E);
  }
#pragma unroll
  for (int w = 1; w < N; w *= 2)
#pragma unroll
    for (int j = 0; j + w < N; j += 2 * w) e[j] += e[j + w];
  s.S += e[0];
}

// The sum over G lanes, in the lanes' common shift.
template <int G, bool ENT>
__device__ __forceinline__ void soft_lanes(Soft &s, float c) {
  s.m = lanes_max<G>(s.m);
  const float R = fmaxf(s.m * c, kNoShift), d = s.R - R, r = exp2_raw(d);
  if (ENT) s.E = lanes_sum<G>(r * __builtin_fmaf(s.S, d, s.E));
  s.S = lanes_sum<G>(s.S * r);
  s.R = R;
}

// m c is too large for the fma form, or not a number that can be a shift. What the form made
// of such a row (an R that is off by more than an exponent holds gives infinities) is not used.
__device__ __forceinline__ bool soft_is_huge(float m, float c) {
  return !(fabsf(m * c) <= kPlainShift) && m != -__builtin_inff();
}

// Takes the rounding of R out of S and E (see the head of the file).
__device__ __forceinline__ void soft_settle(Soft &s, float c) {
  if (s.m != -__builtin_inff()) {  // else no terms; S is 0, or NaN from NaN terms
    const float rho = __builtin_fmaf(s.m, c, -s.R), f = exp2f(-rho);
    s.E = f * __builtin_fmaf(s.S, -rho, s.E);
    s.S *= f;
  }
  s.r = s.S - 1.0f;
}

// Finished sums: S and E of `b` in the shift of m >= b.m.
__device__ __forceinline__ void soft_shift(Soft &b, float m, float c) {
  if (b.S == 0.0f) {
    b.E = 0.0f;
    return;
  }
  const float d = (b.m - m) * c, r = exp2_raw(d);
  b.E = r == 0.0f ? 0.0f : r * __builtin_fmaf(b.S, d, b.E);
  b.S *= r;
}

// Adds a finished sum `b` to `s`, whose m is the largest of all that will be added.
// `one`: b is the first sum that attains m, which brings the 1 that r leaves out.
__device__ __forceinline__ void soft_join(Soft &s, Soft b, float c, bool one) {
  const float r = b.r;
  soft_shift(b, s.m, c);
  s.r += one ? r : b.S;
  s.E += b.E;
}

// Joins up to 128 finished sums, load(p) the p-th, in every lane of a wave: a fixed
// tree. `n` adds up each sum's n.
template <class Load>
__device__ __forceinline__ Soft soft_join_parts(int parts, float c, int &n, Load load) {
  const int lane = threadIdx.x & (kWave - 1);
  Soft b[2], s;
  int k[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + kWave * i < parts) b[i] = load(lane + kWave * i, k[i]);
  s.m = lanes_max<kWave>(fmaxf(b[0].m, b[1].m));
  s.r = 0.0f;
  const float inf = __builtin_inff();
  const uint64_t low = __ballot(b[0].m == s.m && s.m != -inf);
  const uint64_t high = __ballot(b[1].m == s.m && s.m != -inf);
  const int first = low ? __builtin_ctzll(low) : high ? kWave + __builtin_ctzll(high) : -1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    b[i].S = 1.0f + b[i].r;
    soft_join(s, b[i], c, lane + kWave * i == first);
  }
  s.r = lanes_sum<kWave>(s.r);
  s.E = lanes_sum<kWave>(s.E);
  n = lanes_isum<kWave>(k[0] + k[1]);
  if (s.m == -inf) s.r -= 1.0f;  // no class: S = 0 (or NaN)
  s.S = 1.0f + s.r;
  return s;
}

// 2^(c (z - m)) as the gradients need it: the same fma form with the rounding of
// R in a factor of its own, or, for huge m, the difference first.
struct ExpAt {
  float c, R, m, fix;
  bool huge;
  __device__ __forceinline__ ExpAt(float m_, float c_) : c(c_), m(m_) {
    huge = soft_is_huge(m, c);
    R = m * c;
    fix = huge ? 1.0f : exp2f(-__builtin_fmaf(m, c, -R));
  }
  __device__ __forceinline__ float x_plain(float z) const { return __builtin_fmaf(z, c, -R); }
  __device__ __forceinline__ float x_huge(float z) const { return (z - m) * c; }
  // c (z - m), once a row or class rather than in the dense loops
  __device__ __forceinline__ float x(float z) const { return (z - m) * c; }
};

// ---- order of classes: by value, then by the lowest index -------------------------

__device__ __forceinline__ uint32_t order_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);  // -0 and +0 are equal
  return b ^ (static_cast<int32_t>(b) < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o ^ (o & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float z, int i) {
  return static_cast<uint64_t>(order_of(z)) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int key_index(uint64_t k) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
}
// The smallest float above z (z finite or -inf).
__device__ __forceinline__ float next_above(float z) {
  const int32_t b = __float_as_int(z + 0.0f);
  return __int_as_float(b >= 0 ? b + 1 : b - 1);
}

// ---- the k largest keys of a block ---------------------------------------------

// Elements that may reach the bound before it is made exact: rows of equal logits bring
// up to 8 (k + 1), k at most half the groups. Small blocks keep their LDS small (65536 x 1000 bf16,
// 20 alternatives, 64 threads: 178 us with room for 1024, 12 waves on a unit).
constexpr int candidates(int threads) { return (threads < 256 ? threads : 256) * 4 + 64; }
// The threads' keys in groups: 256, or one a thread (at least k either way).
constexpr int key_groups(int threads) { return threads < 256 ? threads : 256; }

template <int NT, int SOURCES = NT>
struct SelectLds {
  static constexpr int kCandidates = candidates(NT), kSources = SOURCES;
  uint64_t key[NT];
  uint64_t cand[kCandidates];
  uint64_t tau;
  int count, sources;
  int source[kSources];
};

// A key that at least k of the groups' keys reach (the largest of their
// threads'), as high as its search finds: bit by bit over the bits in which keys differ
// (not those that 16-bit logits leave empty: 16 x 65536 bf16 with 5 alternatives 10.1 us, over
// all bits 13.5), then over the indices of an equal value,
// ending as soon as exactly k keys reach it. 0 where fewer than k groups have a key. Run by one wave.
template <int NT>
__device__ __forceinline__ uint64_t kth_key(const uint64_t *key, int k) {
  constexpr int groups = key_groups(NT), W = groups / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  uint32_t hi[W], lo[W];
  uint32_t some = 0, all = 0xffffffffu;  // bits that are set in one key, in every key
  int n = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    uint64_t q = key[lane + kWave * i];
#pragma unroll
    for (int t = 1; t < NT / groups; ++t) {
      const uint64_t o = key[lane + kWave * i + groups * t];
      q = o > q ? o : q;
    }
    hi[i] = static_cast<uint32_t>(q >> 32);
    lo[i] = static_cast<uint32_t>(q);
    n += __popcll(__ballot(hi[i] != 0));
    some |= hi[i];
    if (hi[i] != 0) all &= hi[i];
  }
  if (n < k) return 0;
  // every key has the bits of p, so that a test of one more compares whole words
  uint32_t p = __builtin_amdgcn_readfirstlane(lanes_and<kWave>(all));
  uint32_t open = __builtin_amdgcn_readfirstlane(lanes_or<kWave>(some)) & ~p;
  while (open != 0) {
    const uint32_t bit = 0x80000000u >> __builtin_clz(open), t = p | bit;
    open ^= bit;
    n = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) n += __popcll(__ballot(hi[i] >= t));
    if (n >= k) p = t;
    if (n == k) return static_cast<uint64_t>(p) << 32;
  }
  int above = 0;
  some = 0;
  all = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    above += __popcll(__ballot(hi[i] > p));
    if (hi[i] == p) {
      some |= lo[i];
      all &= lo[i];
    }
  }
  uint32_t q = __builtin_amdgcn_readfirstlane(lanes_and<kWave>(all));
  open = __builtin_amdgcn_readfirstlane(lanes_or<kWave>(some)) & ~q;
  while (open != 0) {
    const uint32_t bit = 0x80000000u >> __builtin_clz(open), t = q | bit;
    open ^= bit;
    n = above;
#pragma unroll
    for (int i = 0; i < W; ++i) n += __popcll(__ballot(hi[i] == p && lo[i] >= t));
    if (n >= k) q = t;
    if (n == k) break;
  }
  return static_cast<uint64_t>(p) << 32 | q;
}

// The k largest keys of the block's elements, in order, to put(j, key) for j up
// to the returned count (fewer than k where the block has fewer). The elements belong
// to sources of `vectors` groups each: visit(source, i, f) calls f(key) for a source's
// i-th group, and each(f) calls f(source, key) for the thread's own sources with a key
// that one of the source's elements reaches (0: it has none) and whose high word none
// of them exceeds; `mine` is the largest of these.
//
// No element costs anything beyond the running maximum of the first pass: the k-th
// largest of the groups' maxima bounds the answer from below, and the block looks
// again only at the sources that reach it (about k of them, and about
// k (1 + k / 512) elements that reach it, in no special order). Where more elements do than
// there is room for, the bound is made exact by counting.
template <int NT, int SOURCES, class Each, class Visit, class Put>
__device__ __forceinline__ int block_select(SelectLds<NT, SOURCES> &s, uint64_t mine, int k,
                                            int vectors, Each each, Visit visit, Put put) {
  constexpr int kCandidates = candidates(NT), kSources = SOURCES;
  const int tid = threadIdx.x;
  s.key[tid] = mine;
  if (tid == 0) {
    s.count = 0;
    s.sources = 0;
  }
  __syncthreads();
  if (tid < kWave) {
    const uint64_t t = kth_key<NT>(s.key, k);
    if (tid == 0) s.tau = t;
  }
  __syncthreads();
  uint64_t tau = s.tau;
  auto gather = [&](uint64_t q) {
    if (q >= tau) {
      const int at = atomicAdd(&s.count, 1);
      if (at < kCandidates) s.cand[at] = q;
    }
  };
  if ((mine | 0xffffffffu) >= tau)
    each([&](int source, uint64_t key) {
      if (key != 0 && (key | 0xffffffffu) >= tau) {
        const int at = atomicAdd(&s.sources, 1);
        if (at < kSources) s.source[at] = source;
      }
    });
  __syncthreads();
  const int sources = s.sources;
  if (sources <= kSources) {
    for (int i = tid; i < sources * vectors; i += NT)
      visit(s.source[i % sources], i / sources, gather);
    __syncthreads();
  }
  int n = s.count;
  if (n > kCandidates || sources > kSources) {
    auto all_mine = [&](auto f) {
      each([&](int source, uint64_t key) {
        if (key != 0)
          for (int i = 0; i < vectors; ++i) visit(source, i, f);
      });
    };
    uint64_t t = 0;
    for (int b = 63; b >= 0; --b) {
      const uint64_t test = t | 1ull << b;
      __syncthreads();
      if (tid == 0) s.count = 0;
      __syncthreads();
      int c = 0;
      all_mine([&](uint64_t q) { c += q >= test; });
      if (c) atomicAdd(&s.count, c);
      __syncthreads();
      if (s.count >= k) t = test;
    }
    __syncthreads();
    if (tid == 0) s.count = 0;
    __syncthreads();
    tau = t;
    all_mine(gather);
    __syncthreads();
    n = s.count;
  }
  // the place of a candidate is the number of larger ones
  for (int i = tid; i < n; i += NT) {
    const uint64_t q = s.cand[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += s.cand[j] > q;
    if (place < k) put(place, q);
  }
  return n < k ? n : k;
}

// Whether an earlier entry of a list in LDS, 16-byte aligned and filled up with -1 to a
// multiple of four, has the same id as entry `j`.
__device__ __forceinline__ bool listed_before(const int *ids, int k, int j, int id) {
  bool before = false;
  for (int i = 0; i < k; i += 4) {
    const int4 q = *reinterpret_cast<const int4 *>(ids + i);
    before |= (i < j && q.x == id) || (i + 1 < j && q.y == id) || (i + 2 < j && q.z == id) ||
              (i + 3 < j && q.w == id);
  }
  return before;
}

}  // namespace tmnn_hip
