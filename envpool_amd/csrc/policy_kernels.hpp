// policy_kernels.hpp - device code of the masked choice and its training counterpart (policy.hip).
//
// Both need, per row, one pass that carries the running maximum m, the sum S of exp(y - m) and the sum
// E of exp(y - m) (y - m): log p_j = y_j - m - log S and the entropy is log S - E / S. The choice works
// in 64 bits (R = double): which option a uniform number falls on is decided by comparing it with
// cumulated weights, and 32-bit sums over 10^5 options are off by more than one option is wide. The
// log-probabilities of stored actions (R = float) need no more than 32.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace epp {

using bf16 = __bf16;
using f16 = _Float16;

// one row set as the kernels see it (ep_policy_rows after the host's checks)
struct Rows {
  int64_t rows, options;
  const void* logits;
  int64_t logits_stride;
  const int32_t* num_options;
  const void* mask;
  int32_t mask_bits;  // 0 bytes, 1 bit words
  int64_t mask_stride;
  const void* bias;
  int32_t bias_f32;
  int64_t bias_stride;
  const int32_t* history;
  int64_t history_len, history_stride;
  const float *repetition, *frequency, *presence, *temperature;
  double repetition_all, frequency_all, presence_all, temperature_all;
  double inv_t_all;  // 1 / temperature_all, and the same in 32 bits
  float inv_t_all_32;
  int32_t vec;  // rows of logits, 32-bit biases and byte masks start on boundaries of their 8-option loads (with
                // options a multiple of 8 too, every row is made of whole eights: kWhole)
};

constexpr int kThreads = 256;
constexpr int kPer = 8;                      // options per thread and piece
constexpr int kPiece = kThreads * kPer;      // options per piece of a row

// What stands for "no weight" among the y: illegal options, and legal ones that are -inf. In 64 bits no legal
// value comes near it. In 32 bits a legal value is held one step above (HoldRange), so that an option masked
// with the type's lowest value keeps its (vanishing) weight and a row of nothing else is uniform.
template <class R> struct Num;
template <> struct Num<double> {
  static constexpr double kNone = -1.7976931348623157e308;
  static constexpr double kUnit = 0.6931471805599453;
  static constexpr double kFloor = -1100.0;  // 2^d of this and less is 0
  static constexpr double kLeast = 6.2e-306;  // kNone times this is below kFloor, a difference of logits times it nothing
};
template <> struct Num<float> {
  static constexpr float kNone = -3.40282347e38f;
  static constexpr float kLow = -3.40282326e38f, kHigh = 3.40282326e38f;
  static constexpr float kUnit = 0.693147181f;  // exponents d count octaves, weights are 2^d
  static constexpr float kFloor = -10000.f;
  static constexpr float kLeast = 4.5e-37f;  // kNone times this is an exponent of -153 (the differences of logits up to 1e29 nothing)
};

// 2^d for d in [-1100, 0] in 64 bits: d = n + r, |r| <= 1/2, the series of exp(r ln 2) to the 11th power (the first
// term left out is below 7e-15), times 2^n. Half the library function's instructions: there are no
// overflows or positive arguments to look after, and the octaves come for free with the factor 1 / t.
__device__ inline double weight(double d) {
  constexpr double l = 0.6931471805599453;
  constexpr double c2 = l * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5, c6 = c5 * l / 6, c7 = c6 * l / 7, c8 = c7 * l / 8,
                   c9 = c8 * l / 9, c10 = c9 * l / 10, c11 = c10 * l / 11;
  const double n = rint(d), r = d - n;
  double p = fma(c11, r, c10);
  p = fma(p, r, c9);
  p = fma(p, r, c8);
  p = fma(p, r, c7);
  p = fma(p, r, c6);
  p = fma(p, r, c5);
  p = fma(p, r, c4);
  p = fma(p, r, c3);
  p = fma(p, r, c2);
  p = fma(p, r, l);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}
__device__ inline float weight(float x) { return __builtin_amdgcn_exp2f(x); }
// (maximum without the NaN rules of fmax's library form: the operands are numbers, or a NaN that must not win)
__device__ inline double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ inline float larger(float a, float b) { return __builtin_fmaxf(a, b); }

__device__ inline double mul_add(double a, double b, double c) { return __builtin_fma(a, b, c); }
__device__ inline float mul_add(float a, float b, float c) { return __builtin_fmaf(a, b, c); }

// what is the same for all options of a row
template <class R> struct RowConst {
  R rep, inv_rep, freq, pres, inv_t;
  R k;              // (z - m) * k is a weight's exponent
  int64_t n_legal;  // options below this are legal as far as num_options goes
  bool bad;
};

template <class R, bool kHist> __device__ inline RowConst<R> row_const(const Rows& p, int64_t row) {
  RowConst<R> c{};
  const R t = p.temperature ? (R)p.temperature[row] : (R)p.temperature_all;
  if (p.temperature) c.inv_t = (R)1 / t;
  else c.inv_t = sizeof(R) == 8 ? (R)p.inv_t_all : (R)p.inv_t_all_32;
  c.k = c.inv_t * ((R)1 / Num<R>::kUnit);
  c.bad = !(t > (R)0) || !(t < (R)INFINITY) || !(c.k < (R)INFINITY);
  c.k = larger(c.k, Num<R>::kLeast);  // (however high the temperature, what has no weight gets none)
  if (kHist) {
    c.rep = p.repetition ? (R)p.repetition[row] : (R)p.repetition_all;
    c.inv_rep = (R)1 / c.rep;
    c.freq = p.frequency ? (R)p.frequency[row] : (R)p.frequency_all;
    c.pres = p.presence ? (R)p.presence[row] : (R)p.presence_all;
    c.bad = c.bad || !(c.rep > (R)0) || !(c.rep < (R)INFINITY) || !(c.inv_rep < (R)INFINITY);
  }
  int64_t n = p.options;
  if (p.num_options) {
    const int64_t k = p.num_options[row];
    n = k < 0 ? 0 : (k < n ? k : n);
  }
  c.n_legal = n;
  return c;
}

// x after the penalties for `count` appearances. Contraction is off: two options whose results are
// equal in plain 64-bit arithmetic have to stay equal (the lowest index wins).
template <class R> __device__ inline R penalized(R x, uint32_t count, const RowConst<R>& c) {
#pragma clang fp contract(off)
  if (count) {
    x = x > (R)0 ? x / c.rep : x * c.rep;
    const R f = c.freq * (R)count;
    x = x - f;
    x = x - c.pres;
  }
  return x;
}

template <class T> struct Vec8 {
  alignas(16) T v[8];
};

// The penalized logits of a row's options that stand in its history: `count` per option, `value` where it is
// not 0. (A long row's workgroup computes them once per entry: of 2048 options a few dozen have any.)
template <class R> struct Seen {
  const uint32_t* count = nullptr;
  const R* value = nullptr;  // NULL: computed per option from the count
  __device__ Seen at(int64_t i) const { return {count + i, value ? value + i : nullptr}; }
};

__device__ inline bool bit(uint32_t bits, int i) { return (bits >> i) & 1u; }
// v where bit i is set, else other: two instructions (the bit spread over a word, a bitwise choice)
__device__ inline uint32_t pick(uint32_t bits, int i, uint32_t v, uint32_t other) {
  const uint32_t all = (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
  return (v & all) | (other & ~all);
}
__device__ inline float pick(uint32_t bits, int i, float v, float other) {
  return __builtin_bit_cast(float, pick(bits, i, __builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, other)));
}
__device__ inline double pick(uint32_t bits, int i, double v, double other) {
  const uint64_t a = __builtin_bit_cast(uint64_t, v), b = __builtin_bit_cast(uint64_t, other);
  const uint32_t lo = pick(bits, i, (uint32_t)a, (uint32_t)b), hi = pick(bits, i, (uint32_t)(a >> 32), (uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The operands of options j0 .. j0+7 of a row (j0 a multiple of 8, below the row's end) as they lie in memory. With
// kWhole every row is made of whole eights that can be read at once: all operands are then asked for before the first
// is used, and a walk asks for its next eight before it works on these. Ragged rows are read where they are used:
// eight guarded loads each, in more registers (524288 x 16 bf16: choose 36 us, whole 18; 524288 x 24: evaluate 36
// and 15, its gradients 42 and 21; 2048 x 32768: gradients 71 and 59).
template <class T, bool kWhole> struct Raw {
  __device__ void ask_row(const Rows&, int64_t, int64_t) {}
  __device__ void ask_bias(const Rows&, int64_t, int64_t) {}
};
template <class T> struct Raw<T, true> {
  typedef uint32_t Words __attribute__((ext_vector_type(kPer * sizeof(T) / 4), aligned(16)));
  Words x;
  uint64_t m;  // eight mask bytes, or the word that holds the eight bits
  float b[kPer];
  __device__ void ask_row(const Rows& p, int64_t row, int64_t j0) {
    if (p.mask) {
      if (p.mask_bits) m = ((const uint32_t*)p.mask)[row * p.mask_stride + (j0 >> 5)];
      else m = *(const uint64_t*)((const uint8_t*)p.mask + row * p.mask_stride + j0);
    }
    x = *(const Words*)((const T*)p.logits + row * p.logits_stride + j0);
  }
  __device__ void ask_bias(const Rows& p, int64_t row, int64_t j0) {
    if (!p.bias) return;
    const int64_t b0 = row * p.bias_stride + j0;
    if (p.bias_f32) {
      *(Vec8<float>*)b = *(const Vec8<float>*)((const float*)p.bias + b0);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) b[i] = (float)((const T*)p.bias)[b0 + i];
    }
  }
  __device__ float logit(int i) const {
    T v[sizeof(x[0]) / sizeof(T)];
    const uint32_t word = x[i * (int)sizeof(T) / 4];
    __builtin_memcpy(v, &word, 4);
    return (float)v[i % (4 / (int)sizeof(T))];
  }
};

// Options j0 .. j0+7 of a row (j0 a multiple of 8, below the row's end): y before the temperature, as they
// come. Returns which are legal (bit i = option j0 + i); the y of the others are unspecified.
// whole: all eight exist and every operand can be read eight at a time. slope: d y / d logit.
template <class T, class R, bool kHist, bool kWhole>
__device__ inline uint32_t load_y(const Rows& p, const RowConst<R>& c, int64_t row, int64_t j0, bool whole, const Raw<T, kWhole>& raw, const Seen<R>& seen,
                                  R (&y)[kPer], R* slope = nullptr) {
  const int64_t left = c.n_legal - j0;
  uint32_t legal = left >= kPer ? 0xffu : left > 0 ? (1u << left) - 1u : 0u;
  if (p.mask) {
    if (p.mask_bits) {
      if constexpr (kWhole) legal &= (uint32_t)raw.m >> (j0 & 31);
      else legal &= ((const uint32_t*)p.mask)[row * p.mask_stride + (j0 >> 5)] >> (j0 & 31);
    } else {
      uint64_t w = 0;
      if constexpr (kWhole) {
        w = raw.m;
      } else {
        const uint8_t* m = (const uint8_t*)p.mask + row * p.mask_stride + j0;
        if (whole) {
          w = *(const uint64_t*)m;
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (j0 + i < p.options) w |= (uint64_t)m[i] << (8 * i);
        }
      }
      // nonzero bytes to bits: every byte folded onto its lowest bit, four of them gathered by a product
      w |= w >> 4;
      w |= w >> 2;
      w |= w >> 1;
      const uint32_t lo = (uint32_t)w & 0x01010101u, hi = (uint32_t)(w >> 32) & 0x01010101u;
      legal &= ((lo * 0x01020408u) >> 24) | (((hi * 0x01020408u) >> 24) << 4);
    }
  }
  if constexpr (kWhole) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) y[i] = (R)raw.logit(i);
  } else {
    const T* x = (const T*)p.logits + row * p.logits_stride + j0;
    T xv[kPer];
    if (whole) {
      *(Vec8<T>*)xv = *(const Vec8<T>*)x;
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) xv[i] = j0 + i < p.options ? x[i] : (T)0.f;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) y[i] = (R)(float)xv[i];
  }
  if (kHist) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t n = seen.count[i];
      if (slope) slope[i] = n ? (y[i] > (R)0 ? c.inv_rep : c.rep) : (R)1;
      if (seen.value) y[i] = n ? seen.value[i] : y[i];
      else y[i] = penalized<R>(y[i], n, c);
    }
  }
  if constexpr (kWhole) {
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) y[i] += (R)raw.b[i];
    }
  } else if (p.bias) {
    const int64_t b0 = row * p.bias_stride + j0;
    if (p.bias_f32) {
      const float* b = (const float*)p.bias + b0;
      if (whole) {
        const Vec8<float> v = *(const Vec8<float>*)b;
#pragma unroll
        for (int i = 0; i < kPer; ++i) y[i] += (R)v.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) y[i] += j0 + i < p.options ? (R)b[i] : (R)0;
      }
    } else {
      const T* b = (const T*)p.bias + b0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) y[i] += j0 + i < p.options ? (R)(float)b[i] : (R)0;
    }
  }
  return legal;
}

// In 32 bits the sum of finite values may leave the range: the end of it stands for the sum then, so that it
// is not taken for a logit that was infinite.
template <class T> __device__ inline float hold_range(const Rows& p, int64_t row, int64_t j, float y) {
  if (fabsf(y) != INFINITY) return y;
  const float x = (float)((const T*)p.logits)[row * p.logits_stride + j];
  float b = 0.f;
  if (p.bias) {
    const int64_t at = row * p.bias_stride + j;
    b = p.bias_f32 ? ((const float*)p.bias)[at] : (float)((const T*)p.bias)[at];
  }
  return fabsf(x) < INFINITY && fabsf(b) < INFINITY ? (y > 0.f ? Num<float>::kHigh : Num<float>::kLow) : y;
}

// What a row, or a part of it, holds among its legal values
enum : int {
  kBad = 1,    // NaN or +inf
  kBelow = 2,  // in 32 bits, a sum below the range, held at its end
  kGone = 4,   // in 32 bits, a logit or a bias of -inf
};
// Option j of a row, where load_ready says that it has no weight: the lower end of the range, if that is only because its
// neighbours are larger (it is legal, and has the lowest value), else still kNone.
template <class T> __device__ inline float lowest_or_none(const Rows& p, const RowConst<float>& c, int64_t row, int64_t j) {
  if (j < 0 || j >= c.n_legal) return Num<float>::kNone;
  if (p.mask) {
    const int64_t at = row * p.mask_stride;
    if (p.mask_bits ? !((((const uint32_t*)p.mask)[at + (j >> 5)] >> (j & 31)) & 1u) : !((const uint8_t*)p.mask)[at + j]) return Num<float>::kNone;
  }
  return larger(hold_range<T>(p, row, j, -INFINITY), Num<float>::kNone);
}

// load_y made ready for sums: kNone where there is no weight, m the largest. Returns what of the above there is. Nearly
// always all are finite, which one product with 0 per option shows (0 * inf and 0 * NaN are NaN).
template <class T, class R, bool kHist, bool kWhole>
__device__ inline int load_ready(const Rows& p, const RowConst<R>& c, int64_t row, int64_t j0, bool whole, const Raw<T, kWhole>& raw, const Seen<R>& seen,
                                  R (&y)[kPer], R& m) {
  m = Num<R>::kNone;
  if (j0 >= c.n_legal) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) y[i] = Num<R>::kNone;
    return 0;
  }
  const uint32_t legal = load_y<T, R, kHist, kWhole>(p, c, row, j0, whole, raw, seen, y);
  R odd = (R)0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    y[i] = pick(legal, i, y[i], Num<R>::kNone);
    odd = mul_add(y[i], (R)0, odd);
    m = larger(m, y[i]);
  }
  if (odd == (R)0 && (m > Num<R>::kNone || !legal)) return 0;
  int what = 0;
  m = Num<R>::kNone;  // (of the values as they are held)
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (!bit(legal, i)) continue;
    if constexpr (sizeof(R) == 4) {
      const bool below = y[i] == -INFINITY;
      y[i] = hold_range<T>(p, row, j0 + i, y[i]);
      if (below) what |= y[i] == -INFINITY ? kGone : kBelow;
    }
    if (!(y[i] < (R)INFINITY)) what |= kBad;
    if (y[i] == -(R)INFINITY) y[i] = Num<R>::kNone;
    else if constexpr (sizeof(R) == 4) y[i] = larger(y[i], Num<float>::kLow);
    m = larger(m, y[i]);
  }
  return what;
}

// running statistics of a row, or of a part of it
template <class R> struct Stat {
  R m;           // largest y
  R s, e;        // sum w, sum w d with d = (y - m) k, w = exp(d kUnit)
  int64_t best;  // lowest index with y == m
  int32_t what;  // kBad, kBelow, kGone
};
template <class R> __device__ inline Stat<R> stat_zero() { return {Num<R>::kNone, (R)0, (R)0, INT64_MAX, 0}; }
template <class R> __device__ inline R exponent(R y, R m, R k) { return larger((y - m) * k, Num<R>::kFloor); }

// brings s, e from reference a.m to reference m >= a.m
template <class R> __device__ inline void stat_rebase(Stat<R>& a, R m, R k) {
  const R d = exponent(a.m, m, k);
  const R f = weight(d);
  a.e = f * mul_add(a.s, d, a.e);
  a.s = f * a.s;
  a.m = m;
}
// adds the options j0 .. j0+7, m the largest of them (kBest: and notes where the largest is)
template <class R, bool kBest> __device__ inline void stat_add(Stat<R>& a, const R (&y)[kPer], R m, int64_t j0, R k) {
  if (m == Num<R>::kNone) return;
  if (m > a.m) {
    if (kBest) {
      int at = 0;
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i) at = y[i] == m ? i : at;
      a.best = j0 + at;
    }
    stat_rebase(a, m, k);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const R d = exponent(y[i], a.m, k);
    const R w = weight(d);
    a.s += w;
    a.e = mul_add(w, d, a.e);
  }
}

// Over `width` neighbouring lanes (a power of two up to 64), the same result in all of them. Six exchanges between
// registers (no trip through LDS): with the neighbour, the neighbouring pair, the mirrored four and eight - by then every
// quad and octet holds one value - and the neighbouring row of 16 and half of the wave.
template <int kDpp, class V> __device__ inline V moved(V v) {
  union { V v; int w[sizeof(V) / 4]; } u;
  u.v = v;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) u.w[i] = __builtin_amdgcn_update_dpp(u.w[i], u.w[i], kDpp, 0xf, 0xf, true);
  return u.v;
}
template <int kLanes, class V, class Op> __device__ inline V across(V v, Op op) {
  union { V v; uint32_t w[sizeof(V) / 4]; } x, y;
  x.v = v;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
    const auto r = kLanes == 16 ? __builtin_amdgcn_permlane16_swap(x.w[i], x.w[i], false, false) : __builtin_amdgcn_permlane32_swap(x.w[i], x.w[i], false, false);
    x.w[i] = r[0], y.w[i] = r[1];
  }
  return op(x.v, y.v);
}
template <class V, class Op> __device__ inline V lanes_reduce(V v, int width, Op op) {
  if (width > 1) v = op(v, moved<0xb1>(v));
  if (width > 2) v = op(v, moved<0x4e>(v));
  if (width > 4) v = op(v, moved<0x141>(v));
  if (width > 8) v = op(v, moved<0x140>(v));
  if (width > 16) v = across<16>(v, op);
  if (width > 32) v = across<32>(v, op);
  return v;
}
template <class V> __device__ inline V lanes_max(V v, int width) {
  return lanes_reduce(v, width, [](V a, V b) { return a > b ? a : b; });
}
template <class V> __device__ inline V lanes_min(V v, int width) {
  return lanes_reduce(v, width, [](V a, V b) { return a < b ? a : b; });
}
__device__ inline int32_t lanes_or(int32_t v, int width) {
  return lanes_reduce(v, width, [](int32_t a, int32_t b) { return a | b; });
}
template <class V> __device__ inline V lanes_sum(V v, int width) {
  return lanes_reduce(v, width, [](V a, V b) { return a + b; });
}
// sum over the lanes up to and including this one, of `width`
template <class V> __device__ inline V lanes_scan(V v, int width) {
  const int at = threadIdx.x & (width - 1);
  for (int o = 1; o < width; o <<= 1) {
    const V b = __shfl_up(v, o, 64);
    if (at >= o) v += b;
  }
  return v;
}

// over the workgroup, the same result in every thread: the maximum first, then every thread moves its own
// sums to it (one exponential each) and they are added
template <class R, bool kBest> __device__ inline Stat<R> stat_block(Stat<R> a, R k, Stat<R>* lds) {
  constexpr int kWaves = kThreads / 64;
  const int wave = threadIdx.x >> 6;
  const R m_wave = lanes_max(a.m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[wave].m = m_wave;
  __syncthreads();
  R m = lds[0].m;
  for (int i = 1; i < kWaves; ++i) m = larger(m, lds[i].m);
  const int64_t best = kBest ? lanes_min((long long)(a.m == m ? a.best : INT64_MAX), 64) : INT64_MAX;
  stat_rebase(a, m, k);
  const R sum = lanes_sum(a.s, 64), e = lanes_sum(a.e, 64);
  const int what = lanes_or(a.what, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[wave] = {m, sum, e, best, what};
  __syncthreads();
  Stat<R> r = lds[0];
  for (int i = 1; i < kWaves; ++i) {
    r.s += lds[i].s, r.e += lds[i].e, r.what |= lds[i].what;
    if (lds[i].best < r.best) r.best = lds[i].best;
  }
  return r;
}

// the options [j0, j0 + kPiece) of a row that stand in its history: counts and penalized logits
template <class T, class R> struct SeenPiece {
  uint32_t count[kPiece];
  R value[kPiece];
  uint16_t list[kPiece];
  int n;
};
template <class T, class R>
__device__ inline Seen<R> count_piece(const Rows& p, const RowConst<R>& c, int64_t row, int64_t j0, SeenPiece<T, R>& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < kPiece; i += kThreads) s.count[i] = 0;
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  const int32_t* h = p.history + row * p.history_stride;
  const uint32_t size = (uint32_t)min((int64_t)kPiece, p.options - j0);
  // (eight entries under way at once: one after the other, each would wait for its load and its two additions)
  constexpr int kAhead = 8;
  for (int64_t i0 = threadIdx.x; i0 < p.history_len; i0 += kAhead * kThreads) {
    uint32_t j[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) j[i] = i0 + i * kThreads < p.history_len ? (uint32_t)h[i0 + i * kThreads] - (uint32_t)j0 : size;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (j[i] < size && atomicAdd(&s.count[j[i]], 1u) == 0) s.list[atomicAdd(&s.n, 1)] = (uint16_t)j[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < s.n; i += kThreads) {
    const int j = s.list[i];
    s.value[j] = penalized<R>((R)(float)((const T*)p.logits)[row * p.logits_stride + j0 + j], s.count[j], c);
  }
  __syncthreads();
  return {s.count, s.value};
}
template <class T, class R, bool kHist> struct PieceMemory {
  SeenPiece<T, R> s;
  __device__ Seen<R> count(const Rows& p, const RowConst<R>& c, int64_t row, int64_t j0) { return count_piece<T, R>(p, c, row, j0, s).at(threadIdx.x * kPer); }
};
template <class T, class R> struct PieceMemory<T, R, false> {
  __device__ Seen<R> count(const Rows&, const RowConst<R>&, int64_t, int64_t) { return {}; }
};

template <class R> __device__ inline R quiet_nan() { return (R)__builtin_nanf(""); }

// ---- results ------------------------------------------------------------------------------------------
struct ChooseOut {
  int32_t* action;
  float *log_prob, *entropy;
};
__device__ inline void finish_choose(const ChooseOut& o, int64_t row, const Stat<double>& a, const RowConst<double>& c, int64_t pick, double y_pick) {
  const bool bad = (a.what & kBad) || c.bad;
  const bool empty = !bad && a.m == Num<double>::kNone;
  const double log_s = log(a.s);
  o.action[row] = bad || empty ? -1 : (int32_t)pick;
  o.log_prob[row] = bad ? quiet_nan<float>() : empty ? 0.f : (float)((y_pick - a.m) * c.inv_t - log_s);
  o.entropy[row] = bad ? quiet_nan<float>() : empty ? 0.f : (float)(log_s - a.e / a.s * Num<double>::kUnit);
}

struct EvaluateOut {
  const int32_t* action;
  // stats: {largest y, log2 of the sum of weights}; {-inf, 0}: EMPTY; {NaN, NaN}: BAD. A row whose largest y is the lower end
  // of the range that values are held at has {kLow, ..} if sums below the range are among them, which the gradients'
  // kernels see as -inf: all legal options are equal then. With -inf logits or biases beside such sums {kLow, NaN}: the gradients cannot
  // tell them apart, and are NaN. Without such sums {the lowest value, ..}, from which the others' distance shows.
  float *log_prob, *entropy, *stats;
};
__device__ inline void finish_evaluate(const EvaluateOut& o, int64_t row, int64_t options, const Stat<float>& a, const RowConst<float>& c, int32_t act,
                                       float y_act) {
  const bool bad = (a.what & kBad) || c.bad;
  const bool empty = !bad && a.m == Num<float>::kNone;
  const float log_s = __builtin_amdgcn_logf(a.s);
  float lp;
  if (act == -1) lp = 0.f;
  else if (act < 0 || act >= options) lp = quiet_nan<float>();
  else if (empty || y_act == Num<float>::kNone) lp = -INFINITY;
  else if (y_act - a.m < -1e38f) lp = (y_act - a.m) * c.inv_t;  // (times k first it may leave the range)
  else lp = ((y_act - a.m) * c.k - log_s) * Num<float>::kUnit;
  o.log_prob[row] = bad ? quiet_nan<float>() : lp;
  o.entropy[row] = bad ? quiet_nan<float>() : empty ? 0.f : (log_s - a.e / a.s) * Num<float>::kUnit;
  const bool lowest = a.m == Num<float>::kLow, below = lowest && (a.what & kBelow);
  o.stats[2 * row] = bad ? quiet_nan<float>() : empty ? -INFINITY : lowest && !below ? Num<float>::kNone : a.m;
  o.stats[2 * row + 1] = bad || (below && (a.what & kGone)) ? quiet_nan<float>() : empty ? 0.f : log_s;
}

// ---- rows of up to 64 * 8 * NP options: `width` lanes per row, a lane's options in registers -----------
// Option j of a row sits in lane (j / 8) % width, piece j / 8 / width. Neighbouring rows are neighbouring lanes,
// so that a wave reads one contiguous stretch however short the rows are.
struct Group {
  int64_t row;
  int lane, width;
  bool there;
  __device__ int64_t j(int piece) const { return ((int64_t)piece * width + lane) * kPer; }
};
__device__ inline Group group_of(const Rows& p, int64_t block, int width_log) {
  Group g;
  g.width = 1 << width_log;
  g.lane = threadIdx.x & (g.width - 1);
  g.row = block * (kThreads >> width_log) + (threadIdx.x >> width_log);
  g.there = g.row < p.rows;
  if (!g.there) g.row = 0;
  return g;
}
// the histories of a workgroup's rows, counted; returns this row's counts
template <int NP> __device__ inline const uint32_t* count_groups(const Rows& p, const Group& g, uint32_t* counts) {
  uint32_t* mine = counts + (threadIdx.x - g.lane) * kPer * NP;
  __syncthreads();
  for (int i = threadIdx.x; i < kThreads * kPer * NP; i += kThreads) counts[i] = 0;
  __syncthreads();
  const int32_t* h = p.history + g.row * p.history_stride;
  for (int64_t i = g.lane; i < p.history_len; i += g.width) {
    const int32_t j = h[i];
    if (j >= 0 && j < p.options) atomicAdd(&mine[j], 1u);
  }
  __syncthreads();
  return mine;
}

// choose: one pass, the weights stay in registers between the sum and the choice. Bound by the 64-bit arithmetic of the
// weights (some 25 of 57 instructions an option): 524288 x 16 bf16 with byte masks and a shared bias 18 us = 1.8 TB/s
// of 33 MB; 1024 x 16 f32 4.8 us, which is a launch.
template <class T, int NP, bool kHist, bool kWhole>
__global__ __launch_bounds__(kThreads) void choose_group(Rows p, int width_log, const void* u, int u_f64, ChooseOut out) {
  extern __shared__ uint32_t counts[];
  const Group g = group_of(p, blockIdx.x, width_log);
  const RowConst<double> c = row_const<double, kHist>(p, g.row);
  const uint32_t* n = kHist ? count_groups<NP>(p, g, counts) : nullptr;
  constexpr bool whole = kWhole;
  double y[NP][kPer];
  Stat<double> a = stat_zero<double>();
  Raw<T, kWhole> raw[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k)
    if (g.j(k) < c.n_legal) raw[k].ask_row(p, g.row, g.j(k)), raw[k].ask_bias(p, g.row, g.j(k));
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    double m;
    a.what |= load_ready<T, double, kHist, kWhole>(p, c, g.row, g.j(k), whole, raw[k], Seen<double>{n}.at(kHist ? g.j(k) : 0), y[k], m);
    a.m = larger(a.m, m);
  }
  a.m = lanes_max(a.m, g.width);
  a.what = lanes_or(a.what, g.width);
  double w[NP][kPer];
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const double d = exponent(y[k][i], a.m, c.k);
      w[k][i] = weight(d);
      a.s += w[k][i];
      a.e = fma(w[k][i], d, a.e);
    }
  a.e = lanes_sum(a.e, g.width);
  int32_t pick;
  double y_pick = a.m;
  if (!u) {
    a.s = lanes_sum(a.s, g.width);
    int32_t best = INT32_MAX;
#pragma unroll
    for (int k = NP - 1; k >= 0; --k)
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i) best = y[k][i] == a.m ? (int32_t)g.j(k) + i : best;
    pick = lanes_min(best, g.width);
  } else {
    // cumulated from option 0 on: piece by piece, lane by lane
    double sum[NP], incl[NP], before = 0;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      sum[k] = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum[k] += w[k][i];
      incl[k] = lanes_scan(sum[k], g.width) + before;
      before = __shfl(incl[k], (threadIdx.x & 63) | (g.width - 1), 64);
    }
    a.s = before;
    const double target = (u_f64 ? ((const double*)u)[g.row] : (double)((const float*)u)[g.row]) * a.s;
    int32_t hit = INT32_MAX;
    double hit_y = Num<double>::kNone;
#pragma unroll
    for (int k = NP - 1; k >= 0; --k) {
      // from the lane's end: the lowest option whose sum is above the target stays
      double cum = incl[k];
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i) {
        const bool is = cum > target && w[k][i] > 0;
        hit = is ? (int32_t)g.j(k) + i : hit;
        hit_y = is ? y[k][i] : hit_y;
        cum = i ? cum - w[k][i] : cum;
      }
    }
    pick = lanes_min(hit, g.width);
    if (pick == INT32_MAX) {  // (u at the upper end: the last option with any weight)
      hit = -1;
#pragma unroll
      for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (w[k][i] > 0) hit = (int32_t)g.j(k) + i, hit_y = y[k][i];
      pick = lanes_max(hit, g.width);
    }
    y_pick = lanes_max(hit == pick ? hit_y : Num<double>::kNone, g.width);
  }
  if (g.lane == 0 && g.there) finish_choose(out, g.row, a, c, pick, y_pick);
}

// evaluate: the same in 32 bits. Bound by instructions (30 an option of a lane, whether the row has it or not: a quarter
// of the lanes of 24 options): 524288 x 24 bf16 16 us = 2.9 TB/s of 46 MB.
template <class T, int NP, bool kHist, bool kWhole> __global__ __launch_bounds__(kThreads) void evaluate_group(Rows p, int width_log, EvaluateOut out) {
  extern __shared__ uint32_t counts[];
  const Group g = group_of(p, blockIdx.x, width_log);
  const RowConst<float> c = row_const<float, kHist>(p, g.row);
  const uint32_t* n = kHist ? count_groups<NP>(p, g, counts) : nullptr;
  constexpr bool whole = kWhole;
  const int32_t act = out.action[g.row];
  float y[NP][kPer];
  Stat<float> a = stat_zero<float>();
  float y_act = Num<float>::kNone;
  Raw<T, kWhole> raw[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k)
    if (g.j(k) < c.n_legal) raw[k].ask_row(p, g.row, g.j(k)), raw[k].ask_bias(p, g.row, g.j(k));
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    float m;
    a.what |= load_ready<T, float, kHist, kWhole>(p, c, g.row, g.j(k), whole, raw[k], Seen<float>{n}.at(kHist ? g.j(k) : 0), y[k], m);
    a.m = larger(a.m, m);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      y_act = act == g.j(k) + i ? y[k][i] : y_act;
    }
  }
  a.m = lanes_max(a.m, g.width);
  a.what = lanes_or(a.what, g.width);
  y_act = lanes_max(y_act, g.width);
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float d = exponent(y[k][i], a.m, c.k);
      const float w = weight(d);
      a.s += w;
      a.e = fmaf(w, d, a.e);
    }
  a.s = lanes_sum(a.s, g.width);
  a.e = lanes_sum(a.e, g.width);
  if (g.lane == 0 && g.there) {
    if (y_act == Num<float>::kNone) y_act = lowest_or_none<T>(p, c, g.row, act);
    finish_evaluate(out, g.row, p.options, a, c, act, y_act);
  }
}

// ---- longer rows: a workgroup per part of a row (`pieces` pieces of kPiece options), parts joined after ---
// 64 x 131072 bf16, bit masks, a shared bias and 2048 entries of history a row: 30 us. A third of it is the history
// (every part reads all of its row's entries), the rest the weights in 64 bits; 29 KB of LDS let five workgroups stand
// on a CU (six, with the list inside the values' memory and the registers kept to it, took 38 us).
template <class T, bool kHist, bool kWhole, bool kBest>
__global__ __launch_bounds__(kThreads) void choose_parts(Rows p, int pieces, int n_parts, Stat<double>* parts) {
  __shared__ PieceMemory<T, double, kHist> mem;
  __shared__ Stat<double> red[kThreads / 64];
  const int64_t row = blockIdx.x / n_parts, part = blockIdx.x % n_parts;
  const RowConst<double> c = row_const<double, kHist>(p, row);
  Stat<double> a = stat_zero<double>();
  const int64_t j_end = min((part + 1) * pieces * (int64_t)kPiece, c.n_legal);
  const int64_t j_first = part * pieces * (int64_t)kPiece;
  Raw<T, kWhole> raw;
  const auto ask = [&](int64_t j) {
    if (j < j_end) raw.ask_row(p, row, j), raw.ask_bias(p, row, j);
  };
  ask(j_first + threadIdx.x * kPer);
  for (int64_t j0 = j_first; j0 < j_end; j0 += kPiece) {
    const auto seen = mem.count(p, c, row, j0);
    const int64_t j = j0 + threadIdx.x * kPer;
    double y[kPer], m;
    a.what |= load_ready<T, double, kHist, kWhole>(p, c, row, j, p.vec && j0 + kPiece <= p.options, raw, seen, y, m);
    ask(j + kPiece);
    stat_add<double, kBest>(a, y, m, j, c.k);
  }
  a = stat_block<double, kBest>(a, c.k, red);
  if (threadIdx.x == 0) parts[blockIdx.x] = a;
}

// joins a row's parts, and finds the option that u falls on by walking down the one part it lies in: one workgroup a
// row and a chain of reads that depend on each other, 12 us at 64 x 131072
template <class T, bool kHist, bool kWhole>
__global__ __launch_bounds__(kThreads) void choose_join(Rows p, int pieces, int n_parts, const Stat<double>* all_parts, const void* u, int u_f64, ChooseOut out) {
  __shared__ PieceMemory<T, double, kHist> mem;
  __shared__ Stat<double> red[kThreads / 64];
  __shared__ double wave_sum[kThreads / 64];
  __shared__ long long found;
  __shared__ double found_y, part_before;
  __shared__ int part_at;
  const int64_t row = blockIdx.x;
  const Stat<double>* parts = all_parts + row * n_parts;
  const RowConst<double> c = row_const<double, kHist>(p, row);
  Stat<double> a = stat_zero<double>();
  for (int i = threadIdx.x; i < n_parts; i += kThreads) {
    Stat<double> b = parts[i];
    const double m = larger(a.m, b.m);
    const int64_t best = a.m > b.m ? a.best : (b.m > a.m ? b.best : min(a.best, b.best));
    stat_rebase(a, m, c.k);
    stat_rebase(b, m, c.k);
    a = {m, a.s + b.s, a.e + b.e, best, a.what | b.what};
  }
  a = stat_block<double, true>(a, c.k, red);
  int64_t pick = a.best;
  double y_pick = a.m;
  if (u && !(a.what & kBad) && !c.bad && a.m != Num<double>::kNone) {
    const double target = (u_f64 ? ((const double*)u)[row] : (double)((const float*)u)[row]) * a.s;
    // the part: its weights, moved to the row's maximum, cumulated 64 parts at a time by one wave
    if (threadIdx.x < 64) {
      double before = 0;
      int at = -1, last = 0;
      double at_before = 0, last_before = 0;
      for (int i0 = 0; i0 < n_parts && at < 0; i0 += 64) {
        double w = 0;
        if (i0 + (int)threadIdx.x < n_parts) {
          Stat<double> b = parts[i0 + threadIdx.x];
          stat_rebase(b, a.m, c.k);
          w = b.s;
        }
        const double incl = before + lanes_scan(w, 64);
        const uint64_t over = __ballot(incl > target && w > 0), any = __ballot(w > 0);
        if (over) {
          const int k = __ffsll((unsigned long long)over) - 1;
          at = i0 + k;
          at_before = __shfl(incl - w, k, 64);
        }
        if (any) {
          const int k = 63 - __clzll(any);
          last = i0 + k;
          last_before = __shfl(incl - w, k, 64);
        }
        before = __shfl(incl, 63, 64);
      }
      if (threadIdx.x == 0) part_at = at >= 0 ? at : last, part_before = at >= 0 ? at_before : last_before, found = INT64_MAX;
    }
    __syncthreads();
    double before = part_before;
    int64_t last = -1;
    double last_y = 0;
    const int64_t j_first = part_at * (int64_t)pieces * kPiece, j_end = min(j_first + pieces * (int64_t)kPiece, c.n_legal);
    for (int64_t j0 = j_first; j0 < j_end; j0 += kPiece) {
      const int64_t j = j0 + threadIdx.x * kPer;
      Raw<T, kWhole> raw;
      if (j < j_end) raw.ask_row(p, row, j), raw.ask_bias(p, row, j);
      const auto seen = mem.count(p, c, row, j0);
      double y[kPer], w[kPer], m, sum = 0;
      (void)load_ready<T, double, kHist, kWhole>(p, c, row, j, p.vec && j0 + kPiece <= p.options, raw, seen, y, m);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        w[i] = weight(exponent(y[i], a.m, c.k));
        sum += w[i];
        if (w[i] > 0) last = j + i, last_y = y[i];
      }
      const double incl = lanes_scan(sum, 64);
      __syncthreads();
      if ((threadIdx.x & 63) == 63) wave_sum[threadIdx.x >> 6] = incl;
      __syncthreads();
      double cum = before + incl - sum;
      for (int i = 0; i < (int)(threadIdx.x >> 6); ++i) cum += wave_sum[i];
      int64_t hit = INT64_MAX;
      double hit_y = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        cum += w[i];
        if (hit == INT64_MAX && w[i] > 0 && cum > target) hit = j + i, hit_y = y[i];
      }
      if (hit != INT64_MAX) atomicMin(&found, (long long)hit);
      __syncthreads();
      if (hit != INT64_MAX && hit == found) found_y = hit_y;
      if (found != INT64_MAX) break;
      for (int i = 0; i < kThreads / 64; ++i) before += wave_sum[i];
    }
    __syncthreads();
    if (found == INT64_MAX) {  // rounding: the last option of the part with any weight
      __syncthreads();
      if (threadIdx.x == 0) found = -1;
      __syncthreads();
      atomicMax(&found, (long long)last);
      __syncthreads();
      if (last == found) found_y = last_y;
      __syncthreads();
    }
    pick = found;
    y_pick = found_y;
  }
  if (threadIdx.x == 0) finish_choose(out, row, a, c, pick, y_pick);
}

// The same walk in 32 bits. One part: the row's results at once; several: partial sums, with the logit of the
// action from the part that holds it. 2048 x 32768 bf16 with bit masks: 45 us = 3.1 TB/s of 142 MB, bound by
// instructions (20 an option: 45 us with the registers kept to eight workgroups a CU, one round of them; 60 in two).
struct EvaluatePart {
  Stat<float> stat;
  float y_act;
};
template <class T, bool kHist, bool kWhole>
__global__ __launch_bounds__(kThreads, kHist ? 6 : 8) void evaluate_parts(Rows p, int pieces, int n_parts, EvaluatePart* parts, EvaluateOut out) {
  __shared__ PieceMemory<T, float, kHist> mem;
  __shared__ Stat<float> red[kThreads / 64];
  __shared__ float y_act;
  const int64_t row = blockIdx.x / n_parts, part = blockIdx.x % n_parts;
  const RowConst<float> c = row_const<float, kHist>(p, row);
  const int32_t act = out.action[row];
  Stat<float> a = stat_zero<float>();
  const int64_t j_end = min((part + 1) * pieces * (int64_t)kPiece, c.n_legal);
  const int64_t j_first = part * pieces * (int64_t)kPiece;
  Raw<T, kWhole> raw;
  const auto ask = [&](int64_t j) {
    if (j < j_end) raw.ask_row(p, row, j), raw.ask_bias(p, row, j);
  };
  ask(j_first + threadIdx.x * kPer);
  // (what the action has if the walk finds no weight there; here, where few registers are held)
  if (threadIdx.x == 0) y_act = act >= j_first && act < j_end ? lowest_or_none<T>(p, c, row, act) : Num<float>::kNone;
  __syncthreads();
  for (int64_t j0 = j_first; j0 < j_end; j0 += kPiece) {
    const auto seen = mem.count(p, c, row, j0);
    const int64_t j = j0 + threadIdx.x * kPer;
    float y[kPer], m;
    a.what |= load_ready<T, float, kHist, kWhole>(p, c, row, j, p.vec && j0 + kPiece <= p.options, raw, seen, y, m);
    ask(j + kPiece);
    stat_add<float, false>(a, y, m, j, c.k);
    if ((uint64_t)(act - j) < kPer) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (act == j + i && y[i] != Num<float>::kNone) y_act = y[i];
    }
  }
  a = stat_block<float, false>(a, c.k, red);
  if (threadIdx.x != 0) return;
  if (n_parts == 1) finish_evaluate(out, row, p.options, a, c, act, y_act);
  else parts[blockIdx.x] = {a, y_act};
}
__global__ __launch_bounds__(kThreads) inline void evaluate_join(Rows p, int n_parts, const EvaluatePart* all_parts, EvaluateOut out) {
  // one wave per row
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const RowConst<float> c = p.history ? row_const<float, true>(p, row) : row_const<float, false>(p, row);
  const EvaluatePart* parts = all_parts + row * n_parts;
  Stat<float> a = stat_zero<float>();
  float y_act = Num<float>::kNone;
  for (int i = threadIdx.x & 63; i < n_parts; i += 64) {
    EvaluatePart b = parts[i];
    const float m = larger(a.m, b.stat.m);
    stat_rebase(a, m, c.k);
    stat_rebase(b.stat, m, c.k);
    a.s += b.stat.s, a.e += b.stat.e, a.what |= b.stat.what;
    y_act = larger(y_act, b.y_act);
  }
  const float m = lanes_max(a.m, 64);
  stat_rebase(a, m, c.k);
  a.s = lanes_sum(a.s, 64), a.e = lanes_sum(a.e, 64), a.what = lanes_or(a.what, 64);
  y_act = lanes_max(y_act, 64);
  if ((threadIdx.x & 63) == 0) finish_evaluate(out, row, p.options, a, c, out.action[row], y_act);
}

// workgroups of the gradients' kernels that a CU holds at once: their registers are kept to as many, and the walks
// down the rows are cut for as many (one round of equal walks, none that waits for a place). 524288 x 24 bf16, one
// piece a lane: 21.2 us with five, 22.5 with four, 25.4 with six (registers spill)
constexpr int kGradPieceBlocks = 6;
constexpr int grad_group_per_cu(int pieces) { return pieces == 4 ? 2 : pieces == 2 ? 4 : 5; }

struct GradArgs {
  const int32_t* action;
  const float *entropy, *stats, *g_lp, *g_h;
  void* grad_logits;
  int64_t grad_logits_stride;
  void* grad_bias;          // per-row biases: written here
  int64_t grad_bias_stride;
  float* partial;           // shared biases: [row blocks][options] sums
  int32_t vec_out;
};

// What the gradient of a row needs, all scaled by 1 / temperature: with d = log2 p_j,
// d/dy_j = [j = act] g1 - p_j (g1 + g2 (H + ln p_j)).
struct GradRow {
  float m, k, log_s;
  float flat, lean;  // g1 + g2 H, g2 ln 2
  float g1;
  int32_t act;
  bool empty;
};
template <bool kHist> __device__ inline GradRow grad_row(const GradArgs& g, const RowConst<float>& c, int64_t row) {
  GradRow r;
  r.m = g.stats[2 * row];
  r.log_s = g.stats[2 * row + 1];
  r.k = r.m == Num<float>::kLow ? -2e-38f : c.k;  // (all are equal, see EvaluateOut: what is below the largest counts as above)
  r.act = g.action[row];
  const float g_lp = g.g_lp ? g.g_lp[row] : 0.f, g2 = g.g_h ? g.g_h[row] : 0.f, entropy = g.entropy[row];
  const float g1 = r.act != -1 ? g_lp : 0.f;
  r.empty = r.m == -INFINITY;
  const float nan = r.log_s != r.log_s ? r.log_s : 0.f;  // (a BAD row) its gradient is NaN where legal
  r.g1 = g1 * c.inv_t;
  r.flat = (g1 + g2 * entropy) * c.inv_t + nan;
  r.lean = g2 * Num<float>::kUnit * c.inv_t;
  return r;
}
// the gradient with respect to y / temperature's argument for options j .. j+7; 0 where illegal
__device__ inline void grad_y(const GradRow& r, const float (&y)[kPer], uint32_t legal, int64_t j, float (&out)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    // (no probability is above that of the row's largest value, which a sum that left the range of 32 bits upwards is)
    const float d = __builtin_amdgcn_fmed3f(fmaf(y[i] - r.m, r.k, -r.log_s), Num<float>::kFloor, -r.log_s);
    out[i] = pick(legal, i, -weight(d) * fmaf(r.lean, d, r.flat), 0.f);
  }
  if ((uint64_t)(r.act - j) < kPer) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (r.act == j + i && bit(legal, i)) out[i] += r.g1;
  }
}

template <class T> __device__ inline void store8(T* out, const float (&v)[kPer], int64_t j, int64_t options, bool vec) {
  if (vec && j + kPer <= options) {
    Vec8<T> o;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o.v[i] = (T)v[i];
    *(Vec8<T>*)out = o;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (j + i < options) out[i] = (T)v[i];
  }
}

// short rows: the lanes of evaluate_group, walking down the rows; a shared bias' gradient is summed per lane, then
// over the workgroup's row slots. 524288 x 24 bf16: 21 us = 3.4 TB/s of 73 MB
template <class T, int NP, bool kHist, bool kWhole> __global__ __launch_bounds__(kThreads, grad_group_per_cu(NP)) void evaluate_grad_group(Rows p, GradArgs g, int width_log, int64_t blocks_of_rows) {
  extern __shared__ uint32_t counts[];  // (as floats for the sums afterwards)
  float sum[NP][kPer];
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum[k][i] = 0.f;
  Raw<T, kWhole> raw[NP];
  const int64_t rows_on = (int64_t)gridDim.x * (kThreads >> width_log);  // from a lane's row to its next
  const auto ask = [&](int k, int64_t j, int64_t row, bool first) {
    if (j >= p.options || row >= p.rows) return;
    raw[k].ask_row(p, row, j);
    if (p.bias_stride != 0 || first) raw[k].ask_bias(p, row, j);
  };
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const Group at = group_of(p, blockIdx.x, width_log);
    if (at.there) ask(k, at.j(k), at.row, true);
  }
  for (int64_t b = blockIdx.x; b < blocks_of_rows; b += gridDim.x) {
    const Group at = group_of(p, b, width_log);
    const uint32_t* n = kHist ? count_groups<NP>(p, at, counts) : nullptr;
    constexpr bool whole = kWhole;
    if (!at.there) continue;
    const RowConst<float> c = row_const<float, kHist>(p, at.row);
    const GradRow r = grad_row<kHist>(g, c, at.row);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int64_t j = at.j(k);
      if (j >= p.options) continue;
      float y[kPer], slope[kPer], dx[kPer], db[kPer];
      const uint32_t legal = load_y<T, float, kHist, kWhole>(p, c, at.row, j, whole, raw[k], Seen<float>{n}.at(kHist ? j : 0), y, slope);
      ask(k, j, at.row + rows_on, false);
      grad_y(r, y, r.empty ? 0u : legal, j, db);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        dx[i] = kHist ? db[i] * slope[i] : db[i];
        sum[k][i] += db[i];
      }
      if (g.grad_logits) store8<T>((T*)g.grad_logits + at.row * g.grad_logits_stride + j, dx, j, kWhole ? INT64_MAX : p.options, kWhole || g.vec_out);
      if (g.grad_bias) {
        const int64_t to = at.row * g.grad_bias_stride + j;
        if (p.bias_f32) store8<float>((float*)g.grad_bias + to, db, j, p.options, false);
        else store8<T>((T*)g.grad_bias + to, db, j, p.options, false);
      }
    }
  }
  if (!g.partial) return;
  float* sums = (float*)counts;
  const int width = 1 << width_log, per_row = width * kPer * NP;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      sums[(threadIdx.x >> width_log) * per_row + (k * width + (threadIdx.x & (width - 1))) * kPer + i] = sum[k][i];
  __syncthreads();
  for (int64_t j = threadIdx.x; j < p.options; j += kThreads) {
    float s = 0.f;
    for (int i = 0; i < (kThreads >> width_log); ++i) s += sums[i * per_row + j];
    g.partial[blockIdx.x * p.options + j] = s;
  }
}

// a workgroup owns kPiece columns and walks down its rows: the sum of a shared bias' gradient stays in registers.
// Reads the logits again and writes as much: 2048 x 32768 bf16 59 us = 4.7 TB/s of 276 MB, what a large copy reaches
// (90 us in workgroups that waited for a place on the chip)
template <class T, bool kHist, bool kWhole>
__global__ __launch_bounds__(kThreads, kGradPieceBlocks) void evaluate_grad_piece(Rows p, GradArgs g, int64_t rows_per_block) {
  __shared__ PieceMemory<T, float, kHist> mem;
  const int64_t j0 = (int64_t)blockIdx.x * kPiece;
  const int64_t j = j0 + threadIdx.x * kPer;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per_block;
  const int64_t r1 = r0 + rows_per_block < p.rows ? r0 + rows_per_block : p.rows;
  float sum[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum[i] = 0.f;
  Raw<T, kWhole> raw;
  if (r0 < r1 && j < p.options) raw.ask_row(p, r0, j), raw.ask_bias(p, r0, j);
  for (int64_t row = r0; row < r1; ++row) {
    const RowConst<float> c = row_const<float, kHist>(p, row);
    const GradRow r = grad_row<kHist>(g, c, row);
    const auto seen = mem.count(p, c, row, j0);
    if (j >= p.options) continue;
    float y[kPer], slope[kPer], dx[kPer], db[kPer];
    const uint32_t legal = load_y<T, float, kHist, kWhole>(p, c, row, j, p.vec && j0 + kPiece <= p.options, raw, seen, y, slope);
    if (row + 1 < r1) {
      raw.ask_row(p, row + 1, j);
      if (p.bias_stride != 0) raw.ask_bias(p, row + 1, j);
    }
    grad_y(r, y, r.empty ? 0u : legal, j, db);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      dx[i] = kHist ? db[i] * slope[i] : db[i];
      sum[i] += db[i];
    }
    if (g.grad_logits) store8<T>((T*)g.grad_logits + row * g.grad_logits_stride + j, dx, j, kWhole ? INT64_MAX : p.options, kWhole || g.vec_out);
    if (g.grad_bias) {
      const int64_t at = row * g.grad_bias_stride + j;
      if (p.bias_f32) store8<float>((float*)g.grad_bias + at, db, j, p.options, false);
      else store8<T>((T*)g.grad_bias + at, db, j, p.options, false);
    }
  }
  if (g.partial && j < p.options) {
    float* o = g.partial + (int64_t)blockIdx.y * p.options + j;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (j + i < p.options) o[i] = sum[i];
  }
}

// column sums of partial [n][options] (4 us at 1280 x 24 and at 94 x 32768), in a fixed order: kCols columns a workgroup, the other threads down the rows
template <class T, int kCols>
__global__ __launch_bounds__(kThreads) void sum_partials(const float* partial, int64_t n, int64_t options, T* out) {
  __shared__ float red[kThreads];
  constexpr int kDown = kThreads / kCols;
  for (int64_t j0 = (int64_t)blockIdx.x * kCols; j0 < options; j0 += (int64_t)gridDim.x * kCols) {
    const int64_t j = j0 + threadIdx.x % kCols;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (j < options) {
      int64_t i = threadIdx.x / kCols;
      for (; i + 3 * kDown < n; i += 4 * kDown)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += partial[(i + q * kDown) * options + j];
      for (; i < n; i += kDown) s[0] += partial[i * options + j];
    }
    red[threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    for (int o = kDown / 2; o > 0; o >>= 1) {
      if ((int)threadIdx.x < o * kCols) red[threadIdx.x] += red[threadIdx.x + o * kCols];
      __syncthreads();
    }
    if (threadIdx.x < kCols && j < options) out[j] = (T)red[threadIdx.x];
    __syncthreads();
  }
}

}  // namespace epp
