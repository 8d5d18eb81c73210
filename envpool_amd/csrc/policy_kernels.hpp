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
  int32_t vec;  // logits rows (and biases, if any) start on 8-element boundaries: load 8 at a time
};

constexpr int kThreads = 256;
constexpr int kPer = 8;                      // options per thread and piece
constexpr int kPiece = kThreads * kPer;      // options per piece of a row

template <class R> __device__ inline R neg_inf() { return -(R)INFINITY; }

// what is the same for all options of a row
template <class R> struct RowConst {
  R rep, freq, pres, inv_t;
  int64_t n_legal;  // options below this are legal as far as num_options goes
  bool bad;
};

template <class R> __device__ inline RowConst<R> row_const(const Rows& p, int64_t row) {
  RowConst<R> c;
  const R t = p.temperature ? (R)p.temperature[row] : (R)p.temperature_all;
  c.rep = p.repetition ? (R)p.repetition[row] : (R)p.repetition_all;
  c.freq = p.frequency ? (R)p.frequency[row] : (R)p.frequency_all;
  c.pres = p.presence ? (R)p.presence[row] : (R)p.presence_all;
  c.inv_t = (R)1 / t;
  c.bad = !(t > (R)0) || !(t < (R)INFINITY) || !(c.inv_t < (R)INFINITY) || (p.history && !(c.rep > (R)0));
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

// finite inputs whose 32-bit sum leaves the range stay at its end: a mask of the type's lowest value
// plus a negative bias is still a (vanishing) weight and not an illegal option
__device__ inline float hold_range(float z, float x, float b) {
  if (fabsf(z) == INFINITY && fabsf(x) < INFINITY && fabsf(b) < INFINITY) return z > 0 ? 3.402823466e38f : -3.402823466e38f;
  return z;
}
__device__ inline double hold_range(double z, double, double) { return z; }

template <class T> struct Vec8 {
  alignas(16) T v[8];
};

template <class T> __device__ inline bool legal_at(const Rows& p, int64_t row, int64_t j) {
  if (!p.mask) return true;
  if (p.mask_bits) return (((const uint32_t*)p.mask)[row * p.mask_stride + (j >> 5)] >> (j & 31)) & 1u;
  return ((const uint8_t*)p.mask)[row * p.mask_stride + j] != 0;
}

// z of options j0 .. j0+7 (j0 a multiple of 8): logits after penalties and bias, before the temperature;
// -inf where illegal. legal: bit i = option j0 + i is legal. slope: d z / d logit, for the gradient.
template <class T, class R>
__device__ inline uint32_t load_z(const Rows& p, const RowConst<R>& c, int64_t row, int64_t j0, const uint32_t* counts,
                                  R (&z)[kPer], R* slope = nullptr) {
  uint32_t legal = 0;
  const int64_t left = c.n_legal - j0;
  if (left <= 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) z[i] = neg_inf<R>();
    return 0;
  }
  legal = left >= kPer ? 0xffu : (1u << left) - 1u;
  if (p.mask) {
    if (p.mask_bits) {
      legal &= ((const uint32_t*)p.mask)[row * p.mask_stride + (j0 >> 5)] >> (j0 & 31);
    } else {
      const uint8_t* m = (const uint8_t*)p.mask + row * p.mask_stride + j0;
      if (((uintptr_t)m & 7) == 0 && j0 + kPer <= p.options) {
        const uint64_t w = *(const uint64_t*)m;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (!((w >> (8 * i)) & 0xff)) legal &= ~(1u << i);
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (j0 + i < p.options && !m[i]) legal &= ~(1u << i);
      }
    }
  }
  const T* x = (const T*)p.logits + row * p.logits_stride + j0;
  T xv[kPer];
  if (p.vec && j0 + kPer <= p.options) {
    *(Vec8<T>*)xv = *(const Vec8<T>*)x;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) xv[i] = j0 + i < p.options ? x[i] : (T)0.f;
  }
  float bv[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) bv[i] = 0.f;
  if (p.bias) {
    const int64_t b0 = row * p.bias_stride + j0;
    if (p.bias_f32) {
      const float* b = (const float*)p.bias + b0;
      if (p.vec && j0 + kPer <= p.options) {
        *(Vec8<float>*)bv = *(const Vec8<float>*)b;
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) bv[i] = j0 + i < p.options ? b[i] : 0.f;
      }
    } else {
      const T* b = (const T*)p.bias + b0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) bv[i] = j0 + i < p.options ? (float)b[i] : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const R x0 = (R)(float)xv[i];
    R y = x0;
    if (counts) {
      const uint32_t n = counts[i];
      y = penalized<R>(x0, n, c);
      if (slope) slope[i] = n ? (x0 > (R)0 ? (R)1 / c.rep : c.rep) : (R)1;
    } else if (slope) {
      slope[i] = (R)1;
    }
    const R b = (R)bv[i];
    z[i] = (legal >> i) & 1 ? hold_range(y + b, x0, b) : neg_inf<R>();
  }
  return legal;
}

// exp of x <= 0 in 64 bits: x = n ln 2 + r, |r| <= ln 2 / 2, the series of exp r to r^11 (the first term left
// out is below 7e-15), times 2^n. About two thirds of the library function's instructions: there are no
// overflows or positive arguments to look after, and what is below e^-745 is 0.
__device__ inline double exp_of(double x) {
  x = fmax(x, -800.0);
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0.6931471805599453, x);  // ln 2 to 53 bits, then what it lacks
  r = fma(n, -2.3190468138462996e-17, r);
  double p = 1.0 / 39916800;
  p = fma(p, r, 1.0 / 3628800);
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}
__device__ inline float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896f); }

// running statistics of a row, or of a part of it
template <class R> struct Stat {
  R m;       // largest z
  R s, e;    // sum w, sum w (y - ym) with w = exp((z - m) / t); in units of 1/t: y - ym = (z - m) / t
  int64_t best;  // lowest index with z == m
  int32_t bad;
};
template <class R> __device__ inline Stat<R> stat_zero() { return {neg_inf<R>(), (R)0, (R)0, INT64_MAX, 0}; }

// brings s, e from reference a.m to reference m >= a.m
template <class R> __device__ inline void stat_rebase(Stat<R>& a, R m, R inv_t) {
  if (a.m == m) return;
  if (a.m == neg_inf<R>()) {
    a.s = a.e = (R)0;
  } else {
    const R d = (a.m - m) * inv_t;
    const R f = exp_of(d);
    a.e = f > (R)0 ? f * (a.e + a.s * d) : (R)0;
    a.s = f * a.s;
  }
  a.m = m;
}
// adds the options j0 .. j0+7
template <class R> __device__ inline void stat_add(Stat<R>& a, const R (&z)[kPer], int64_t j0, R inv_t) {
  R m = neg_inf<R>();
  int at = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (!(z[i] < (R)INFINITY)) a.bad = 1;
    if (z[i] > m) m = z[i], at = i;
  }
  if (m == neg_inf<R>()) return;
  if (m > a.m) {
    a.best = j0 + at;
    stat_rebase(a, m, inv_t);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const R d = (z[i] - a.m) * inv_t;
    const R w = exp_of(d);
    if (w > (R)0) a.s += w, a.e += w * d;
  }
}

// over `width` neighbouring lanes (a power of two up to 64), the same result in all of them
template <class V> __device__ inline V lanes_max(V v, int width) {
  for (int o = 1; o < width; o <<= 1) {
    const V b = __shfl_xor(v, o, 64);
    v = v > b ? v : b;
  }
  return v;
}
template <class V> __device__ inline V lanes_min(V v, int width) { return -lanes_max(-v, width); }
template <class V> __device__ inline V lanes_sum(V v, int width) {
  for (int o = 1; o < width; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
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
template <class R> __device__ inline Stat<R> stat_block(Stat<R> a, R inv_t, Stat<R>* lds) {
  constexpr int kWaves = kThreads / 64;
  const int wave = threadIdx.x >> 6;
  const R m_wave = lanes_max(a.m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[wave].m = m_wave;
  __syncthreads();
  R m = lds[0].m;
  for (int i = 1; i < kWaves; ++i) m = m > lds[i].m ? m : lds[i].m;
  const int64_t best = lanes_min((long long)(a.m == m ? a.best : INT64_MAX), 64);
  stat_rebase(a, m, inv_t);
  const R sum = lanes_sum(a.s, 64), e = lanes_sum(a.e, 64);
  const int bad = __any(a.bad);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[wave] = {m, sum, e, best, bad};
  __syncthreads();
  Stat<R> r = lds[0];
  for (int i = 1; i < kWaves; ++i) {
    r.s += lds[i].s, r.e += lds[i].e, r.bad |= lds[i].bad;
    if (lds[i].best < r.best) r.best = lds[i].best;
  }
  return r;
}

// how often each option of [j0, j0 + kPiece) stands in the row's history
__device__ inline void count_piece(const Rows& p, int64_t row, int64_t j0, uint32_t* counts) {
  __syncthreads();
  for (int i = threadIdx.x; i < kPiece; i += kThreads) counts[i] = 0;
  __syncthreads();
  const int32_t* h = p.history + row * p.history_stride;
  for (int64_t i = threadIdx.x; i < p.history_len; i += kThreads) {
    const int64_t j = h[i];
    if (j >= j0 && j < j0 + kPiece && j < p.options) atomicAdd(&counts[j - j0], 1u);
  }
  __syncthreads();
}

template <class R> __device__ inline R quiet_nan() { return (R)__builtin_nanf(""); }

// ---- results ------------------------------------------------------------------------------------------
struct ChooseOut {
  int32_t* action;
  float *log_prob, *entropy;
};
__device__ inline void finish_choose(const ChooseOut& o, int64_t row, const Stat<double>& a, bool bad_row, double inv_t, int64_t pick, double z_pick) {
  const bool bad = a.bad || bad_row;
  const bool empty = !bad && a.m == neg_inf<double>();
  const double log_s = log(a.s);
  o.action[row] = bad || empty ? -1 : (int32_t)pick;
  o.log_prob[row] = bad ? quiet_nan<float>() : empty ? 0.f : (float)((z_pick - a.m) * inv_t - log_s);
  o.entropy[row] = bad ? quiet_nan<float>() : empty ? 0.f : (float)(log_s - a.e / a.s);
}

struct EvaluateOut {
  const int32_t* action;
  float *log_prob, *entropy, *stats;
};
__device__ inline void finish_evaluate(const EvaluateOut& o, int64_t row, int64_t options, const Stat<float>& a, bool bad_row, float inv_t, int32_t act,
                                       float z_act) {
  const bool bad = a.bad || bad_row;
  const bool empty = !bad && a.m == -INFINITY;
  const float log_s = logf(a.s);
  float lp;
  if (act == -1) lp = 0.f;
  else if (act < 0 || act >= options) lp = quiet_nan<float>();
  else if (empty || z_act == -INFINITY) lp = -INFINITY;
  else lp = (z_act - a.m) * inv_t - log_s;
  o.log_prob[row] = bad ? quiet_nan<float>() : lp;
  o.entropy[row] = bad ? quiet_nan<float>() : empty ? 0.f : log_s - a.e / a.s;
  o.stats[2 * row] = bad ? quiet_nan<float>() : a.m;
  o.stats[2 * row + 1] = bad ? quiet_nan<float>() : empty ? 0.f : log_s;
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
  if (!p.history) return nullptr;
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

template <class T, int NP>
__global__ __launch_bounds__(kThreads) void choose_group(Rows p, int width_log, const void* u, int u_f64, ChooseOut out) {
  extern __shared__ uint32_t counts[];
  const Group g = group_of(p, blockIdx.x, width_log);
  const RowConst<double> c = row_const<double>(p, g.row);
  const uint32_t* n = count_groups<NP>(p, g, counts);
  double z[NP][kPer];
  Stat<double> a = stat_zero<double>();
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    load_z<T, double>(p, c, g.row, g.j(k), n ? n + g.j(k) : nullptr, z[k]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (!(z[k][i] < (double)INFINITY)) a.bad = 1;
      if (z[k][i] > a.m) a.m = z[k][i], a.best = g.j(k) + i;
    }
  }
  const double m = lanes_max(a.m, g.width);
  int32_t best = a.m == m && a.best < INT32_MAX ? (int32_t)a.best : INT32_MAX;
  a.m = m;
  a.best = lanes_min(best, g.width);
  a.bad = lanes_max(a.bad, g.width);
  double w[NP][kPer];
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const double d = (z[k][i] - m) * c.inv_t;
      w[k][i] = exp_of(d);
      a.s += w[k][i];
      if (w[k][i] > 0) a.e += w[k][i] * d;
    }
  a.s = lanes_sum(a.s, g.width);
  a.e = lanes_sum(a.e, g.width);
  int32_t pick = (int32_t)a.best;
  double z_pick = m;
  if (u) {
    const double target = (u_f64 ? ((const double*)u)[g.row] : (double)((const float*)u)[g.row]) * a.s;
    double before = 0;
    int32_t hit = INT32_MAX, last = -1;
    double hit_z = 0, last_z = 0;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      double sum = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum += w[k][i];
      const double incl = lanes_scan(sum, g.width);
      double cum = before + incl - sum;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        cum += w[k][i];
        if (w[k][i] > 0) {
          last = (int32_t)g.j(k) + i, last_z = z[k][i];
          if (hit == INT32_MAX && cum > target) hit = last, hit_z = last_z;
        }
      }
      before += __shfl(incl, (threadIdx.x & 63) | (g.width - 1), 64);
    }
    pick = lanes_min(hit, g.width);
    if (pick == INT32_MAX) {  // (a sum that rounding left short of the target: the last option with any weight)
      pick = lanes_max(last, g.width);
      hit = last, hit_z = last_z;
    }
    z_pick = lanes_max(hit == pick ? hit_z : neg_inf<double>(), g.width);
  }
  if (g.lane == 0 && g.there) finish_choose(out, g.row, a, c.bad, c.inv_t, pick, z_pick);
}

template <class T, int NP> __global__ __launch_bounds__(kThreads) void evaluate_group(Rows p, int width_log, EvaluateOut out) {
  extern __shared__ uint32_t counts[];
  const Group g = group_of(p, blockIdx.x, width_log);
  const RowConst<float> c = row_const<float>(p, g.row);
  const uint32_t* n = count_groups<NP>(p, g, counts);
  const int32_t act = out.action[g.row];
  float z[NP][kPer];
  Stat<float> a = stat_zero<float>();
  float z_act = -INFINITY;
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    load_z<T, float>(p, c, g.row, g.j(k), n ? n + g.j(k) : nullptr, z[k]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (!(z[k][i] < INFINITY)) a.bad = 1;
      a.m = fmaxf(a.m, z[k][i]);
      if (act == g.j(k) + i) z_act = z[k][i];
    }
  }
  a.m = lanes_max(a.m, g.width);
  a.bad = lanes_max(a.bad, g.width);
  z_act = lanes_max(z_act, g.width);
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float d = (z[k][i] - a.m) * c.inv_t;
      const float w = exp_of(d);
      if (w > 0.f) a.s += w, a.e += w * d;
    }
  a.s = lanes_sum(a.s, g.width);
  a.e = lanes_sum(a.e, g.width);
  if (g.lane == 0 && g.there) finish_evaluate(out, g.row, p.options, a, c.bad, c.inv_t, act, z_act);
}

// ---- longer rows: a workgroup per part of a row (`pieces` pieces of kPiece options), parts joined after ---
template <class T>
__global__ __launch_bounds__(kThreads) void choose_parts(Rows p, int pieces, int n_parts, Stat<double>* parts) {
  __shared__ uint32_t counts[kPiece];
  __shared__ Stat<double> red[kThreads / 64];
  const int64_t row = blockIdx.x / n_parts, part = blockIdx.x % n_parts;
  const RowConst<double> c = row_const<double>(p, row);
  Stat<double> a = stat_zero<double>();
  const int64_t j_end = min((part + 1) * pieces * (int64_t)kPiece, c.n_legal);
  for (int64_t j0 = part * pieces * (int64_t)kPiece; j0 < j_end; j0 += kPiece) {
    if (p.history) count_piece(p, row, j0, counts);
    const int64_t j = j0 + threadIdx.x * kPer;
    double z[kPer];
    load_z<T, double>(p, c, row, j, p.history ? counts + threadIdx.x * kPer : nullptr, z);
    stat_add(a, z, j, c.inv_t);
  }
  a = stat_block(a, c.inv_t, red);
  if (threadIdx.x == 0) parts[blockIdx.x] = a;
}

// joins a row's parts, and finds the option that u falls on by walking down the one part it lies in
template <class T>
__global__ __launch_bounds__(kThreads) void choose_join(Rows p, int pieces, int n_parts, const Stat<double>* all_parts, const void* u, int u_f64, ChooseOut out) {
  __shared__ uint32_t counts[kPiece];
  __shared__ Stat<double> red[kThreads / 64];
  __shared__ double wave_sum[kThreads / 64];
  __shared__ long long found;
  __shared__ double found_z, part_before;
  __shared__ int part_at;
  const int64_t row = blockIdx.x;
  const Stat<double>* parts = all_parts + row * n_parts;
  const RowConst<double> c = row_const<double>(p, row);
  Stat<double> a = stat_zero<double>();
  for (int i = threadIdx.x; i < n_parts; i += kThreads) {
    Stat<double> b = parts[i];
    const double m = a.m > b.m ? a.m : b.m;
    const int64_t best = a.m > b.m ? a.best : (b.m > a.m ? b.best : min(a.best, b.best));
    stat_rebase(a, m, c.inv_t);
    stat_rebase(b, m, c.inv_t);
    a = {m, a.s + b.s, a.e + b.e, best, a.bad | b.bad};
  }
  a = stat_block(a, c.inv_t, red);
  const bool bad = a.bad || c.bad, empty = !bad && a.m == neg_inf<double>();
  int64_t pick = a.best;
  double z_pick = a.m;
  if (u && !bad && !empty) {
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
          stat_rebase(b, a.m, c.inv_t);
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
    double last_z = 0;
    const int64_t j_first = part_at * (int64_t)pieces * kPiece, j_end = min(j_first + pieces * (int64_t)kPiece, c.n_legal);
    for (int64_t j0 = j_first; j0 < j_end; j0 += kPiece) {
      if (p.history) count_piece(p, row, j0, counts);
      const int64_t j = j0 + threadIdx.x * kPer;
      double z[kPer], w[kPer], sum = 0;
      load_z<T, double>(p, c, row, j, p.history ? counts + threadIdx.x * kPer : nullptr, z);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        w[i] = exp_of((z[i] - a.m) * c.inv_t);
        sum += w[i];
        if (w[i] > 0) last = j + i, last_z = z[i];
      }
      const double incl = lanes_scan(sum, 64);
      __syncthreads();
      if ((threadIdx.x & 63) == 63) wave_sum[threadIdx.x >> 6] = incl;
      __syncthreads();
      double cum = before + incl - sum;
      for (int i = 0; i < (int)(threadIdx.x >> 6); ++i) cum += wave_sum[i];
      int64_t hit = INT64_MAX;
      double hit_z = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        cum += w[i];
        if (hit == INT64_MAX && w[i] > 0 && cum > target) hit = j + i, hit_z = z[i];
      }
      if (hit != INT64_MAX) atomicMin(&found, (long long)hit);
      __syncthreads();
      if (hit != INT64_MAX && hit == found) found_z = hit_z;
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
      if (last == found) found_z = last_z;
      __syncthreads();
    }
    pick = found;
    z_pick = found_z;
  }
  if (threadIdx.x == 0) finish_choose(out, row, a, c.bad, c.inv_t, pick, z_pick);
}

// The same walk in 32 bits. One part: the row's results at once; several: partial sums, with the logit of the
// action from the part that holds it.
struct EvaluatePart {
  Stat<float> stat;
  float z_act;
};
template <class T>
__global__ __launch_bounds__(kThreads) void evaluate_parts(Rows p, int pieces, int n_parts, EvaluatePart* parts, EvaluateOut out) {
  __shared__ uint32_t counts[kPiece];
  __shared__ Stat<float> red[kThreads / 64];
  __shared__ float z_act;
  const int64_t row = blockIdx.x / n_parts, part = blockIdx.x % n_parts;
  const RowConst<float> c = row_const<float>(p, row);
  const int32_t act = out.action[row];
  Stat<float> a = stat_zero<float>();
  if (threadIdx.x == 0) z_act = -INFINITY;
  __syncthreads();
  const int64_t j_end = min((part + 1) * pieces * (int64_t)kPiece, c.n_legal);
  for (int64_t j0 = part * pieces * (int64_t)kPiece; j0 < j_end; j0 += kPiece) {
    if (p.history) count_piece(p, row, j0, counts);
    const int64_t j = j0 + threadIdx.x * kPer;
    float z[kPer];
    load_z<T, float>(p, c, row, j, p.history ? counts + threadIdx.x * kPer : nullptr, z);
    stat_add(a, z, j, c.inv_t);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (act == j + i) z_act = z[i];
  }
  a = stat_block(a, c.inv_t, red);
  if (threadIdx.x != 0) return;
  if (n_parts == 1) finish_evaluate(out, row, p.options, a, c.bad, c.inv_t, act, z_act);
  else parts[blockIdx.x] = {a, z_act};
}
__global__ __launch_bounds__(kThreads) inline void evaluate_join(Rows p, int n_parts, const EvaluatePart* all_parts, EvaluateOut out) {
  // one wave per row
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const RowConst<float> c = row_const<float>(p, row);
  const EvaluatePart* parts = all_parts + row * n_parts;
  Stat<float> a = stat_zero<float>();
  float z_act = -INFINITY;
  for (int i = threadIdx.x & 63; i < n_parts; i += 64) {
    EvaluatePart b = parts[i];
    const float m = fmaxf(a.m, b.stat.m);
    stat_rebase(a, m, c.inv_t);
    stat_rebase(b.stat, m, c.inv_t);
    a.s += b.stat.s, a.e += b.stat.e, a.bad |= b.stat.bad;
    z_act = fmaxf(z_act, b.z_act);
  }
  const float m = lanes_max(a.m, 64);
  stat_rebase(a, m, c.inv_t);
  a.s = lanes_sum(a.s, 64), a.e = lanes_sum(a.e, 64), a.bad = lanes_max(a.bad, 64);
  z_act = lanes_max(z_act, 64);
  if ((threadIdx.x & 63) == 0) finish_evaluate(out, row, p.options, a, c.bad, c.inv_t, out.action[row], z_act);
}

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

// per-row factors of the gradient
struct GradRow {
  float m, log_s, h, g1, g2;
  int32_t act;
};
__device__ inline GradRow grad_row(const GradArgs& g, int64_t row) {
  GradRow r;
  r.m = g.stats[2 * row];
  r.log_s = g.stats[2 * row + 1];
  r.h = g.entropy[row];
  r.g1 = g.g_lp ? g.g_lp[row] : 0.f;
  r.g2 = g.g_h ? g.g_h[row] : 0.f;
  r.act = g.action[row];
  if (r.act == -1) r.g1 = 0.f;
  return r;
}
// d/dy of g1 log p[act] + g2 H for one option
__device__ inline float grad_y(const GradRow& r, float z, bool legal, bool is_act, float inv_t) {
  if (!legal || r.m == -INFINITY) return 0.f;
  const float d = (z - r.m) * inv_t - r.log_s;
  const float pr = exp_of(d);
  const float ent = pr > 0.f ? r.g2 * pr * (d + r.h) : 0.f;
  return r.g1 * ((is_act ? 1.f : 0.f) - pr) - ent + (pr != pr ? pr : 0.f);
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
// over the workgroup's row slots
template <class T, int NP> __global__ __launch_bounds__(kThreads) void evaluate_grad_group(Rows p, GradArgs g, int width_log, int64_t blocks_of_rows) {
  extern __shared__ uint32_t counts[];  // (as floats for the sums afterwards)
  float sum[NP][kPer];
#pragma unroll
  for (int k = 0; k < NP; ++k)
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum[k][i] = 0.f;
  for (int64_t b = blockIdx.x; b < blocks_of_rows; b += gridDim.x) {
    const Group at = group_of(p, b, width_log);
    const uint32_t* n = count_groups<NP>(p, at, counts);
    if (!at.there) continue;
    const RowConst<float> c = row_const<float>(p, at.row);
    const GradRow r = grad_row(g, at.row);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int64_t j = at.j(k);
      if (j >= p.options) continue;
      float z[kPer], slope[kPer], dx[kPer], db[kPer];
      const uint32_t legal = load_z<T, float>(p, c, at.row, j, n ? n + j : nullptr, z, slope);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const bool ok = (legal >> i) & 1;
        db[i] = grad_y(r, z[i], ok, r.act == j + i, c.inv_t) * c.inv_t;
        dx[i] = ok ? db[i] * slope[i] : 0.f;
        sum[k][i] += db[i];
      }
      if (g.grad_logits) store8<T>((T*)g.grad_logits + at.row * g.grad_logits_stride + j, dx, j, p.options, g.vec_out);
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

// a workgroup owns kPiece columns and walks down its rows: the sum of a shared bias' gradient stays in registers
template <class T>
__global__ __launch_bounds__(kThreads) void evaluate_grad_piece(Rows p, GradArgs g, int64_t rows_per_block) {
  __shared__ uint32_t counts[kPiece];
  const int64_t j0 = (int64_t)blockIdx.x * kPiece;
  const int64_t j = j0 + threadIdx.x * kPer;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per_block;
  const int64_t r1 = r0 + rows_per_block < p.rows ? r0 + rows_per_block : p.rows;
  float sum[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum[i] = 0.f;
  for (int64_t row = r0; row < r1; ++row) {
    const RowConst<float> c = row_const<float>(p, row);
    const GradRow r = grad_row(g, row);
    if (p.history) count_piece(p, row, j0, counts);
    if (j >= p.options) continue;
    float z[kPer], slope[kPer], dx[kPer], db[kPer];
    const uint32_t legal = load_z<T, float>(p, c, row, j, p.history ? counts + threadIdx.x * kPer : nullptr, z, slope);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool ok = (legal >> i) & 1;
      db[i] = grad_y(r, z[i], ok, r.act == j + i, c.inv_t) * c.inv_t;
      dx[i] = ok ? db[i] * slope[i] : 0.f;
      sum[i] += db[i];
    }
    if (g.grad_logits) store8<T>((T*)g.grad_logits + row * g.grad_logits_stride + j, dx, j, p.options, g.vec_out);
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

// column sums of partial [n][options], in order of the rows
template <class T>
__global__ __launch_bounds__(kThreads) void sum_partials(const float* partial, int64_t n, int64_t options, T* out) {
  __shared__ float red[kThreads];
  // 16 columns a workgroup, 16 threads down each
  const int64_t j = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  float s = 0.f;
  if (j < options)
    for (int64_t i = threadIdx.x >> 4; i < n; i += kThreads / 16) s += partial[i * options + j];
  red[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 16 && j < options) {
    for (int i = 1; i < kThreads / 16; ++i) s += red[threadIdx.x + 16 * i];
    out[j] = (T)s;
  }
}

}  // namespace epp
