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

__device__ inline double exp_of(double x) { return exp(x); }
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
template <class R> __device__ inline Stat<R> stat_join(Stat<R> a, Stat<R> b, R inv_t) {
  const R m = a.m > b.m ? a.m : b.m;
  const int64_t best = a.m > b.m ? a.best : (b.m > a.m ? b.best : (a.best < b.best ? a.best : b.best));
  stat_rebase(a, m, inv_t);
  stat_rebase(b, m, inv_t);
  return {m, a.s + b.s, a.e + b.e, best, a.bad | b.bad};
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

template <class R> __device__ inline R shfl_xor_of(R v, int lane_mask) { return __shfl_xor(v, lane_mask, 64); }
template <class R> __device__ inline Stat<R> stat_shfl(const Stat<R>& a, int lane_mask) {
  return {shfl_xor_of(a.m, lane_mask), shfl_xor_of(a.s, lane_mask), shfl_xor_of(a.e, lane_mask),
          (int64_t)__shfl_xor((long long)a.best, lane_mask, 64), __shfl_xor(a.bad, lane_mask, 64)};
}
// over the block; the result is the same in every thread
template <class R> __device__ inline Stat<R> stat_block(Stat<R> a, R inv_t, Stat<R>* lds) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Stat<R> b = stat_shfl(a, o);
    // the same order of the two in both lanes, so that both get the same bits
    a = (threadIdx.x & o) ? stat_join(b, a, inv_t) : stat_join(a, b, inv_t);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  Stat<R> r = lds[0];
  for (int i = 1; i < kThreads / 64; ++i) r = stat_join(r, lds[i], inv_t);
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

// ---- one workgroup per row --------------------------------------------------------------------------
template <class T>
__global__ __launch_bounds__(kThreads) void choose_row(Rows p, const void* u, int u_f64, int32_t* action, float* log_prob,
                                                       float* entropy) {
  __shared__ uint32_t counts[kPiece];
  __shared__ Stat<double> red[kThreads / 64];
  __shared__ double wave_sum[kThreads / 64];
  __shared__ int64_t found;
  __shared__ double found_z;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const RowConst<double> c = row_const<double>(p, row);
    Stat<double> a = stat_zero<double>();
    for (int64_t j0 = 0; j0 < c.n_legal; j0 += kPiece) {
      if (p.history) count_piece(p, row, j0, counts);
      const int64_t j = j0 + threadIdx.x * kPer;
      double z[kPer];
      load_z<T, double>(p, c, row, j, p.history ? counts + threadIdx.x * kPer : nullptr, z);
      stat_add(a, z, j, c.inv_t);
    }
    a = stat_block(a, c.inv_t, red);
    const bool bad = a.bad || c.bad;
    const bool empty = !bad && a.m == neg_inf<double>();
    int64_t pick = a.best;
    double z_pick = a.m;
    if (u && !bad && !empty) {
      const double target = (u_f64 ? ((const double*)u)[row] : (double)((const float*)u)[row]) * a.s;
      if (threadIdx.x == 0) found = INT64_MAX;
      double before = 0;
      int64_t last = -1;  // the last option with any weight: where a sum that rounding left short ends
      double last_z = 0;
      for (int64_t j0 = 0; j0 < c.n_legal; j0 += kPiece) {
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
        double incl = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const double t = __shfl_up(incl, o, 64);
          if ((int)(threadIdx.x & 63) >= o) incl += t;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 63) wave_sum[threadIdx.x >> 6] = incl;
        __syncthreads();
        double base = before;
        for (int i = 0; i < (int)(threadIdx.x >> 6); ++i) base += wave_sum[i];
        double cum = base + incl - sum;
        int64_t hit = INT64_MAX;
        double hit_z = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          cum += w[i];
          if (hit == INT64_MAX && w[i] > 0 && cum > target) hit = j + i, hit_z = z[i];
        }
        if (hit != INT64_MAX) atomicMin((unsigned long long*)&found, (unsigned long long)hit);
        __syncthreads();
        if (hit != INT64_MAX && hit == found) found_z = hit_z;
        __syncthreads();
        if (found != INT64_MAX) break;
        for (int i = 0; i < kThreads / 64; ++i) before += wave_sum[i];
      }
      if (found == INT64_MAX) {
        __syncthreads();
        if (threadIdx.x == 0) found = -1;
        __syncthreads();
        atomicMax((long long*)&found, (long long)last);
        __syncthreads();
        if (last == found) found_z = last_z;
        __syncthreads();
      }
      pick = found;
      z_pick = found_z;
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      const double log_s = log(a.s);
      action[row] = bad || empty ? -1 : (int32_t)pick;
      log_prob[row] = bad ? quiet_nan<float>() : empty ? 0.f : (float)((z_pick - a.m) * c.inv_t - log_s);
      entropy[row] = bad ? quiet_nan<float>() : empty ? 0.f : (float)(log_s - a.e / a.s);
    }
  }
}

// results of one row of ep_policy_evaluate, from its statistics
__device__ inline void finish_evaluate(int64_t row, const Rows& p, const RowConst<float>& c, const Stat<float>& a, int32_t act,
                                       float z_act, float* log_prob, float* entropy, float* stats) {
  const bool bad = a.bad || c.bad;
  const bool empty = !bad && a.m == -INFINITY;
  const float log_s = logf(a.s);
  float lp;
  if (act == -1) lp = 0.f;
  else if (act < 0 || act >= p.options) lp = quiet_nan<float>();
  else if (empty || z_act == -INFINITY) lp = -INFINITY;
  else lp = (z_act - a.m) * c.inv_t - log_s;
  log_prob[row] = bad ? quiet_nan<float>() : lp;
  entropy[row] = bad ? quiet_nan<float>() : empty ? 0.f : log_s - a.e / a.s;
  stats[2 * row] = bad ? quiet_nan<float>() : a.m;
  stats[2 * row + 1] = bad ? quiet_nan<float>() : empty ? 0.f : log_s;
}

template <class T>
__global__ __launch_bounds__(kThreads) void evaluate_row(Rows p, const int32_t* action, float* log_prob, float* entropy, float* stats) {
  __shared__ uint32_t counts[kPiece];
  __shared__ Stat<float> red[kThreads / 64];
  __shared__ float z_act;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const RowConst<float> c = row_const<float>(p, row);
    const int32_t act = action[row];
    Stat<float> a = stat_zero<float>();
    __syncthreads();
    if (threadIdx.x == 0) z_act = -INFINITY;
    __syncthreads();
    for (int64_t j0 = 0; j0 < c.n_legal; j0 += kPiece) {
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
    if (threadIdx.x == 0) finish_evaluate(row, p, c, a, act, z_act, log_prob, entropy, stats);
  }
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
