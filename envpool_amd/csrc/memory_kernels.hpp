// memory_kernels.hpp - device code of the per-env linear-attention memory (memory.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace epm {

using bf16 = __bf16;
using f16 = _Float16;

struct Step {
  int64_t num_envs, rows;
  int32_t heads, kv_group, dk, dv;
  const void *q, *k, *v;
  int64_t q_stride[2], k_stride[2], v_stride[2], out_stride[2];
  void* out;
  const float* log_decay;
  float* state;
  const int32_t* env_id;
  int32_t env_id_offset;
  const void* fresh;
  int32_t fresh_i32;
  float scale;
  int32_t* error;
  int32_t* claims;  // [num_envs]: how many rows name the env (NULL: look the ids through instead)
};

__device__ inline bool starts(const Step& p, int64_t row) {
  if (!p.fresh) return false;
  return p.fresh_i32 ? ((const int32_t*)p.fresh)[row] == 0 : ((const uint8_t*)p.fresh)[row] != 0;
}

// claims of the envs that this batch names: zeroed, then counted
static __global__ __launch_bounds__(256) void clear_claims(Step p) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= p.rows) return;
  const int64_t e = (int64_t)p.env_id[r] - p.env_id_offset;
  if (e >= 0 && e < p.num_envs) p.claims[e] = 0;
}
static __global__ __launch_bounds__(256) void count_claims(Step p) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= p.rows) return;
  const int64_t e = (int64_t)p.env_id[r] - p.env_id_offset;
  if (e >= 0 && e < p.num_envs) atomicAdd(&p.claims[e], 1);
}

// the states of the envs that a batch names, zeroed: a workgroup per row and stretch of it
static __global__ __launch_bounds__(256) void reset_rows(Step p, int64_t size, int64_t stretches) {
  for (int64_t i = blockIdx.x; i < p.rows * stretches; i += gridDim.x) {
    const int64_t row = i / stretches, e = p.env_id ? (int64_t)p.env_id[row] - p.env_id_offset : row;
    if (e < 0 || e >= p.num_envs) {
      if (threadIdx.x == 0 && p.error) *p.error = 1;
      continue;
    }
    for (int64_t j = i % stretches * 256 + threadIdx.x; j < size; j += stretches * 256) p.state[e * size + j] = 0.f;
  }
}

// One wave per (row, head) streams the state through its registers: a lane holds kVec neighbouring value columns (or
// kCols such pieces, 64 apart) and walks down the keys, 64 / (lanes per key row) keys an instruction, so that the load
// instructions of the wave are one contiguous stretch. Nothing is read twice; HBM bounds it (8 bytes moved per 5 flops), so what matters
// is bytes in flight: 128 of every lane (32 / kVec loads) before the first is used. State loads and stores bypass the caches'
// retention (a step touches each value once). 4096 rows x 8 heads of 64 x 64, bf16: 195 us = 5.6 TB/s; 65536 x 4
// heads of 32 x 32: 433 us = 5.1 TB/s; a pool of 8 envs 6.6 us.
// orders a wave's LDS accesses across its lanes (the hardware keeps them in order; this tells the compiler)
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
template <int kVec> struct Piece {
  typedef float type __attribute__((ext_vector_type(kVec)));
};
template <> struct Piece<1> {
  typedef float type;
};

template <class T, int kVec, int kCols> __device__ inline void step_one(const Step& p, int64_t row, int64_t e, int h, float decay, float* qs, float* ks, float* red) {
  using V = typename Piece<kVec>::type;
  const int lane = threadIdx.x & 63;
  const bool drop = starts(p, row);
  const T* q = (const T*)p.q + row * p.q_stride[0] + h * p.q_stride[1];
  const T* k = (const T*)p.k + row * p.k_stride[0] + (h / p.kv_group) * p.k_stride[1];
  const T* v = (const T*)p.v + row * p.v_stride[0] + (h / p.kv_group) * p.v_stride[1];
  T* out = (T*)p.out + row * p.out_stride[0] + h * p.out_stride[1];
  float* state = p.state + (e * p.heads + h) * (int64_t)p.dk * p.dv;
  wave_sync();
  for (int i = lane; i < p.dk; i += 64) qs[i] = (float)q[i] * p.scale, ks[i] = (float)k[i];
  wave_sync();
  // columns of kVec values (dv is a multiple of it): up to 64 side by side, a lane holds every 64th of more
  const int columns = p.dv / kVec, width = columns < 64 ? columns : 64;
  const int down = kCols == 1 ? 64 / width : 1;  // keys per instruction
  const int c = lane % width, d0 = lane / width;
  const bool on = d0 < down;
  // (`on` again inside the walk keeps the loads of narrow pieces together: 2692 states of 101 x 66 take 45 us with it, 54
  // without. Wide ones take 429 us for 262144 states of 32 x 32 without it and with five workgroups a CU, 464 with it
  // and four)
  const auto has = [&](int j) { return kCols == 1 ? kVec == 4 || on : c + 64 * j < columns; };
  float* s = state + c * kVec;
  V vv[kCols], acc[kCols];
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    acc[j] = (V)0.f;
    if constexpr (kVec == 1) vv[j] = on && has(j) ? (float)v[c + 64 * j] : 0.f;
    else
#pragma unroll
      for (int r = 0; r < kVec; ++r) vv[j][r] = on && has(j) ? (float)v[(c + 64 * j) * kVec + r] : 0.f;
  }
  constexpr int kKeys = 32 / (kVec * kCols);
  for (int i0 = on ? d0 : p.dk; i0 < p.dk; i0 += down * kKeys) {
    V old[kKeys][kCols];
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int d = i0 + i * down;
        old[i][j] = (V)0.f;
        if (d < p.dk && !drop && has(j)) old[i][j] = __builtin_nontemporal_load((const V*)(s + (int64_t)d * p.dv + 64 * kVec * j));
      }
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const int d = i0 + i * down;
        if (d < p.dk && has(j)) {
          const V now = old[i][j] * decay + ks[d] * vv[j];
          __builtin_nontemporal_store(now, (V*)(s + (int64_t)d * p.dv + 64 * kVec * j));
          acc[j] += qs[d] * now;
        }
      }
  }
  if (kCols > 1) {  // (a lane has been down all keys of its columns)
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (has(j)) {
        if constexpr (kVec == 1) out[c + 64 * j] = (T)acc[j];
        else
#pragma unroll
          for (int r = 0; r < kVec; ++r) out[(c + 64 * j) * kVec + r] = (T)acc[j][r];
      }
    return;
  }
  // the sums over the keys: `down` lanes apart by `width`
  wave_sync();
#pragma unroll
  for (int r = 0; r < kVec; ++r) {
    if constexpr (kVec == 1) red[lane] = acc[0];
    else red[r * 64 + lane] = acc[0][r];
  }
  wave_sync();
  if (lane < width) {
#pragma unroll
    for (int r = 0; r < kVec; ++r) {
      float sum = 0.f;
      for (int i = 0; i < down; ++i) sum += red[r * 64 + i * width + lane];
      out[c * kVec + r] = (T)sum;
    }
  }
}

// Rows of one env are stepped by the wave of the first of them, in order.
template <class T, int kVec, int kCols> __global__ __launch_bounds__(256, kVec == 4 ? 5 : 3) void step_rows(Step p) {
  __shared__ float lds[4][256 + 256 + 64 * kVec];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float *qs = lds[wave], *ks = qs + 256, *red = ks + 256;  // a wave's own: its LDS operations are in order
  const int64_t item = (int64_t)blockIdx.x * 4 + wave;
  if (item >= p.rows * p.heads) return;
  const int64_t row0 = item / p.heads;
  const int h = (int)(item % p.heads);
  const float decay = expf(p.log_decay[h]);
  const int64_t id = p.env_id ? p.env_id[row0] : row0 + p.env_id_offset;
  const int64_t e = id - p.env_id_offset;
  if (e < 0 || e >= p.num_envs) {
    if (lane == 0 && h == 0 && p.error) *p.error = 1;
    for (int j = lane; j < p.dv; j += 64) ((T*)p.out)[row0 * p.out_stride[0] + h * p.out_stride[1] + j] = (T)__builtin_nanf("");
    return;
  }
  int again = 0;
  if (p.env_id && (!p.claims || p.claims[e] > 1)) {
    int earlier = 0;
    for (int64_t r = lane; r < p.rows; r += 64)
      if (p.env_id[r] == id) {
        if (r < row0) earlier = 1;
        if (r > row0) again = 1;
      }
    if (__any(earlier)) return;
    again = __any(again);
  }
  step_one<T, kVec, kCols>(p, row0, e, h, decay, qs, ks, red);
  if (!again) return;
  for (int64_t base = row0 / 64 * 64; base < p.rows; base += 64) {
    uint64_t hits = __ballot(base + lane < p.rows && base + lane > row0 && p.env_id[base + lane] == id);
    for (; hits; hits &= hits - 1) {
      __threadfence_block();  // (the state written for the row before is read again)
      step_one<T, kVec, kCols>(p, base + __ffsll((unsigned long long)hits) - 1, e, h, decay, qs, ks, red);
    }
  }
}

struct Scan {
  int64_t steps, rows;
  int32_t heads, q_group, k_group, v_group, dk, dv;
  const void *q, *k, *v;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
  void* out;
  int32_t out_f32;
  const float* log_decay;
  const uint8_t* fresh;
  int64_t fresh_stride[2];
  const float* state_in;
  float* state_out;
  int64_t in_stride[4], outs_stride[4];
  float inc_scale, out_scale;
  int32_t reverse;
};

// A scan of few steps (ep_memory_scan, either direction of time): step by step, one wave per state, which stays in the
// wave's registers from the first step to the last. Lane (d0, c) holds kKeys keys from d0 * kKeys on and the four values
// from 4c on; a step's q, k and v go through LDS, the next one's are on their way meanwhile. A chunk of the matrix-core
// walk costs the same however few of its steps there are; this costs kKeys * 12 multiplications and additions a
// step and lane, and moves nothing twice. Up to 64 x 64, any strides.
typedef float f32x4_few __attribute__((ext_vector_type(4)));
template <class T, int kKeys> __global__ __launch_bounds__(256) void scan_few(Scan p, int width_log, int in_rows, int in_cols, int out_rows, int out_cols) {
  using V = f32x4_few;
  __shared__ __align__(16) float lds[4][2][3][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * 4 + wave;
  if (item >= p.rows * p.heads) return;
  const int64_t row = item / p.heads;
  const int h = (int)(item % p.heads);
  const int width = 1 << width_log, c = lane & (width - 1), first = (lane >> width_log) * kKeys;
  const float decay = expf(p.log_decay[h]);
  const T* gq = (const T*)p.q + row * p.q_stride[1] + (h / p.q_group) * p.q_stride[2] + lane;
  const T* gk = (const T*)p.k + row * p.k_stride[1] + (h / p.k_group) * p.k_stride[2] + lane;
  const T* gv = (const T*)p.v + row * p.v_stride[1] + (h / p.v_group) * p.v_stride[2] + lane;
  T rq = (T)0.f, rk = (T)0.f, rv = (T)0.f;
  uint8_t rf = 0;
  const auto ask = [&](int64_t t) {
    if (lane < p.dk) rq = gq[t * p.q_stride[0]], rk = gk[t * p.k_stride[0]];
    if (lane < p.dv) rv = gv[t * p.v_stride[0]];
    if (p.fresh) rf = p.fresh[t * p.fresh_stride[0] + row * p.fresh_stride[1]];
  };
  ask(p.reverse ? p.steps - 1 : 0);

  V s[kKeys];
#pragma unroll
  for (int i = 0; i < kKeys; ++i) s[i] = (V)0.f;
  if (p.state_in) {
    const float* a = p.state_in + row * p.in_stride[0] + h * p.in_stride[1];
    if (in_rows) {  // a key's values follow one another, in 16-byte pieces
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
        if (first + i < p.dk && 4 * c < p.dv) s[i] = *(const V*)(a + (first + i) * p.in_stride[2] + 4 * c);
    } else if (in_cols) {  // a value's keys do
#pragma unroll
      for (int i = 0; i < kKeys; i += 4)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (first + i < p.dk && 4 * c + r < p.dv) {
            const V x = *(const V*)(a + (4 * c + r) * p.in_stride[3] + first + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i + e][r] = x[e];
          }
    } else {
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (first + i < p.dk && 4 * c + r < p.dv) s[i][r] = a[(first + i) * p.in_stride[2] + (4 * c + r) * p.in_stride[3]];
    }
  }
  float carry = p.reverse ? 1.f : decay;  // (back in time, what enters the last step has not decayed)
  bool drop = false;
  for (int64_t n = 0; n < p.steps; ++n) {
    const int64_t t = p.reverse ? p.steps - 1 - n : n;
    float(*now)[64] = lds[wave][n & 1];
    now[0][lane] = (float)rq, now[1][lane] = (float)rk, now[2][lane] = (float)rv * p.inc_scale;
    const bool fresh = rf != 0;
    if (n + 1 < p.steps) ask(p.reverse ? t - 1 : t + 1);
    wave_sync();
    if (!p.reverse) drop = fresh;
    if (drop) {  // (not a product with 0: what was there may not be finite)
#pragma unroll
      for (int i = 0; i < kKeys; ++i) s[i] = (V)0.f;
    }
    const V v = *(const V*)&now[2][4 * c];
    V acc = (V)0.f;
#pragma unroll
    for (int i = 0; i < kKeys; i += 4) {
      const V q = *(const V*)&now[0][first + i], k = *(const V*)&now[1][first + i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i + e] = s[i + e] * carry + k[e] * v;
        acc += q[e] * s[i + e];
      }
    }
    carry = decay, drop = fresh;
    if (!p.out) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      for (int o = 32; o >= width; o >>= 1) acc[r] += __shfl_xor(acc[r], o, 64);
    if (first == 0) {
      const int64_t to = t * p.out_stride[0] + row * p.out_stride[1] + h * p.out_stride[2] + 4 * c;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * c + r < p.dv) {
          if (p.out_f32) ((float*)p.out)[to + r] = acc[r] * p.out_scale;
          else ((T*)p.out)[to + r] = (T)(acc[r] * p.out_scale);
        }
    }
  }
  if (!p.state_out) return;
  if (p.reverse) {
#pragma unroll
    for (int i = 0; i < kKeys; ++i) s[i] = drop ? (V)0.f : s[i] * decay;
  }
  float* a = p.state_out + row * p.outs_stride[0] + h * p.outs_stride[1];
  if (out_rows) {
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
      if (first + i < p.dk && 4 * c < p.dv) *(V*)(a + (first + i) * p.outs_stride[2] + 4 * c) = s[i];
  } else if (out_cols) {
#pragma unroll
    for (int i = 0; i < kKeys; i += 4)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (first + i < p.dk && 4 * c + r < p.dv) *(V*)(a + (4 * c + r) * p.outs_stride[3] + first + i) = V{s[i][r], s[i + 1][r], s[i + 2][r], s[i + 3][r]};
  } else {
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (first + i < p.dk && 4 * c + r < p.dv) a[(first + i) * p.outs_stride[2] + (4 * c + r) * p.outs_stride[3]] = s[i][r];
  }
}

// gradients of heads that share keys and values, summed in 32 bits and rounded once (5 us at 777 x 5 x 2 x 112)
template <class T> __global__ __launch_bounds__(256) void sum_heads(const float* src, int64_t total, int32_t group, int32_t dim, T* out) {
  // over [n][heads_out][dim]
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t head = i / dim, d = i % dim;
    float s = 0.f;
    for (int g = 0; g < group; ++g) s += src[(head * group + g) * dim + d];
    out[i] = (T)s;
  }
}

}  // namespace epm
