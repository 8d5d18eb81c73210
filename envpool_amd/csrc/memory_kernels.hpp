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
__global__ __launch_bounds__(256) void clear_claims(Step p) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= p.rows) return;
  const int64_t e = (int64_t)p.env_id[r] - p.env_id_offset;
  if (e >= 0 && e < p.num_envs) p.claims[e] = 0;
}
__global__ __launch_bounds__(256) void count_claims(Step p) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= p.rows) return;
  const int64_t e = (int64_t)p.env_id[r] - p.env_id_offset;
  if (e >= 0 && e < p.num_envs) atomicAdd(&p.claims[e], 1);
}

// One workgroup per (row, head): thread = (value column, key part). Rows of one env are stepped by the
// workgroup of the first of them, in order.
template <class T> __global__ __launch_bounds__(256) void step_row(Step p) {
  __shared__ float qs[256], ks[256];
  __shared__ float part[256];
  __shared__ int earlier, again;
  const int h = blockIdx.y;
  const float decay = expf(p.log_decay[h]);
  for (int64_t row0 = blockIdx.x; row0 < p.rows; row0 += gridDim.x) {
    const int64_t id = p.env_id ? p.env_id[row0] : row0 + p.env_id_offset;
    const int64_t e = id - p.env_id_offset;
    if (e < 0 || e >= p.num_envs) {
      if (threadIdx.x == 0 && h == 0 && p.error) *p.error = 1;
      for (int j = threadIdx.x; j < p.dv; j += 256)
        ((T*)p.out)[row0 * p.out_stride[0] + h * p.out_stride[1] + j] = (T)__builtin_nanf("");
      continue;
    }
    __syncthreads();
    if (threadIdx.x == 0) earlier = again = 0;
    __syncthreads();
    if (p.env_id && (!p.claims || p.claims[e] > 1)) {
      for (int64_t r = threadIdx.x; r < p.rows; r += 256)
        if (r != row0 && p.env_id[r] == id) {
          if (r < row0) earlier = 1;
          else again = 1;
        }
    }
    __syncthreads();
    if (earlier) continue;
    float* s = p.state + (e * p.heads + h) * (int64_t)p.dk * p.dv;
    const bool repeats = again != 0;
    for (int64_t row = row0; row < p.rows; ++row) {
      if (row > row0 && p.env_id[row] != id) continue;
      const float keep = starts(p, row) ? 0.f : decay;
      const T* q = (const T*)p.q + row * p.q_stride[0] + h * p.q_stride[1];
      const T* k = (const T*)p.k + row * p.k_stride[0] + (h / p.kv_group) * p.k_stride[1];
      const T* v = (const T*)p.v + row * p.v_stride[0] + (h / p.kv_group) * p.v_stride[1];
      __syncthreads();
      for (int i = threadIdx.x; i < p.dk; i += 256) qs[i] = (float)q[i], ks[i] = (float)k[i];
      __syncthreads();
      for (int j0 = 0; j0 < p.dv; j0 += 64) {
        const int j = j0 + (threadIdx.x & 63);
        float acc = 0.f;
        if (j < p.dv) {
          const float vj = (float)v[j];
          for (int i = threadIdx.x >> 6; i < p.dk; i += 4) {
            const float old = s[i * p.dv + j];
            const float now = (keep == 0.f ? 0.f : keep * old) + ks[i] * vj;
            s[i * p.dv + j] = now;
            acc += qs[i] * now;
          }
        }
        __syncthreads();
        part[threadIdx.x] = acc;
        __syncthreads();
        if (threadIdx.x < 64 && j < p.dv)
          ((T*)p.out)[row * p.out_stride[0] + h * p.out_stride[1] + j] =
              (T)(p.scale * (part[threadIdx.x] + part[threadIdx.x + 64] + part[threadIdx.x + 128] + part[threadIdx.x + 192]));
      }
      __syncthreads();
      if (!repeats) break;
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

template <class T> __global__ __launch_bounds__(256) void sum_heads(const float* src, int64_t total, int32_t group, int32_t dim, T* out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // over [n][heads_out][dim]
  if (i >= total) return;
  const int64_t head = i / dim, d = i % dim;
  float s = 0.f;
  for (int g = 0; g < group; ++g) s += src[(head * group + g) * dim + d];
  out[i] = (T)s;
}

}  // namespace epm
