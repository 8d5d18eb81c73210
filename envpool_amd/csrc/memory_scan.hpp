// memory_scan.hpp - the chunked form of the memory on matrix cores.
//
// A workgroup of four waves owns one state (row, head) and walks along time in chunks of 32 or 64 steps. Inside
// a chunk, with D[t, s] = decay^|t-s| where s reaches t (no episode starts between them), else 0:
//   P = (Q K^T) * D                       scores, steps x steps
//   O = w_in[t] * (Q S) + P V             S: the state the chunk starts from
//   S = carry * S + (K * w_up[s])^T V
// Everything is computed transposed (scores as [s, t], outputs as [v, t]): the accumulators of one product are
// then laid out as an operand of the next up to a permutation of the summed index, which is applied to the
// other operand as well. So the state never leaves its registers (32 bits), scores cross LDS once because each wave
// computes 16 of the query columns and needs all of them for its quarter of the value columns, and an output row is
// written 4 values a lane.
// What 32-bit values become as operands of 16-bit products (every sum is kept in 32 bits):
//   weighted values in K^T V   three pieces (bf16) or two scaled ones (f16): the state keeps what 32 bits keep (f16: of terms
//                              below 2^-14, where the type's own steps stop shrinking, 2^-36 each)
//   the state in Q S           two pieces: 16 bits of it in bf16, 22 in f16
//   scores in P V              two pieces, the same
// so that an output is off by 2^-16 (2^-22) of its terms before it is rounded to its type once. (With the scores in one
// piece that rounding was one of two of a size: the error of a bf16 result grew from 0.00166 to 0.0020 .. 0.0022.)
// Time backwards (for gradients) is the same chunk with the triangle and the weights mirrored.
#pragma once
#include "memory_kernels.hpp"

namespace epm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
// Steps per chunk. In 32 bits the matrix cores are the bound and half the chunk halves the work inside it (and lets
// two workgroups share a CU); in 16 bits memory is, and the longer chunk moves the state less often.
template <class T> struct ChunkOf {
  static constexpr int value = sizeof(T) == 4 ? 32 : 64;
};

template <class T> struct Mma;

template <class T, class V8, class V4> struct Mma16 {
  using frag = V8;
  static constexpr int K = 32;  // summed index per fragment: lane group g = lane / 16 holds 8g .. 8g+7
  static __device__ frag row(const T* tile, int stride, int r0, int k0, int lane) {
    return *(const V8*)(tile + (r0 + (lane & 15)) * stride + k0 + 8 * (lane >> 4));
  }
  // the order that a pair of accumulators has: 4g .. 4g+3, then 16 + 4g .. 16 + 4g+3
  static __device__ frag row_as_acc(const T* tile, int stride, int r0, int k0, int lane) {
    const T* p = tile + (r0 + (lane & 15)) * stride + k0 + 4 * (lane >> 4);
    const V4 a = *(const V4*)p, b = *(const V4*)(p + 16);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // column c0 + lane % 16 of rows k0 + 8g .. k0 + 8g + 7: the transposing LDS read takes 4 rows x 16 columns
  // per 16 lanes, lane i addressing 4 values of row i / 4
  static __device__ frag col(const T* tile, int stride, int k0, int c0, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const T* p = tile + (k0 + 8 * g + (i >> 2)) * stride + c0 + 4 * (i & 3);
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4* lp;
    union { s4 s[2]; V8 v; } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * stride));
    return u.v;
  }
  // the value of element e (0 .. 7) from a pair of accumulators, in row_as_acc's order
  static __device__ float of(f32x4 a, f32x4 b, int e) { return e < 4 ? a[e] : b[e - 4]; }
  static __device__ void put4(T* p, f32x4 a) {
    V4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (T)a[r];
    *(V4*)p = v;
  }
  // the first pieces of four values to p, the second ones returned
  static __device__ uint2 put4_first(T* p, f32x4 a) {
    V4 v, w;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x = a[r];
      asm volatile("" : "+v"(x));  // (rounded once, from 32 bits: see Mma<f16>::pieces)
      v[r] = (T)x;
      w[r] = (T)(x - (float)v[r]);
    }
    *(V4*)p = v;
    return __builtin_bit_cast(uint2, w);
  }
};
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
// 32-bit values as operands of 16-bit products. Rounded once (a score next to its value) they cost half a step of
// the type per term; where a result is kept in 32 bits they go in as several pieces whose sum is the value.
// bf16: the pieces are plain remainders, three of them hold 24 bits, and add up in one accumulator. f16: 11 bits a
// piece and a narrow range, so the second piece is scaled by 2^11 and has an accumulator of its own, and what may
// be large or small as a whole is brought to the middle of the range first (kNarrow).
template <> struct Mma<bf16> : Mma16<bf16, bf16x8, bf16x4> {
  static constexpr uint32_t kInf = 0x7f80;
  static constexpr bool kNarrow = false;
  static __device__ f32x4 mul(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  // two values a conversion, and back by shift and mask
  template <int N> static __device__ void pieces(const float (&v)[8], frag (&out)[N]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
    union { uint32_t w[4]; frag f; } u[N];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f32x2 x = {v[2 * e], v[2 * e + 1]};
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
        u[c].w[e] = w;
        x[0] -= __builtin_bit_cast(float, w << 16);
        x[1] -= __builtin_bit_cast(float, w & 0xffff0000u);
      }
    }
#pragma unroll
    for (int c = 0; c < N; ++c) out[c] = u[c].f;
  }
};
template <> struct Mma<f16> : Mma16<f16, f16x8, f16x4> {
  static constexpr uint32_t kInf = 0x7c00;
  static constexpr bool kNarrow = true;
  static __device__ f32x4 mul(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  template <int N> static __device__ void pieces(const float (&v)[8], frag (&out)[N], float step = 1.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = v[e];
      // (opaque: where x is a product the compiler rounds it to 16 bits at once in one place and by way of 32 in the
      // other, and at a tie the remainder is then that of a neighbouring piece)
      asm volatile("" : "+v"(x));
#pragma unroll
      for (int c = 0; c < N; ++c) {
        out[c][e] = (f16)x;
        x = (x - (float)out[c][e]) * step;
      }
    }
  }
};
// the power of two that brings a largest magnitude of `top` to 2^13 .. 2^14 (1 for 0 and for what is not finite; not
// beyond 2^40 or below 2^-60, so that two of them against each other stay in the range of 32 bits: what is that
// small is 0 in a float16 result, what is that large infinite)
__device__ inline float to_middle(float top) {
  const int e = __builtin_amdgcn_frexp_expf(top);
  return top > 0.f && top < INFINITY ? __builtin_amdgcn_ldexpf(1.f, max(-60, min(40, 14 - e))) : 1.f;
}
template <> struct Mma<float> {
  using frag = f32x4;
  static constexpr int K = 16;  // four products of 4: lane group g holds 4g + r in step r
  static constexpr uint32_t kInf = 0x7f800000u;
  static constexpr bool kNarrow = false;
  static __device__ frag row(const float* tile, int stride, int r0, int k0, int lane) {
    return *(const f32x4*)(tile + (r0 + (lane & 15)) * stride + k0 + 4 * (lane >> 4));
  }
  static __device__ frag row_as_acc(const float* tile, int stride, int r0, int k0, int lane) { return row(tile, stride, r0, k0, lane); }
  static __device__ frag col(const float* tile, int stride, int k0, int c0, int lane) {
    const float* p = tile + (k0 + 4 * (lane >> 4)) * stride + c0 + (lane & 15);
    return frag{p[0], p[stride], p[2 * stride], p[3 * stride]};
  }
  static __device__ void put4(float* p, f32x4 a) { *(f32x4*)p = a; }
  static __device__ f32x4 mul(frag a, frag b, f32x4 c) {
#pragma unroll
    for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
    return c;
  }
};

// Keeps the compiler from moving a later phase's LDS reads up here: it would need registers for all of them, and
// the waves that those registers cost hide more latency than the early reads.
__device__ inline void keep_order() { __builtin_amdgcn_sched_barrier(0); }

// After products that a wave may have skipped, or whose results it may not use, before their registers are touched: the
// compiler counts a matrix instruction's wait states along the straight path, and has been seen to come up short
// where the skipping path joins it from elsewhere. Sixteen are more than any of them needs.
template <bool kSkips> __device__ inline void settle() {
  if constexpr (kSkips) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// how a launch's states come and go
struct Parts {
  int64_t seg_len;     // steps per part of the time axis (whole chunks), blockIdx.y counts parts in time
  int32_t n_seg;
  f32x4* ws_state;     // [row * heads][n_seg][DK * DV / 4] in accumulator order: what a part starts from (read), or
  float* ws_carry;     // its own contribution and how far it lets the state before it through, -1: not at all (written)
  int32_t state_only;  // the first of two passes over split time: contributions only
  int32_t state_vec;   // state_in's rows are 16-byte pieces when its key stride is 1
};

template <class T, int DK, int DV> struct ScanTile {
  static constexpr int kChunk = ChunkOf<T>::value;
  static constexpr int kVec = 16 / sizeof(T);                // values of one 16-byte load
  // LDS row strides. 16 bytes of padding let 16 lanes read 16 bytes of a row each without a bank twice; the
  // transposing reads take 32 bytes of 4 rows, which 32 bytes of padding keep apart
  static constexpr int SQ = DK + kVec, SK = DK + 32 / (int)sizeof(T), SV = DV + 32 / (int)sizeof(T);
  static constexpr int SP = kChunk + kVec;
  static constexpr int kQ = kChunk * DK / kVec / 256;        // 16-byte loads per thread and tile
  static constexpr int kV = kChunk * DV / kVec / 256;
  static constexpr size_t kLds = (size_t)kChunk * (SQ + SK + SV + SP) * sizeof(T) + 4 * kChunk * sizeof(float);
  // workgroups (one wave per SIMD each) that LDS lets a CU hold, three at most in 32 bits (whose operands take twice
  // the registers): the registers are kept to as many (value-by-value addressing needs more of them: half as many)
  static constexpr int kFit = (int)(163840 / kLds), kPerCu = sizeof(T) == 4 && kFit > 3 ? 3 : kFit;
  static constexpr int kWaves(bool aligned) { return aligned || kPerCu == 1 ? kPerCu : kPerCu / 2; }
};

// largest magnitude bits seen: of each 16-bit half, or of the word
template <class T> __device__ inline uint32_t top_bits(uint32_t top, uint32_t x) {
  if constexpr (sizeof(T) == 2) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    union { uint32_t u; u16x2 v; } a, b;
    a.u = top, b.u = x & 0x7fff7fffu;
    a.v = __builtin_elementwise_max(a.v, b.v);
    return a.u;
  } else {
    const uint32_t y = x & 0x7fffffffu;
    return top > y ? top : y;
  }
}
// `odd` plus 0 times every value of x: 0, or NaN where one is not finite. One instruction a word, whose products are exact
__device__ inline float plus_nothing(float odd, uint32_t x, bf16) {
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), bf16x2{(bf16)0.f, (bf16)0.f}, odd, false);
}
__device__ inline float plus_nothing(float odd, uint32_t x, f16) {
  typedef f16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), f16x2{(f16)0.f, (f16)0.f}, odd, false);
}
__device__ inline float plus_nothing(float odd, uint32_t x, float) { return __builtin_fmaf(__builtin_bit_cast(float, x), 0.f, odd); }
template <class T> __device__ inline bool not_finite(uint32_t top) {
  if constexpr (sizeof(T) == 2) return (top & 0xffffu) >= Mma<T>::kInf || (top >> 16) >= Mma<T>::kInf;
  else return top >= Mma<T>::kInf;
}

// Buffer addressing: a 64-bit base that the whole workgroup shares plus a 32-bit byte offset per lane; loads past
// `bytes` give 0 and stores there are dropped, so that ragged ends cost no instructions. kOutside plus anything below
// 2^31 is past every buffer.
constexpr uint32_t kOutside = 0x80000000u;
__device__ inline __amdgpu_buffer_rsrc_t buffer(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// What the workgroup knows about the chunk it is at.
struct Now {
  uint64_t starts;  // bit t: step t starts an episode
  int64_t start;    // its first step
  int n;            // its steps
  float l2;         // log2 of the decay
  float lambda;
  int ln, wave;     // lane and wave
  float *w_up, *w_in, *p_top;
};

// The pieces of a walk in one direction. kAligned: every operand in 16-byte pieces through buffers (offsets below
// 2^31, rows that do not overlap); otherwise value by value.
template <class T, int DK, int DV, bool kAligned, bool rev> struct Walk {
  using M = Mma<T>;
  using Tile = ScanTile<T, DK, DV>;
  using frag = typename M::frag;
  static constexpr int kChunk = Tile::kChunk, kBlocks = kChunk / 16;
  static constexpr int K = M::K, kVec = Tile::kVec, SP = Tile::SP;
  static constexpr int ND = DK / 16, NV = DV / 64;  // state tiles of a wave: all keys, 16 of every 64 value columns
  // tiles that the operands' sizes reach (in 32 bits the matrix cores are the bound, so padding is not multiplied)
  static constexpr bool kTrim = sizeof(T) == 4 && kAligned;
  // (opaque, or the compiler makes a copy of everything that follows for every number of tiles)
  static __device__ int tiles(int dim, int unit, int all) {
    if constexpr (!kTrim) return all;
    int n = (dim + unit - 1) / unit;
    asm volatile("" : "+s"(n));
    return n;
  }
  static __device__ int nk(const Scan& p) { return tiles(p.dk, K, DK / K); }
  static __device__ int nd(const Scan& p) { return tiles(p.dk, 16, ND); }
  using State = f32x4[ND][NV];

  static __device__ void load_tile(uint4* r, int count, const T* base, int64_t step_stride, int width, int padded, int64_t start, int n) {
    const int per_row = padded / kVec;
    if constexpr (kAligned) {
      const auto b = buffer(base + start * step_stride, ((n - 1) * step_stride + width) * (int64_t)sizeof(T));
      const int t = threadIdx.x / per_row, c = (threadIdx.x % per_row) * kVec;
      const uint32_t stride = (uint32_t)step_stride * (uint32_t)sizeof(T);
      const uint32_t at = c < width ? t * stride + c * (uint32_t)sizeof(T) : kOutside;
#pragma unroll
      for (int i = 0; i < count; ++i) {
        const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(b, at + i * (256 / per_row) * stride, 0, 0);
        r[i] = make_uint4(x.x, x.y, x.z, x.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < count; ++i) {
        const int at = i * 256 + threadIdx.x;
        const int t = at / per_row, c = (at % per_row) * kVec;
        union { uint4 u; T e[kVec]; } x;
        x.u = make_uint4(0, 0, 0, 0);
        if (t < n && c < width) {
          const T* a = base + (start + t) * step_stride + c;
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (c + e < width) x.e[e] = a[e];
        }
        r[i] = x.u;
      }
    }
  }
  static __device__ void put_tile(const uint4* r, int count, T* tile, int padded, int stride) {
    const int per_row = padded / kVec;
    T* to = tile + (threadIdx.x / per_row) * stride + (threadIdx.x % per_row) * kVec;
#pragma unroll
    for (int i = 0; i < count; ++i) *(uint4*)(to + i * (256 / per_row) * stride) = r[i];
  }
  // marks the steps of a chunk (bit t of the two words) whose keys or values are not finite; nearly always none
  static __device__ void mark_sick(const uint4* k, int count_k, const uint4* v, int count_v, uint32_t* sick) {
    float odd[2] = {0.f, 0.f};
    const auto look = [&](const uint4* r, int count) {
#pragma unroll
      for (int i = 0; i < count; ++i) {
        odd[0] = plus_nothing(odd[0], r[i].x, T{});
        odd[1] = plus_nothing(odd[1], r[i].y, T{});
        odd[0] = plus_nothing(odd[0], r[i].z, T{});
        odd[1] = plus_nothing(odd[1], r[i].w, T{});
      }
    };
    look(k, count_k);
    look(v, count_v);
    if (odd[0] + odd[1] == 0.f) return;
    const auto mark = [&](const uint4* r, int count, int padded) {
      const int per_row = padded / kVec;
#pragma unroll
      for (int i = 0; i < count; ++i) {
        const int t = threadIdx.x / per_row + i * (256 / per_row);
        const uint32_t top = top_bits<T>(top_bits<T>(top_bits<T>(top_bits<T>(0, r[i].x), r[i].y), r[i].z), r[i].w);
        if (not_finite<T>(top)) atomicOr(&sick[t >> 5], 1u << (t & 31));
      }
    };
    mark(k, count_k, DK);
    mark(v, count_v, DV);
  }
  static __device__ uint64_t marked(const uint32_t* sick) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(sick[0]), hi = __builtin_amdgcn_readfirstlane(sick[1]);
    return (uint64_t)hi << 32 | lo;
  }

  static __device__ void load_state(const Scan& p, bool state_vec, int64_t row, int h, int lane, int wave, State& s) {
    const int v0 = 16 * wave, g = lane >> 4, l16 = lane & 15;
    const float* base = p.state_in + row * p.in_stride[0] + h * p.in_stride[1];
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = v0 + 64 * j + l16, d = 16 * i + 4 * g;
        if constexpr (kAligned) {
          const auto b = buffer(base, 0x7fffffff);
          const uint32_t sd = (uint32_t)p.in_stride[2] * 4u, sv = (uint32_t)p.in_stride[3] * 4u;
          const uint32_t at = v < p.dv && d < p.dk ? d * sd + v * sv : kOutside;
          if (sd == 4 && state_vec) {
            union { u32x4 u; f32x4 f; } x;
            x.u = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0);
            s[i][j] = x.f;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][j][r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, at + r * sd, 0, 0));
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (v < p.dv && d + r < p.dk) s[i][j][r] = base[(d + r) * p.in_stride[2] + v * p.in_stride[3]];
        }
      }
  }
  static __device__ void store_state(const Scan& p, int64_t row, int h, int lane, int wave, const State& s) {
    const int v0 = 16 * wave, g = lane >> 4, l16 = lane & 15;
    float* base = p.state_out + row * p.outs_stride[0] + h * p.outs_stride[1];
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = v0 + 64 * j + l16, d = 16 * i + 4 * g;
        if constexpr (kAligned) {
          const auto b = buffer(base, 0x7fffffff);
          const uint32_t sd = (uint32_t)p.outs_stride[2] * 4u, sv = (uint32_t)p.outs_stride[3] * 4u;
          const uint32_t at = v < p.dv && d < p.dk ? d * sd + v * sv : kOutside;
#pragma unroll
          for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, (float)s[i][j][r]), b, at + r * sd, 0, 0);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (v < p.dv && d + r < p.dk) base[(d + r) * p.outs_stride[2] + v * p.outs_stride[3]] = s[i][j][r];
        }
      }
  }

  // the weights of the chunk's steps: in the state that leaves it, and of the state that enters it in their outputs (NaN:
  // it does not reach them, which a weight that is 0 for its smallness must not be taken for where the state is infinite)
  static __device__ void weights(const Scan& p, const Now& c) {
    if (threadIdx.x < 2 * kChunk) {
      const int t = threadIdx.x % kChunk;
      const uint64_t until = c.starts & ((2ull << t) - 1), later = t < 63 ? c.starts >> (t + 1) : 0;
      const float from_0 = __builtin_amdgcn_exp2f(c.l2 * (t + 1)), to_end = __builtin_amdgcn_exp2f(c.l2 * (c.n - 1 - t));
      if (threadIdx.x < kChunk) c.w_up[t] = t < c.n && (rev ? until : later) == 0 ? (rev ? from_0 : to_end) * (M::kNarrow ? 1.f : p.inc_scale) : 0.f;
      else c.w_in[t] = t < c.n && (rev ? later : until) == 0 ? (rev ? to_end : from_0) * p.out_scale : __builtin_nanf("");
    }
  }

  // scores of 16 query steps per wave, or per two waves that take every other tile of them; their second pieces stay in
  // registers (16-bit types) until put_seconds
  using Seconds = uint2[kBlocks];
  static __device__ void scores(const Scan& p, const Now& c, const T* qs, int SQ, const T* ks, int SK, T* ps, Seconds& second) {
    const int wave = c.wave, ln = c.ln, g = ln >> 4, l16 = ln & 15, nk = Walk::nk(p);
    const uint64_t starts = c.starts;
    const float l2 = c.l2, lambda = c.lambda;
    float* p_top = c.p_top;
    constexpr int kShare = 4 / kBlocks;
    static_assert(kShare == 1 || !M::kNarrow, "a step's largest score is found within one wave");
    const int strip = wave % kBlocks, t = 16 * strip + l16;
    int lo, hi;  // the steps that reach step t
    if (rev) {
      const uint64_t later = t < 63 ? starts >> (t + 1) : 0;
      lo = t;
      hi = later ? t + __ffsll((unsigned long long)later) - 1 : kChunk - 1;
    } else {
      const uint64_t until = starts & ((2ull << t) - 1);
      lo = until ? 63 - __clzll(until) : 0;
      hi = t;
    }
    frag q[DK / K];
#pragma unroll
    for (int k = 0; k < DK / K; ++k) q[k] = M::row(qs, SQ, 16 * strip, k * K, ln);
    const int i0 = first_tile(strip), i1 = last_tile(strip);
    const float scale = p.inc_scale * p.out_scale;
    f32x4 score[kBlocks];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      if (kShare > 1 && i % kShare != wave / kBlocks) continue;
      f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
      if (rev ? i >= strip : i <= strip) {
#pragma unroll
        for (int k = 0; k < DK / K; ++k)
          if (k < nk) a = M::mul(M::row(ks, SK, 16 * i, k * K, ln), q[k], a);
        settle<kTrim>();
        const int u = 16 * i + 4 * g;
        f32x4 w;
        if (i == strip) {
#pragma unroll
          for (int r = 0; r < 4; ++r) w[r] = __builtin_amdgcn_exp2f(l2 * (float)(rev ? u + r - t : t - u - r)) * scale;
        } else if (rev) {  // the nearest of the four, then one decay each
          w[0] = __builtin_amdgcn_exp2f(l2 * (float)(u - t)) * scale;
          w[1] = w[0] * lambda, w[2] = w[1] * lambda, w[3] = w[2] * lambda;
        } else {
          w[3] = __builtin_amdgcn_exp2f(l2 * (float)(t - u - 3)) * scale;
          w[2] = w[3] * lambda, w[1] = w[2] * lambda, w[0] = w[1] * lambda;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) a[r] = u + r >= lo && u + r <= hi ? a[r] * w[r] : 0.f;
      }
      if constexpr (M::kNarrow) {
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(a[r]));
        score[i] = a;
      } else if (i >= i0 && i < i1) {
        if constexpr (sizeof(T) == 2) second[i] = M::put4_first(ps + t * SP + 16 * i + 4 * g, a);
        else M::put4(ps + t * SP + 16 * i + 4 * g, a);
      }
    }
    if constexpr (M::kNarrow) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float f = to_middle(top);
      if (g == 0) p_top[t] = f;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
        if (i >= i0 && i < i1) second[i] = M::put4_first(ps + t * SP + 16 * i + 4 * g, score[i] * f);
    }
  }
  // the tiles of a strip of scores that P V reads: all of whole fragments, so that what lies across the diagonal is 0
  static __device__ int first_tile(int strip) { return rev ? (16 * strip) / K * K / 16 : 0; }
  static __device__ int last_tile(int strip) { return rev ? kChunk / 16 : ((16 * strip) / K + 1) * K / 16; }
  static __device__ void put_seconds(const Now& c, const Seconds& second, T* ps2) {
    if constexpr (sizeof(T) == 2) {
      const int strip = c.wave % kBlocks, i0 = first_tile(strip), i1 = last_tile(strip);
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
        if (i >= i0 && i < i1) *(uint2*)(ps2 + (16 * strip + (c.ln & 15)) * SP + 16 * i + 4 * (c.ln >> 4)) = second[i];
    }
  }

  // outputs: what the entering state gives (not weighted yet; returns what the state was multiplied by) ..
  using Outs = f32x4[kBlocks][NV];
  static __device__ float from_state(const Scan& p, const Now& c, const State& s, const T* qs, int SQ, Outs& a) {
    const int ln = c.ln, v0 = 16 * c.wave, nk = Walk::nk(p);
    const auto there = [&](int j) { return !kTrim || j == 0 || v0 + 64 * j < p.dv; };  // (the same for the whole wave)
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int j = 0; j < NV; ++j) a[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float s_scale = 1.f;
    if constexpr (M::kNarrow) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(s[i][j][r]));
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
      s_scale = to_middle(top);
    }
#pragma unroll
    for (int k = 0; k < DK / K; ++k) {
      if (k >= nk) continue;
      // the state rounded, and what that left out
      frag sf[NV][2];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if constexpr (sizeof(T) == 2) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = M::of(s[2 * k][j], s[2 * k + 1][j], e) * s_scale;
          M::pieces(x, sf[j]);
        } else {
          sf[j][0] = s[k][j];
        }
      }
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const frag qf = M::row_as_acc(qs, SQ, 16 * b, k * K, ln);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!there(j)) continue;
          a[b][j] = M::mul(sf[j][0], qf, a[b][j]);
          if constexpr (sizeof(T) == 2) a[b][j] = M::mul(sf[j][1], qf, a[b][j]);
        }
      }
      keep_order();
    }
    settle<kTrim>();
    return s_scale;
  }
  // .. then the chunk's own steps
  static __device__ void outputs(const Scan& p, const Now& c, int64_t row, int h, Outs& a, float s_scale, const T* vs, int SV, const T* ps, const T* ps2) {
    const int wave = c.wave, ln = c.ln, g = ln >> 4, l16 = ln & 15, v0 = 16 * wave, n_now = c.n;
    const float *w_in = c.w_in, *p_top = c.p_top;
    const uint32_t out_size = p.out_f32 ? 4u : (uint32_t)sizeof(T);
    const T* out_row = (const T*)((const char*)p.out + (c.start * p.out_stride[0] + row * p.out_stride[1] + h * p.out_stride[2]) * (int64_t)out_size);
    const auto there = [&](int j) { return !kTrim || j == 0 || v0 + 64 * j < p.dv; };
    frag vf[NV][kChunk / K];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < kChunk / K; ++k) vf[j][k] = M::col(vs, SV, k * K, v0 + 64 * j, ln);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int t = 16 * b + l16;
      const float f = M::kNarrow ? p_top[t] : 1.f;
      const float w = w_in[t], ws_ = w * f / s_scale;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) a[b][j][r] = w == w ? a[b][j][r] * ws_ : 0.f;
#pragma unroll
      for (int k = 0; k < kChunk / K; ++k)
        if (rev ? (k + 1) * K > 16 * b : k * K <= 16 * b) {
          const frag pf = M::row(ps, SP, 16 * b, k * K, ln);
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (there(j)) a[b][j] = M::mul(vf[j][k], pf, a[b][j]);
          if constexpr (sizeof(T) == 2) {
            const frag pf2 = M::row(ps2, SP, 16 * b, k * K, ln);
#pragma unroll
            for (int j = 0; j < NV; ++j) a[b][j] = M::mul(vf[j][k], pf2, a[b][j]);
          }
        }
      settle<true>();  // (how results are stored is a branch)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        f32x4 x = a[b][j];
        if constexpr (M::kNarrow) x *= 1.f / f;
        const int v = v0 + 64 * j + 4 * g;
        if constexpr (kAligned) {
          const auto o = buffer(out_row, p.out ? ((n_now - 1) * p.out_stride[0] + p.dv) * (int64_t)out_size : 0);
          const uint32_t at = v < p.dv ? (uint32_t)(t * (uint32_t)p.out_stride[0] + v) * out_size : kOutside;
          if (sizeof(T) == 4 || p.out_f32) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), o, at, 0, 0);
          } else if constexpr (sizeof(T) == 2) {
            alignas(8) T y[4];
            M::put4(y, x);
            __builtin_amdgcn_raw_buffer_store_b64(*(const u32x2*)y, o, at, 0, 0);
          }
        } else if (t < n_now && p.out) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (v + r < p.dv) {
              if (p.out_f32) ((float*)out_row)[t * p.out_stride[0] + v + r] = x[r];
              else ((T*)out_row)[t * p.out_stride[0] + v + r] = (T)x[r];
            }
        }
      }
      keep_order();
    }
  }

  // the state that leaves the chunk: keys as rows, weighted values as columns
  static __device__ void update(const Scan& p, const Now& c, State& s, const T* ks, int SK, const T* vs, int SV) {
    const int wave = c.wave, ln = c.ln, g = ln >> 4, v0 = 16 * wave, nd = Walk::nd(p);
    const uint64_t starts = c.starts;
    const float* w_up = c.w_up;
    const float carry = __builtin_amdgcn_exp2f(c.l2 * c.n);
    const auto there = [&](int j) { return !kTrim || j == 0 || v0 + 64 * j < p.dv; };
    if (starts) {  // nothing from before the chunk leaves it (and 0 * inf must not)
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int j = 0; j < NV; ++j) s[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    } else {
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int j = 0; j < NV; ++j) s[i][j] *= carry;
    }
    if (!(rev && (starts & 1))) {  // (else nothing of the chunk itself leaves it)
#pragma unroll
      for (int k = 0; k < kChunk / K; ++k) {
        const float* w = w_up + k * K + (K / 4) * g;
        constexpr int kPieces = sizeof(T) == 4 ? 1 : M::kNarrow ? 2 : 3;
        frag vw[NV][kPieces];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const frag v = M::col(vs, SV, k * K, v0 + 64 * j, ln);
          float x[K / 4];
#pragma unroll
          for (int e = 0; e < K / 4; ++e) x[e] = (float)v[e] * w[e];
          if constexpr (M::kNarrow) M::pieces(x, vw[j], 2048.f);
          else if constexpr (sizeof(T) == 2) M::pieces(x, vw[j]);
          else vw[j][0] = frag{x[0], x[1], x[2], x[3]};
        }
        keep_order();
#pragma unroll
        for (int i = 0; i < ND; ++i)
          if (i < nd) {
            const frag kf = M::col(ks, SK, k * K, 16 * i, ln);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
              if (!there(j)) continue;
              if constexpr (M::kNarrow) {
                f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
                x = M::mul(kf, vw[j][0], x);
                y = M::mul(kf, vw[j][1], y);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][j][r] = fmaf(fmaf(y[r], 1.f / 2048, x[r]), p.inc_scale, s[i][j][r]);
              } else {
#pragma unroll
                for (int c = 0; c < kPieces; ++c) s[i][j] = M::mul(kf, vw[j][c], s[i][j]);
              }
            }
          }
      }
    }
    settle<true>();  // (a whole update may have been skipped)
  }
};

// (a decay of 0 as a very small one, whose power 0 is still 1; NaN stays)
__device__ inline float log2_of_decay(float log_decay) {
  const float x = log_decay * 1.44269504088896f;
  return x < -1e30f ? -1e30f : x;
}

// Where a chunk that holds something not finite ends. The products inside a chunk run over all of its steps, those that
// do not reach a result with the weight 0, and 0 * inf is NaN. So a chunk with a sick step ends where an episode does, and
// at the sick step: forward in time it starts one (and reaches all later steps, as it should), back in time it ends one.
template <bool rev> __device__ inline void cut_chunk(uint64_t starts, uint64_t sick, int64_t& start, int& n) {
  int from = 0, to = n;
  if (rev) {
    const uint64_t before_last = sick & ((1ull << (n - 1)) - 1);
    from = max(starts ? 63 - __clzll(starts) : 0, before_last ? 64 - __clzll(before_last) : 0);
  } else {
    const uint64_t ends = (starts | sick) & ~1ull;
    if (ends) to = __ffsll((unsigned long long)ends) - 1;
  }
  start += from;
  n = to - from;
}

// One walk. 128 steps of 4096 states of 64 x 64 in bf16, states in and out: 108 us = 3.7 TB/s of the 403 MB it moves,
// 76 % of a large copy; vector and matrix instructions share the rest (half of the cycles issue vector instructions).
// 32768 steps of 16 states of 128 x 128 in 32 parts: 187 us for 537 MB and 109 Gflop with the pieces (matrix floor 90
// us). In f32 two chunks of 32 steps of 80 x 112 take 28 us in 390 workgroups: a CU's two workgroups need 11 us on the
// matrix cores, the rest is the state's way in and out and loads that nothing hides.
template <class T, int DK, int DV, bool kAligned, bool rev>
__global__ __launch_bounds__(256, (ScanTile<T, DK, DV>::kWaves(kAligned))) void scan_chunks(Scan p, Parts parts) {
  using W = Walk<T, DK, DV, kAligned, rev>;
  using Tile = ScanTile<T, DK, DV>;
  constexpr int kChunk = Tile::kChunk, SQ = Tile::SQ, SK = Tile::SK, SV = Tile::SV, ND = W::ND, NV = W::NV;
  extern __shared__ __align__(16) char lds[];
  T* qs = (T*)lds;
  T* ks = qs + kChunk * SQ;
  T* vs = ks + kChunk * SK;
  T* ps = vs + kChunk * SV;
  Now c;
  c.w_up = (float*)(ps + kChunk * Tile::SP);
  c.w_in = c.w_up + kChunk;
  c.p_top = c.w_in + kChunk;             // kNarrow: what a step's scores were multiplied by
  uint32_t* sick = (uint32_t*)(c.p_top + kChunk);  // steps of this chunk whose key or value is not finite, two words of bits

  const int64_t rh = blockIdx.x;
  const int64_t row = rh / p.heads;
  const int h = (int)(rh % p.heads);
  // (of the contributions only those are needed that a later part starts from)
  const int seg = blockIdx.y + (parts.state_only && rev ? 1 : 0);
  const int lane = threadIdx.x & 63;
  c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float log2_decay = log2_of_decay(p.log_decay[h]);
  c.lambda = __builtin_amdgcn_exp2f(log2_decay);

  const T* gq = (const T*)p.q + row * p.q_stride[1] + (h / p.q_group) * p.q_stride[2];
  const T* gk = (const T*)p.k + row * p.k_stride[1] + (h / p.k_group) * p.k_stride[2];
  const T* gv = (const T*)p.v + row * p.v_stride[1] + (h / p.v_group) * p.v_stride[2];
  const uint8_t* gf = p.fresh ? p.fresh + row * p.fresh_stride[1] : nullptr;
  const int64_t seg0 = seg * parts.seg_len;
  const int64_t seg1 = seg0 + parts.seg_len < p.steps ? seg0 + parts.seg_len : p.steps;

  // ---- a chunk's tiles, on their way from memory
  uint4 rq[Tile::kQ], rk[Tile::kQ], rv[Tile::kV];
  uint8_t rf = 0;
  const auto load = [&](int64_t start, int n) {
    W::load_tile(rk, Tile::kQ, gk, p.k_stride[0], p.dk, DK, start, n);
    W::load_tile(rv, Tile::kV, gv, p.v_stride[0], p.dv, DV, start, n);
    if (!parts.state_only) W::load_tile(rq, Tile::kQ, gq, p.q_stride[0], p.dk, DK, start, n);
    rf = gf && lane < n ? gf[(start + lane) * p.fresh_stride[0]] : 0;
  };
  const auto put = [&]() {
    if (!parts.state_only) W::put_tile(rq, Tile::kQ, qs, DK, SQ);
    W::put_tile(rk, Tile::kQ, ks, DK, SK);
    W::put_tile(rv, Tile::kV, vs, DV, SV);
  };

  int64_t start = rev ? seg1 - (seg1 - seg0 < kChunk ? seg1 - seg0 : kChunk) : seg0;
  int n = (int)(seg1 - seg0 < kChunk ? seg1 - seg0 : kChunk);
  if (threadIdx.x < 2) sick[threadIdx.x] = 0;
  if (n > 0) load(start, n);

  // ---- the state the part starts from
  typename W::State s;
  f32x4* ws = parts.ws_state ? parts.ws_state + (rh * parts.n_seg + seg) * (DK * DV / 4) : nullptr;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int j = 0; j < NV; ++j) s[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!parts.state_only && parts.n_seg > 1) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < NV; ++j) s[i][j] = ws[((i * NV + j) * 4 + c.wave) * 64 + lane];
  } else if (!parts.state_only && p.state_in) {
    W::load_state(p, parts.state_vec, row, h, lane, c.wave, s);
  }
  float through = 1.f;  // how far the part lets the state before it through, -1: not at all (an episode starts)

  while (n > 0) {
    // (opaque to the compiler here, or it would keep every step's powers of the decay, and every address, in
    // registers across the loop)
    c.l2 = log2_decay;
    c.ln = lane;
    asm volatile("" : "+v"(c.l2), "+v"(c.ln));
    __syncthreads();  // (the tiles of the chunk before have been read)
    put();
    c.starts = __ballot(rf != 0);
    W::mark_sick(rk, Tile::kQ, rv, Tile::kV, sick);
    __syncthreads();
    if (const uint64_t bad = W::marked(sick)) {
      __syncthreads();
      if (threadIdx.x < 2) sick[threadIdx.x] = 0;
      cut_chunk<rev>(c.starts, bad, start, n);
      load(start, n);
      put();
      c.starts = __ballot(rf != 0);
      __syncthreads();
    }
    // the next chunk's loads run under this one's products
    c.n = n;
    c.start = start;
    const int64_t left = rev ? start - seg0 : seg1 - (start + n);
    n = (int)(left < kChunk ? left : kChunk);
    start = rev ? start - n : start + c.n;
    if (n > 0) load(start, n);

    W::weights(p, c);
    through = c.starts || through < 0.f ? -1.f : through * __builtin_amdgcn_exp2f(c.l2 * c.n);
    if (!parts.state_only) {
      typename W::Outs a;
      typename W::Seconds second;
      // (two results that wait for each other: the smaller first, or where values outnumber keys the larger, which spills
      // fewer registers: 128 steps of 2048 states of 64 x 128, bf16 86 us against 91, f16 100 against 101)
      float s_scale = 1.f;
      if constexpr (DK < DV) s_scale = W::from_state(p, c, s, qs, SQ, a);
      W::scores(p, c, qs, SQ, ks, SK, ps, second);
      if constexpr (DK >= DV) s_scale = W::from_state(p, c, s, qs, SQ, a);
      __syncthreads();
      if constexpr (sizeof(T) == 2) {  // (the queries have been read: their place holds the scores' second pieces)
        W::put_seconds(c, second, qs);
        __syncthreads();
      }
      W::outputs(p, c, row, h, a, s_scale, vs, SV, ps, qs);
    } else {
      __syncthreads();
    }
    W::update(p, c, s, ks, SK, vs, SV);
  }

  // ---- the state the part ends with
  if (parts.state_only) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < NV; ++j) ws[((i * NV + j) * 4 + c.wave) * 64 + lane] = s[i][j];
    if (threadIdx.x == 0) parts.ws_carry[rh * parts.n_seg + seg] = through;
    return;
  }
  const bool last = rev ? seg == 0 : seg == parts.n_seg - 1;
  if (last && p.state_out) W::store_state(p, row, h, lane, c.wave, s);
}

// Two walks back in time over the same four tensors, for the gradients of keys and values (a: values, from keys,
// queries and the outputs' gradients; b: keys, from values, the outputs' gradients and queries): the tiles of a chunk
// are read once for both. 16-bit types, sizes up to 64, time not split. 128 steps of 4096 states in bf16: 175 us for the
// 604 MB that the two move (3.45 TB/s); three workgroups a CU (165 and 168 registers, 48 KB of LDS).
template <class T> struct PairTile {
  using Tile = ScanTile<T, 64, 64>;
  static constexpr size_t kLds = (size_t)Tile::kChunk * (2 * Tile::SQ + 2 * Tile::SK + Tile::SP) * sizeof(T) + 4 * Tile::kChunk * sizeof(float);
};
template <class T> __global__ __launch_bounds__(256, 3) void scan_pair(Scan a, Scan b, int state_vec_a, int state_vec_b) {
  using W = Walk<T, 64, 64, true, true>;
  using Tile = ScanTile<T, 64, 64>;
  constexpr int kChunk = Tile::kChunk, SQ = Tile::SQ, SK = Tile::SK, N = Tile::kQ;
  static_assert(Tile::SK == Tile::SV, "keys and values change places");
  extern __shared__ __align__(16) char lds[];
  T* kt = (T*)lds;             // a's queries: the keys
  T* vt = kt + kChunk * SQ;    // b's queries: the values
  T* qt = vt + kChunk * SQ;    // a's keys, b's values
  T* gt = qt + kChunk * SK;    // a's values, b's keys: the outputs' gradients
  T* ps = gt + kChunk * SK;
  Now c;
  c.w_up = (float*)(ps + kChunk * Tile::SP);
  c.w_in = c.w_up + kChunk;
  c.p_top = c.w_in + kChunk;
  uint32_t* sick = (uint32_t*)(c.p_top + kChunk);

  const int64_t row = blockIdx.x / a.heads;
  const int h = (int)(blockIdx.x % a.heads);
  const int lane = threadIdx.x & 63;
  c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float log2_decay = log2_of_decay(a.log_decay[h]);
  c.lambda = __builtin_amdgcn_exp2f(log2_decay);
  const T* gk = (const T*)a.q + row * a.q_stride[1] + (h / a.q_group) * a.q_stride[2];
  const T* gq = (const T*)a.k + row * a.k_stride[1] + (h / a.k_group) * a.k_stride[2];
  const T* gg = (const T*)a.v + row * a.v_stride[1] + (h / a.v_group) * a.v_stride[2];
  const T* gv = (const T*)b.q + row * b.q_stride[1] + (h / b.q_group) * b.q_stride[2];
  const uint8_t* gf = a.fresh ? a.fresh + row * a.fresh_stride[1] : nullptr;

  uint4 rk[N], rq[N], rg[N], rv[N];
  uint8_t rf = 0;
  const auto load = [&](int64_t start, int n) {
    W::load_tile(rq, N, gq, a.k_stride[0], a.dk, 64, start, n);
    W::load_tile(rg, N, gg, a.v_stride[0], a.dv, 64, start, n);
    W::load_tile(rk, N, gk, a.q_stride[0], a.dk, 64, start, n);
    W::load_tile(rv, N, gv, b.q_stride[0], a.dv, 64, start, n);
    rf = gf && lane < n ? gf[(start + lane) * a.fresh_stride[0]] : 0;
  };
  const auto put = [&]() {
    W::put_tile(rq, N, qt, 64, SK);
    W::put_tile(rg, N, gt, 64, SK);
    W::put_tile(rk, N, kt, 64, SQ);
    W::put_tile(rv, N, vt, 64, SQ);
  };
  int n = (int)(a.steps < kChunk ? a.steps : kChunk);
  int64_t start = a.steps - n;
  if (threadIdx.x < 2) sick[threadIdx.x] = 0;
  if (n > 0) load(start, n);
  typename W::State sa, sb;
#pragma unroll
  for (int i = 0; i < W::ND; ++i) sa[i][0] = sb[i][0] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (a.state_in) W::load_state(a, state_vec_a, row, h, lane, c.wave, sa);
  if (b.state_in) W::load_state(b, state_vec_b, row, h, lane, c.wave, sb);

  while (n > 0) {
    c.l2 = log2_decay;
    c.ln = lane;
    asm volatile("" : "+v"(c.l2), "+v"(c.ln));
    __syncthreads();
    put();
    c.starts = __ballot(rf != 0);
    W::mark_sick(rq, N, rg, N, sick);
    __syncthreads();
    if (const uint64_t bad = W::marked(sick)) {
      __syncthreads();
      if (threadIdx.x < 2) sick[threadIdx.x] = 0;
      cut_chunk<true>(c.starts, bad, start, n);
      load(start, n);
      put();
      c.starts = __ballot(rf != 0);
      __syncthreads();
    }
    c.n = n;
    c.start = start;
    n = (int)(start < kChunk ? start : kChunk);
    start -= n;
    if (n > 0) load(start, n);

    W::weights(a, c);
    typename W::Outs o;
    typename W::Seconds second;
    W::scores(a, c, kt, SQ, qt, SK, ps, second);
    float s_scale = W::from_state(a, c, sa, kt, SQ, o);
    __syncthreads();
    W::put_seconds(c, second, kt);  // (a's queries have been read, here and for b: their place is free)
    __syncthreads();
    W::outputs(a, c, row, h, o, s_scale, gt, SK, ps, kt);
    W::update(a, c, sa, qt, SK, gt, SK);
    __syncthreads();  // (the scores have been read)
    W::scores(b, c, vt, SQ, gt, SK, ps, second);
    W::put_seconds(c, second, kt);
    s_scale = W::from_state(b, c, sb, vt, SQ, o);
    __syncthreads();
    W::outputs(b, c, row, h, o, s_scale, qt, SK, ps, kt);
    W::update(b, c, sb, gt, SK, qt, SK);
  }
  if (a.state_out) W::store_state(a, row, h, lane, c.wave, sa);
}

// Turns the parts' own contributions into what each part starts from, in time's direction: one thread per 4
// values of a state. 16 states of 128 x 128 and 32 parts: 14 us for 67 MB (4.7 TB/s).
template <int DK, int DV> __global__ __launch_bounds__(256) void join_parts(Scan p, Parts parts) {
  const int64_t rh = blockIdx.x;
  const int at = blockIdx.y * 256 + threadIdx.x;  // in accumulator order
  const int lane = at & 63, wave = (at >> 6) & 3, tile = at >> 8;
  const int i = tile / (DV / 64), j = tile % (DV / 64);
  const int v = 64 * j + 16 * wave + (lane & 15), d = 16 * i + 4 * (lane >> 4);
  const int64_t row = rh / p.heads;
  const int h = (int)(rh % p.heads);
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
  if (p.state_in) {
    const float* a = p.state_in + row * p.in_stride[0] + h * p.in_stride[1] + v * p.in_stride[3];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (v < p.dv && d + r < p.dk) s[r] = a[(d + r) * p.in_stride[2]];
  }
  // (the parts' own states do not depend on each other: eight are under way at a time)
  f32x4* ws = parts.ws_state + rh * parts.n_seg * (DK * DV / 4) + at;
  constexpr int kAheadParts = 8;
  for (int n0 = 0; n0 < parts.n_seg; n0 += kAheadParts) {
    f32x4 own[kAheadParts];
    float carry[kAheadParts];
#pragma unroll
    for (int i = 0; i < kAheadParts; ++i) {
      const int n = n0 + i, seg = p.reverse ? parts.n_seg - 1 - n : n;
      if (n + 1 < parts.n_seg) {  // (nothing follows the last part)
        own[i] = ws[(int64_t)seg * (DK * DV / 4)];
        carry[i] = parts.ws_carry[rh * parts.n_seg + seg];
      }
    }
#pragma unroll
    for (int i = 0; i < kAheadParts; ++i) {
      const int n = n0 + i, seg = p.reverse ? parts.n_seg - 1 - n : n;
      if (n < parts.n_seg) ws[(int64_t)seg * (DK * DV / 4)] = s;
      if (n + 1 < parts.n_seg) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = (carry[i] < 0.f ? 0.f : s[r] * carry[i]) + own[i][r];
      }
    }
  }
}

// The launches of one call: `parts` says how time is split.
template <class T, int DK, int DV, bool kAligned, bool rev> hipError_t scan_tile(const Scan& k, Parts parts, unsigned states, hipStream_t stream) {
  constexpr size_t lds = ScanTile<T, DK, DV>::kLds;
  const auto fn = scan_chunks<T, DK, DV, kAligned, rev>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  if (parts.n_seg > 1) {
    parts.state_only = 1;
    hipLaunchKernelGGL(fn, dim3(states, (unsigned)parts.n_seg - 1), dim3(256), lds, stream, k, parts);
    hipLaunchKernelGGL((join_parts<DK, DV>), dim3(states, DK * DV / 1024), dim3(256), 0, stream, k, parts);
    parts.state_only = 0;
  }
  hipLaunchKernelGGL(fn, dim3(states, (unsigned)parts.n_seg), dim3(256), lds, stream, k, parts);
  return hipGetLastError();
}
template <class T, bool kAligned, bool rev> hipError_t scan_sizes(const Scan& k, const Parts& parts, unsigned states, hipStream_t stream) {
  if (k.dk <= 64)
    return k.dv <= 64 ? scan_tile<T, 64, 64, kAligned, rev>(k, parts, states, stream) : scan_tile<T, 64, 128, kAligned, rev>(k, parts, states, stream);
  // (in 32 bits the 128 x 128 kernel skips the upper values' tiles; one of its own was built with thousands of spills)
  if constexpr (sizeof(T) == 2)
    if (k.dv <= 64) return scan_tile<T, 128, 64, kAligned, rev>(k, parts, states, stream);
  return scan_tile<T, 128, 128, kAligned, rev>(k, parts, states, stream);
}
// (one source file per type holds these: memory_scan_<type>.hip)
template <class T> hipError_t scan_run(const Scan& k, const Parts& parts, bool aligned, unsigned states, hipStream_t stream);
template <class T> hipError_t scan_run_pair(const Scan& a, const Scan& b, bool state_vec_a, bool state_vec_b, unsigned states, hipStream_t stream);
#define EPM_SCAN_RUN_PAIR(T)                                                                                                          \
  template <>                                                                                                                         \
  hipError_t scan_run_pair<T>(const Scan& a, const Scan& b, bool state_vec_a, bool state_vec_b, unsigned states, hipStream_t stream) { \
    hipLaunchKernelGGL(scan_pair<T>, dim3(states), dim3(256), PairTile<T>::kLds, stream, a, b, (int)state_vec_a, (int)state_vec_b);    \
    return hipGetLastError();                                                                                                         \
  }
#define EPM_SCAN_RUN(T)                                                                                                       \
  template <> hipError_t scan_run<T>(const Scan& k, const Parts& parts, bool aligned, unsigned states, hipStream_t stream) { \
    if (aligned) return k.reverse ? scan_sizes<T, true, true>(k, parts, states, stream) : scan_sizes<T, true, false>(k, parts, states, stream); \
    return k.reverse ? scan_sizes<T, false, true>(k, parts, states, stream) : scan_sizes<T, false, false>(k, parts, states, stream);         \
  }

}  // namespace epm
