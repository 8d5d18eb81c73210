// memory.hip - ep_memory_step / ep_memory_scan: checks and launches.
#include <algorithm>
#include <cmath>

#include "../../include/envpool_amd_policy.h"
#include "common.hpp"
#include "memory_kernels.hpp"
#include "memory_scan.hpp"

namespace {

using epc::fail;
using epc::kMaxGroups256;

bool float_type(int32_t dtype) { return dtype == EP_F32 || dtype == EP_F16 || dtype == EP_BF16; }
size_t size_of(int32_t dtype) { return dtype == EP_F32 ? 4 : 2; }

template <class F> void with_type(int32_t dtype, F f) {
  if (dtype == EP_F32) f(float{});
  else if (dtype == EP_F16) f(epm::f16{});
  else f(epm::bf16{});
}

int check_workspace(const void* ws, int64_t have, int64_t need) {
  if (need > 0 && (!ws || have < need))
    return fail(EP_ERR_INVALID, "workspace of %lld bytes is smaller than the %lld this call needs", (long long)(ws ? have : 0), (long long)need);
  if ((uintptr_t)ws % 16) return fail(EP_ERR_INVALID, "workspace: not aligned to 16 bytes");
  return EP_OK;
}

// Up to this many rows every workgroup looks the whole batch's ids through for a second row of its env
// (a few KB out of L2); above it two small launches count the rows of each env first (9 us: at 4096 rows the step
// takes 195 + 9 us with them and 208 without, at 65536 rows 433 + 10 and 6316).
constexpr int64_t kLookThrough = 1024;

int64_t step_workspace(const ep_memory_step_args* a) {
  return a->env_id && a->rows > kLookThrough ? a->num_envs * 4 : 0;
}

// the sizes of the kernel that a call's sizes run in (epm::scan_sizes chooses the same)
struct Padded {
  int dk, dv;
  int64_t state() const { return (int64_t)dk * dv; }
};
Padded padded(const ep_memory_scan_args* a) {
  const int dk = a->key_dim <= 64 ? 64 : 128;
  return {dk, a->value_dim <= 64 && (dk == 64 || a->dtype != EP_F32) ? 64 : 128};
}

template <class T> int per_cu_of(Padded d) {
  using namespace epm;
  return d.dk == 64 ? (d.dv == 64 ? ScanTile<T, 64, 64>::kPerCu : ScanTile<T, 64, 128>::kPerCu)
                    : (d.dv == 64 ? ScanTile<T, 128, 64>::kPerCu : ScanTile<T, 128, 128>::kPerCu);
}
int64_t chunk_steps(int32_t dtype) { return dtype == EP_F32 ? epm::ChunkOf<float>::value : epm::ChunkOf<epm::bf16>::value; }
int64_t per_cu(const ep_memory_scan_args* a) { return a->dtype == EP_F32 ? per_cu_of<float>(padded(a)) : per_cu_of<epm::bf16>(padded(a)); }

// Split of the time axis. One part per state keeps everything single-pass. With fewer states than the chip holds at
// once, the axis is cut into parts that are walked side by side: keys and values are then read twice (first for the
// states between the parts), which counts as 1.6 times the chunks plus the join. 32768 steps of 16 states of 128 x 128
// in bf16: 82 + 14 + 187 us in 32 parts, 3230 in one; 777 steps of 30 states in f32: 15 + 9 + 28 us, 167 in one.
int64_t scan_parts(const ep_memory_scan_args* a) {
  const int64_t states = a->rows * a->heads, chunk = chunk_steps(a->dtype), chunks = (a->steps + chunk - 1) / chunk;
  if (states <= 0 || chunks < 2) return 1;
  const int64_t slots = 256 * per_cu(a);  // workgroups that run at once
  if (states * 2 > slots) return 1;
  const int64_t per = std::max<int64_t>((chunks * states + slots - 1) / slots, (chunks + 65534) / 65535);
  const int64_t parts = (chunks + per - 1) / per;
  const int64_t rounds = (states * parts + slots - 1) / slots;
  return 10 * chunks > 16 * rounds * per + 20 ? parts : 1;
}
int64_t scan_workspace(const ep_memory_scan_args* a, int64_t n_seg) {
  if (n_seg <= 1) return 0;
  return a->rows * a->heads * n_seg * (padded(a).state() * 4 + 4);
}

// every refusal but the workspace's
int check_scan(const ep_memory_scan_args* a) {
  if (!a) return fail(EP_ERR_INVALID, "null argument");
  if (!float_type(a->dtype)) return fail(EP_ERR_INVALID, "dtype = %d is none of EP_F32, EP_F16, EP_BF16", a->dtype);
  if (a->out_dtype != a->dtype && a->out_dtype != EP_F32) return fail(EP_ERR_INVALID, "out_dtype = %d is neither dtype nor EP_F32", a->out_dtype);
  if (a->steps < 0 || a->steps > INT32_MAX) return fail(EP_ERR_INVALID, "steps = %lld", (long long)a->steps);
  if (a->rows < 0 || a->rows > INT32_MAX) return fail(EP_ERR_INVALID, "rows = %lld", (long long)a->rows);
  if (a->heads < 1 || a->heads > 65535) return fail(EP_ERR_INVALID, "heads = %d is outside [1, 65535]", a->heads);
  const int32_t groups[] = {a->q_group, a->k_group, a->v_group};
  for (int32_t g : groups)
    if (g < 1 || a->heads % g) return fail(EP_ERR_INVALID, "a head group of %d does not divide heads = %d", g, a->heads);
  if (a->key_dim < 1 || a->key_dim > 128 || a->value_dim < 1 || a->value_dim > 128)
    return fail(EP_ERR_INVALID, "key_dim = %d, value_dim = %d: not both in [1, 128]", a->key_dim, a->value_dim);
  if (a->rows > 0 && !a->log_decay) return fail(EP_ERR_INVALID, "log_decay: null pointer");
  if (a->rows > 0 && a->steps > 0 && (!a->q || !a->k || !a->v)) return fail(EP_ERR_INVALID, "q, k, v: null pointer");
  if (a->rows > 0 && a->steps > 0 && !a->out && !a->state_out) return fail(EP_ERR_INVALID, "neither out nor state_out is wanted");
  if (!std::isfinite(a->inc_scale) || !std::isfinite(a->out_scale)) return fail(EP_ERR_INVALID, "inc_scale = %g, out_scale = %g", (double)a->inc_scale, (double)a->out_scale);
  const void* typed[] = {a->q, a->k, a->v};
  for (const void* ptr : typed)
    if ((uintptr_t)ptr % size_of(a->dtype)) return fail(EP_ERR_INVALID, "q, k, v: not aligned to their type");
  if ((uintptr_t)a->out % size_of(a->out_dtype)) return fail(EP_ERR_INVALID, "out: not aligned to its type");
  const void* words[] = {a->log_decay, a->state_in, a->state_out};
  for (const void* ptr : words)
    if ((uintptr_t)ptr % 4) return fail(EP_ERR_INVALID, "an array of 4-byte values is not aligned to 4 bytes");
  if (a->rows * a->heads > kMaxGroups256) return fail(EP_ERR_TOO_LARGE, "%lld rows of %d heads", (long long)a->rows, a->heads);
  return EP_OK;
}
bool nothing_to_do(const ep_memory_scan_args* a) { return a->rows == 0 || (a->steps == 0 && !a->state_out); }

epm::Scan scan_of(const ep_memory_scan_args* a) {
  epm::Scan k{};
  k.steps = a->steps, k.rows = a->rows, k.heads = a->heads;
  k.q_group = a->q_group, k.k_group = a->k_group, k.v_group = a->v_group, k.dk = a->key_dim, k.dv = a->value_dim;
  k.q = a->q, k.k = a->k, k.v = a->v, k.out = a->out, k.out_f32 = a->out_dtype == EP_F32;
  for (int i = 0; i < 3; ++i)
    k.q_stride[i] = a->q_stride[i], k.k_stride[i] = a->k_stride[i], k.v_stride[i] = a->v_stride[i], k.out_stride[i] = a->out_stride[i];
  k.log_decay = a->log_decay, k.fresh = a->fresh;
  for (int i = 0; i < 2; ++i) k.fresh_stride[i] = a->fresh_stride[i];
  k.state_in = a->state_in, k.state_out = a->state_out;
  for (int i = 0; i < 4; ++i) k.in_stride[i] = a->state_in_stride[i], k.outs_stride[i] = a->state_out_stride[i];
  k.inc_scale = a->inc_scale, k.out_scale = a->out_scale, k.reverse = a->reverse;
  return k;
}

// whether a call's operands can be addressed through buffers in 16-byte pieces (memory_scan.hpp: kAligned)
bool buffered(const ep_memory_scan_args* a) {
  const int64_t size = size_of(a->dtype), per_load = 16 / size;
  const int64_t out_size = size_of(a->out_dtype);
  // 16-byte pieces (results: 4 values), rows that follow one another, and a chunk within 2^31 bytes
  const auto aligned = [&](const void* ptr, const int64_t* stride, int64_t width, int64_t unit, int64_t bytes) {
    return (uintptr_t)ptr % unit == 0 && stride[0] * bytes % unit == 0 && stride[1] * bytes % unit == 0 && stride[2] * bytes % unit == 0 &&
           stride[0] >= width && stride[0] * bytes <= (int64_t(1) << 31) / 64;
  };
  const auto state_near = [&](const void* ptr, const int64_t* stride) {
    return !ptr || (stride[2] >= 0 && stride[3] >= 0 && stride[2] < (1 << 20) && stride[3] < (1 << 20));
  };
  return aligned(a->q, a->q_stride, a->key_dim, 16, size) && aligned(a->k, a->k_stride, a->key_dim, 16, size) &&
                   aligned(a->v, a->v_stride, a->value_dim, 16, size) && (!a->out || aligned(a->out, a->out_stride, a->value_dim, 4 * out_size, out_size)) &&
                   state_near(a->state_in, a->state_in_stride) && state_near(a->state_out, a->state_out_stride) && a->key_dim % per_load == 0 &&
                   a->value_dim % per_load == 0;
}
bool state_vec(const ep_memory_scan_args* a) {
  return (uintptr_t)a->state_in % 16 == 0 && a->state_in_stride[0] % 4 == 0 && a->state_in_stride[1] % 4 == 0 && a->state_in_stride[3] % 4 == 0;
}

// Short segments are walked step by step (scan_few). Forward / with all gradients, us, walk of chunks against it:
//   65536 states of 16 x 16 bf16: 4 steps 468 / 1761, 110 / 421; 16 steps 470 / 1769, 310 / 1254; 32 steps 497 / 1834, 611 / 2436
//   65536 states of 32 x 32 bf16: 4 steps 478 / 1781, 133 / 476; 16 steps 484 / 1788, 317 / 1235; 32 steps 537 / 1946, 574 / 2273
//   16384 states of 64 x 64 f32:  4 steps 193 / 727, 125 / 577;  8 steps 198 / 737, 147 / 673;    16 steps 206 / 756, 197 / 877
// In 16 bits states of 64 x 64 stay with the chunks (4 steps 143 / 489, 118 / 556), whose gradients share a launch.
constexpr int64_t kFewSteps = 16, kFewKeySteps = 128;
// how scan_few lays a state over a wave: 2^width_log lanes of four values, `keys` keys a lane; keys 0: not its size
struct Few {
  int width_log, keys;
};
Few few_steps(const ep_memory_scan_args* a);

// whether two scans are the gradients of values (a) and keys (b) of one call, in a form that one kernel covers (128
// steps of 4096 states of 64 x 64 in bf16: 175 us, one after the other 204). Other sizes' two states and six tiles would
// leave a CU one workgroup, and a split axis has two walks that start from different states.
bool pairs_up(const ep_memory_scan_args* a, const ep_memory_scan_args* b) {
  const auto same = [](const int64_t* x, const int64_t* y, int n) { return std::equal(x, x + n, y); };
  return a->reverse && b->reverse && !few_steps(a).keys && a->dtype != EP_F32 && a->dtype == b->dtype && a->steps == b->steps && a->rows == b->rows && a->heads == b->heads &&
         a->key_dim <= 64 && a->value_dim <= 64 && a->key_dim == b->value_dim && a->value_dim == b->key_dim && a->k == b->v && a->v == b->k &&
         a->k_group == b->v_group && a->v_group == b->k_group && same(a->k_stride, b->v_stride, 3) && same(a->v_stride, b->k_stride, 3) &&
         a->log_decay == b->log_decay && a->fresh == b->fresh && same(a->fresh_stride, b->fresh_stride, 2) && a->inc_scale == b->inc_scale &&
         a->out_scale == b->out_scale && !b->state_out && a->steps > 0 && a->rows > 0 && buffered(a) && buffered(b) && scan_parts(a) == 1 && scan_parts(b) == 1;
}

Few few_steps(const ep_memory_scan_args* a) {
  if (a->steps < 1 || a->key_dim > 64 || a->value_dim > 64) return {0, 0};
  Few f{2, 4};
  while (4 << f.width_log < a->value_dim) ++f.width_log;
  while ((64 >> f.width_log) * f.keys < a->key_dim) f.keys *= 2;
  const bool few = a->steps <= kFewSteps && a->steps * f.keys <= kFewKeySteps && (f.keys <= 8 || a->dtype == EP_F32);
  return few ? f : Few{0, 0};
}

int launch_few(const ep_memory_scan_args* a, Few f, hipStream_t stream) {
  const epm::Scan k = scan_of(a);
  // whether states go in 16-byte pieces along the values (rows) or the keys (cols)
  const auto pieces = [](const void* ptr, const int64_t* stride, int along, int other, int width) {
    return (uintptr_t)ptr % 16 == 0 && stride[along] == 1 && stride[0] % 4 == 0 && stride[1] % 4 == 0 && stride[other] % 4 == 0 && width % 4 == 0;
  };
  const int in_rows = pieces(a->state_in, a->state_in_stride, 3, 2, a->value_dim), in_cols = pieces(a->state_in, a->state_in_stride, 2, 3, a->key_dim);
  const int out_rows = pieces(a->state_out, a->state_out_stride, 3, 2, a->value_dim), out_cols = pieces(a->state_out, a->state_out_stride, 2, 3, a->key_dim);
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    const auto kernel = f.keys == 4 ? epm::scan_few<T, 4> : f.keys == 8 ? epm::scan_few<T, 8> : epm::scan_few<T, 16>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a->rows * a->heads + 3) / 4)), dim3(256), 0, stream, k, f.width_log, in_rows, in_cols, out_rows, out_cols);
  });
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

int scan_launch(const ep_memory_scan_args* a, hipStream_t stream) {
  if (const Few f = few_steps(a); f.keys) return launch_few(a, f, stream);
  const epm::Scan k = scan_of(a);
  epm::Parts parts{};
  const int64_t chunk = chunk_steps(a->dtype), chunks = std::max<int64_t>(1, (a->steps + chunk - 1) / chunk);
  const int64_t want = scan_parts(a), per = (chunks + want - 1) / want;
  parts.seg_len = per * chunk;
  parts.n_seg = (int32_t)((chunks + per - 1) / per);
  if (parts.n_seg > 1) {
    parts.ws_state = (epm::f32x4*)a->workspace;
    parts.ws_carry = (float*)((char*)a->workspace + a->rows * a->heads * parts.n_seg * (padded(a).state() * 4));
  }
  parts.state_vec = state_vec(a);
  hipError_t e = hipSuccess;
  with_type(a->dtype, [&](auto t) { e = epm::scan_run<decltype(t)>(k, parts, buffered(a), (unsigned)(a->rows * a->heads), stream); });
  HIP_TRY(e);
  return EP_OK;
}

}  // namespace

extern "C" {

int64_t ep_memory_step_workspace(const ep_memory_step_args* a) { return a ? step_workspace(a) : 0; }

int ep_memory_step(const ep_memory_step_args* a) {
  if (!a) return fail(EP_ERR_INVALID, "null argument");
  if (!float_type(a->dtype)) return fail(EP_ERR_INVALID, "dtype = %d is none of EP_F32, EP_F16, EP_BF16", a->dtype);
  if (a->num_envs < 1 || a->num_envs > INT32_MAX) return fail(EP_ERR_INVALID, "num_envs = %lld", (long long)a->num_envs);
  if (a->rows < 0 || a->rows > INT32_MAX) return fail(EP_ERR_INVALID, "rows = %lld", (long long)a->rows);
  if (a->heads < 1 || a->heads > 65535) return fail(EP_ERR_INVALID, "heads = %d is outside [1, 65535]", a->heads);
  if (a->kv_heads < 1 || a->heads % a->kv_heads) return fail(EP_ERR_INVALID, "kv_heads = %d does not divide heads = %d", a->kv_heads, a->heads);
  if (a->key_dim < 1 || a->key_dim > 256 || a->value_dim < 1 || a->value_dim > 256)
    return fail(EP_ERR_INVALID, "key_dim = %d, value_dim = %d: not both in [1, 256]", a->key_dim, a->value_dim);
  if (!a->env_id && a->rows > a->num_envs) return fail(EP_ERR_INVALID, "rows = %lld of %lld envs without env_id", (long long)a->rows, (long long)a->num_envs);
  if (a->rows > 0 && (!a->q || !a->k || !a->v || !a->out || !a->log_decay || !a->state)) return fail(EP_ERR_INVALID, "q, k, v, out, log_decay, state: null pointer");
  if (a->fresh && a->fresh_dtype != EP_BOOL && a->fresh_dtype != EP_U8 && a->fresh_dtype != EP_I32)
    return fail(EP_ERR_INVALID, "fresh_dtype = %d is none of EP_BOOL, EP_U8, EP_I32", a->fresh_dtype);
  if (!std::isfinite(a->scale)) return fail(EP_ERR_INVALID, "scale = %g", (double)a->scale);
  const void* typed[] = {a->q, a->k, a->v, a->out};
  for (const void* ptr : typed)
    if ((uintptr_t)ptr % size_of(a->dtype)) return fail(EP_ERR_INVALID, "q, k, v, out: not aligned to their type");
  const void* words[] = {a->log_decay, a->state, a->env_id, a->fresh_dtype == EP_I32 ? a->fresh : nullptr, a->error};
  for (const void* ptr : words)
    if ((uintptr_t)ptr % 4) return fail(EP_ERR_INVALID, "an array of 4-byte values is not aligned to 4 bytes");
  if (int rc = check_workspace(a->workspace, a->workspace_bytes, step_workspace(a))) return rc;
  if (a->rows == 0) return EP_OK;
  if (a->rows * a->heads > 4 * kMaxGroups256) return fail(EP_ERR_TOO_LARGE, "%lld rows of %d heads", (long long)a->rows, a->heads);
  EP_ENTER_GPU(a->device_id);
  const hipStream_t stream = (hipStream_t)a->stream;
  epm::Step k{};
  k.num_envs = a->num_envs, k.rows = a->rows;
  k.heads = a->heads, k.kv_group = a->heads / a->kv_heads, k.dk = a->key_dim, k.dv = a->value_dim;
  k.q = a->q, k.k = a->k, k.v = a->v, k.out = a->out;
  for (int i = 0; i < 2; ++i)
    k.q_stride[i] = a->q_stride[i], k.k_stride[i] = a->k_stride[i], k.v_stride[i] = a->v_stride[i], k.out_stride[i] = a->out_stride[i];
  k.log_decay = a->log_decay, k.state = a->state, k.env_id = a->env_id, k.env_id_offset = a->env_id_offset;
  k.fresh = a->fresh, k.fresh_i32 = a->fresh_dtype == EP_I32;
  k.scale = a->scale, k.error = a->error;
  k.claims = step_workspace(a) ? (int32_t*)a->workspace : nullptr;
  if (k.claims) {
    const dim3 grid((unsigned)((a->rows + 255) / 256));
    hipLaunchKernelGGL(epm::clear_claims, grid, dim3(256), 0, stream, k);
    hipLaunchKernelGGL(epm::count_claims, grid, dim3(256), 0, stream, k);
    HIP_TRY(hipGetLastError());
  }
  const int64_t blocks = (a->rows * a->heads + 3) / 4;
  // values a lane holds side by side, as wide as rows of the state are aligned (2692 states of 101 x 66: 45 us two by
  // two, 65 one by one), and how often 64 lanes of them repeat
  const int vec = a->value_dim % 4 == 0 && (uintptr_t)a->state % 16 == 0 ? 4 : a->value_dim % 2 == 0 && (uintptr_t)a->state % 8 == 0 ? 2 : 1;
  const int cols = (a->value_dim + 64 * vec - 1) / (64 * vec);
  with_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    const auto kernel = vec == 4 ? epm::step_rows<T, 4, 1> : vec == 2 ? (cols == 1 ? epm::step_rows<T, 2, 1> : epm::step_rows<T, 2, 2>)
                                  : cols == 1 ? epm::step_rows<T, 1, 1> : cols == 2 ? epm::step_rows<T, 1, 2> : epm::step_rows<T, 1, 4>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, k);
  });
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

int ep_memory_reset(const ep_memory_step_args* a) {
  if (!a) return fail(EP_ERR_INVALID, "null argument");
  if (a->num_envs < 1 || a->num_envs > INT32_MAX) return fail(EP_ERR_INVALID, "num_envs = %lld", (long long)a->num_envs);
  if (a->rows < 0 || a->rows > INT32_MAX) return fail(EP_ERR_INVALID, "rows = %lld", (long long)a->rows);
  if (a->heads < 1 || a->heads > 65535) return fail(EP_ERR_INVALID, "heads = %d is outside [1, 65535]", a->heads);
  if (a->key_dim < 1 || a->key_dim > 256 || a->value_dim < 1 || a->value_dim > 256)
    return fail(EP_ERR_INVALID, "key_dim = %d, value_dim = %d: not both in [1, 256]", a->key_dim, a->value_dim);
  if (!a->env_id && a->rows > a->num_envs) return fail(EP_ERR_INVALID, "rows = %lld of %lld envs without env_id", (long long)a->rows, (long long)a->num_envs);
  if (a->rows > 0 && !a->state) return fail(EP_ERR_INVALID, "state: null pointer");
  const void* words[] = {a->state, a->env_id, a->error};
  for (const void* ptr : words)
    if ((uintptr_t)ptr % 4) return fail(EP_ERR_INVALID, "an array of 4-byte values is not aligned to 4 bytes");
  if (a->rows == 0) return EP_OK;
  EP_ENTER_GPU(a->device_id);
  epm::Step k{};
  k.num_envs = a->num_envs, k.rows = a->rows, k.state = a->state, k.env_id = a->env_id, k.env_id_offset = a->env_id_offset, k.error = a->error;
  const int64_t size = (int64_t)a->heads * a->key_dim * a->value_dim, stretches = std::min<int64_t>((size + 2047) / 2048, 256);
  hipLaunchKernelGGL(epm::reset_rows, dim3((unsigned)std::min<int64_t>(a->rows * stretches, kMaxGroups256)), dim3(256), 0, (hipStream_t)a->stream, k, size, stretches);
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

int64_t ep_memory_scan_workspace(const ep_memory_scan_args* a) { return a ? scan_workspace(a, scan_parts(a)) : 0; }

int ep_memory_scan(const ep_memory_scan_args* a) {
  if (int rc = check_scan(a)) return rc;
  if (int rc = check_workspace(a->workspace, a->workspace_bytes, ep_memory_scan_workspace(a))) return rc;
  if (nothing_to_do(a)) return EP_OK;
  EP_ENTER_GPU(a->device_id);
  return scan_launch(a, (hipStream_t)a->stream);
}

int64_t ep_memory_scan_pair_workspace(const ep_memory_scan_args* a, const ep_memory_scan_args* b) {
  if (!a || !b || pairs_up(a, b)) return 0;
  return std::max(ep_memory_scan_workspace(a), ep_memory_scan_workspace(b));
}

int ep_memory_scan_pair(const ep_memory_scan_args* a, const ep_memory_scan_args* b) {
  if (int rc = check_scan(a)) return rc;
  if (int rc = check_scan(b)) return rc;
  if (a->device_id != b->device_id || a->stream != b->stream) return fail(EP_ERR_INVALID, "the two scans are not on one device and stream");
  if (a->workspace != b->workspace || a->workspace_bytes != b->workspace_bytes) return fail(EP_ERR_INVALID, "the two scans do not name one workspace");
  if (int rc = check_workspace(a->workspace, a->workspace_bytes, ep_memory_scan_pair_workspace(a, b))) return rc;
  if (nothing_to_do(a) && nothing_to_do(b)) return EP_OK;
  EP_ENTER_GPU(a->device_id);
  const hipStream_t stream = (hipStream_t)a->stream;
  if (!pairs_up(a, b)) {
    if (!nothing_to_do(a))
      if (int rc = scan_launch(a, stream)) return rc;
    return nothing_to_do(b) ? EP_OK : scan_launch(b, stream);
  }
  const epm::Scan ka = scan_of(a), kb = scan_of(b);
  const unsigned states = (unsigned)(a->rows * a->heads);
  HIP_TRY(a->dtype == EP_F16 ? epm::scan_run_pair<epm::f16>(ka, kb, state_vec(a), state_vec(b), states, stream)
                             : epm::scan_run_pair<epm::bf16>(ka, kb, state_vec(a), state_vec(b), states, stream));
  return EP_OK;
}

int ep_memory_sum_heads(int32_t device_id, const float* src, int64_t n, int32_t heads_out, int32_t group, int32_t dim, void* out, int32_t dtype,
                        void* stream) {
  if (!float_type(dtype)) return fail(EP_ERR_INVALID, "dtype = %d is none of EP_F32, EP_F16, EP_BF16", dtype);
  if (n < 0 || heads_out < 1 || group < 1 || dim < 1) return fail(EP_ERR_INVALID, "n, heads_out, group, dim: out of range");
  const int64_t total = n * heads_out * dim;
  if (total == 0) return EP_OK;
  if (!src || !out) return fail(EP_ERR_INVALID, "src, out: null pointer");
  if ((uintptr_t)src % 4 || (uintptr_t)out % size_of(dtype)) return fail(EP_ERR_INVALID, "src, out: not aligned to their type");
  EP_ENTER_GPU(device_id);
  with_type(dtype, [&](auto t) {
    hipLaunchKernelGGL(epm::sum_heads<decltype(t)>, dim3((unsigned)std::min<int64_t>((total + 255) / 256, kMaxGroups256)), dim3(256), 0, (hipStream_t)stream, src, total, group, dim,
                       (decltype(t)*)out);
  });
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

}  // extern "C"
