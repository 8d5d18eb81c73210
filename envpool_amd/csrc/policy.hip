// policy.hip - ep_policy_choose / ep_policy_evaluate / ep_policy_evaluate_grad: checks and launches.
#include <algorithm>
#include <cmath>

#include "../../include/envpool_amd_policy.h"
#include "common.hpp"
#include "policy_kernels.hpp"

namespace {

using epc::fail;

size_t size_of(int32_t dtype) { return dtype == EP_F32 ? 4 : 2; }
bool float_type(int32_t dtype) { return dtype == EP_F32 || dtype == EP_F16 || dtype == EP_BF16; }

bool positive(double v) { return std::isfinite(v) && v > 0; }

// every refusal that ep_policy_rows allows for; fills `k`
int check_rows(const ep_policy_rows* r, epp::Rows* k) {
  if (!r) return fail(EP_ERR_INVALID, "null argument");
  if (!float_type(r->dtype)) return fail(EP_ERR_INVALID, "dtype = %d is none of EP_F32, EP_F16, EP_BF16", r->dtype);
  if (r->rows < 0 || r->rows > INT32_MAX) return fail(EP_ERR_INVALID, "rows = %lld", (long long)r->rows);
  if (r->options < 1 || r->options > (int64_t(1) << 30)) return fail(EP_ERR_INVALID, "options = %lld is outside [1, 2^30]", (long long)r->options);
  if (r->rows > 0 && !r->logits) return fail(EP_ERR_INVALID, "logits: null pointer");
  if (r->rows > 1 && r->logits_stride < r->options)
    return fail(EP_ERR_INVALID, "logits_stride = %lld is less than options = %lld", (long long)r->logits_stride, (long long)r->options);
  if ((uintptr_t)r->logits % size_of(r->dtype)) return fail(EP_ERR_INVALID, "logits: not aligned to its type");
  if (r->mask) {
    if (r->mask_dtype != EP_BOOL && r->mask_dtype != EP_U8 && r->mask_dtype != EP_I32)
      return fail(EP_ERR_INVALID, "mask_dtype = %d is none of EP_BOOL, EP_U8, EP_I32", r->mask_dtype);
    const int64_t need = r->mask_dtype == EP_I32 ? (r->options + 31) / 32 : r->options;
    if (r->mask_stride != 0 && r->rows > 1 && r->mask_stride < need)
      return fail(EP_ERR_INVALID, "mask_stride = %lld is neither 0 nor at least %lld", (long long)r->mask_stride, (long long)need);
    if (r->mask_dtype == EP_I32 && (uintptr_t)r->mask % 4) return fail(EP_ERR_INVALID, "mask: not aligned to its type");
  }
  if (r->bias) {
    if (r->bias_dtype != EP_F32 && r->bias_dtype != r->dtype)
      return fail(EP_ERR_INVALID, "bias_dtype = %d is neither EP_F32 nor the logits' type", r->bias_dtype);
    if (r->bias_stride != 0 && r->rows > 1 && r->bias_stride < r->options)
      return fail(EP_ERR_INVALID, "bias_stride = %lld is neither 0 nor at least options", (long long)r->bias_stride);
    if ((uintptr_t)r->bias % size_of(r->bias_dtype)) return fail(EP_ERR_INVALID, "bias: not aligned to its type");
  }
  if (r->history_len < 0) return fail(EP_ERR_INVALID, "history_len = %lld", (long long)r->history_len);
  const bool hist = r->history && r->history_len > 0;
  if (hist && r->rows > 1 && r->history_stride != 0 && r->history_stride < r->history_len)
    return fail(EP_ERR_INVALID, "history_stride = %lld is neither 0 nor at least history_len", (long long)r->history_stride);
  if (!r->temperature && !positive(r->temperature_all)) return fail(EP_ERR_INVALID, "temperature = %g is not a positive number", r->temperature_all);
  if (!r->repetition && !positive(r->repetition_all)) return fail(EP_ERR_INVALID, "repetition = %g is not a positive number", r->repetition_all);
  if (!r->frequency && !std::isfinite(r->frequency_all)) return fail(EP_ERR_INVALID, "frequency = %g", r->frequency_all);
  if (!r->presence && !std::isfinite(r->presence_all)) return fail(EP_ERR_INVALID, "presence = %g", r->presence_all);
  const void* words[] = {r->num_options, r->history, r->repetition, r->frequency, r->presence, r->temperature};
  for (const void* w : words)
    if ((uintptr_t)w % 4) return fail(EP_ERR_INVALID, "an array of 4-byte values is not aligned to 4 bytes");
  *k = epp::Rows{};
  k->rows = r->rows;
  k->options = r->options;
  k->logits = r->logits;
  k->logits_stride = r->logits_stride;
  k->num_options = r->num_options;
  k->mask = r->mask;
  k->mask_bits = r->mask && r->mask_dtype == EP_I32;
  k->mask_stride = r->mask_stride;
  k->bias = r->bias;
  k->bias_f32 = r->bias_dtype == EP_F32;
  k->bias_stride = r->bias_stride;
  k->history = hist ? r->history : nullptr;
  k->history_len = r->history_len;
  k->history_stride = r->history_stride;
  k->repetition = r->repetition, k->repetition_all = r->repetition_all;
  k->frequency = r->frequency, k->frequency_all = r->frequency_all;
  k->presence = r->presence, k->presence_all = r->presence_all;
  k->temperature = r->temperature, k->temperature_all = r->temperature_all;
  const auto rows16 = [&](const void* ptr, int64_t stride, size_t size) {
    return (uintptr_t)ptr % 16 == 0 && (r->rows <= 1 || (stride * (int64_t)size) % 16 == 0);
  };
  k->vec = rows16(r->logits, r->logits_stride, size_of(r->dtype)) &&
           (!r->bias || r->bias_dtype != EP_F32 || rows16(r->bias, r->bias_stride, 4));
  return EP_OK;
}

int check_workspace(const ep_policy_rows* r, int64_t need) {
  if (need > 0 && (!r->workspace || r->workspace_bytes < need))
    return fail(EP_ERR_INVALID, "workspace of %lld bytes is smaller than the %lld this call needs", (long long)(r->workspace ? r->workspace_bytes : 0),
                (long long)need);
  if ((uintptr_t)r->workspace % 16) return fail(EP_ERR_INVALID, "workspace: not aligned to 16 bytes");
  return EP_OK;
}

template <class F> void with_type(int32_t dtype, F f) {
  if (dtype == EP_F32) f(float{});
  else if (dtype == EP_F16) f(epp::f16{});
  else f(epp::bf16{});
}

// rows of the gradient kernel are split so that about this many workgroups stand on the chip (8 a CU)
constexpr int64_t kGradBlocks = 2048;

int64_t grad_row_blocks(int64_t rows, int64_t options) {
  const int64_t pieces = (options + epp::kPiece - 1) / epp::kPiece;
  const int64_t blocks = std::min<int64_t>(std::min<int64_t>(rows, 65535), std::max<int64_t>(1, kGradBlocks / pieces));
  const int64_t per = (rows + blocks - 1) / std::max<int64_t>(blocks, 1);
  return per > 0 ? (rows + per - 1) / per : 0;
}

}  // namespace

extern "C" {

int64_t ep_policy_choose_workspace(const ep_policy_rows*) { return 0; }

int ep_policy_choose(const ep_policy_rows* r, const void* u, int32_t u_dtype, int32_t* action, float* log_prob, float* entropy) {
  epp::Rows k;
  if (int rc = check_rows(r, &k)) return rc;
  if (u && u_dtype != EP_F32 && u_dtype != EP_F64) return fail(EP_ERR_INVALID, "u_dtype = %d is neither EP_F32 nor EP_F64", u_dtype);
  if (u && (uintptr_t)u % (u_dtype == EP_F64 ? 8 : 4)) return fail(EP_ERR_INVALID, "u: not aligned to its type");
  if (r->rows > 0 && (!action || !log_prob || !entropy)) return fail(EP_ERR_INVALID, "action, log_prob, entropy: null pointer");
  if (int rc = check_workspace(r, ep_policy_choose_workspace(r))) return rc;
  if (r->rows == 0) return EP_OK;
  EP_ENTER_DEVICE(r->device_id);
  const unsigned grid = (unsigned)std::min<int64_t>(r->rows, 1 << 20);
  with_type(r->dtype, [&](auto t) {
    hipLaunchKernelGGL(epp::choose_row<decltype(t)>, dim3(grid), dim3(epp::kThreads), 0, (hipStream_t)r->stream, k, u, u_dtype == EP_F64, action,
                       log_prob, entropy);
  });
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

int64_t ep_policy_evaluate_workspace(const ep_policy_rows*) { return 0; }

int ep_policy_evaluate(const ep_policy_rows* r, const int32_t* action, float* log_prob, float* entropy, float* stats) {
  epp::Rows k;
  if (int rc = check_rows(r, &k)) return rc;
  if (r->rows > 0 && (!action || !log_prob || !entropy || !stats)) return fail(EP_ERR_INVALID, "action, log_prob, entropy, stats: null pointer");
  if (int rc = check_workspace(r, ep_policy_evaluate_workspace(r))) return rc;
  if (r->rows == 0) return EP_OK;
  EP_ENTER_DEVICE(r->device_id);
  const unsigned grid = (unsigned)std::min<int64_t>(r->rows, 1 << 20);
  with_type(r->dtype, [&](auto t) {
    hipLaunchKernelGGL(epp::evaluate_row<decltype(t)>, dim3(grid), dim3(epp::kThreads), 0, (hipStream_t)r->stream, k, action, log_prob, entropy, stats);
  });
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

int64_t ep_policy_evaluate_grad_workspace(const ep_policy_rows* r, int32_t with_bias) {
  if (!r || !with_bias || !r->bias || r->bias_stride != 0 || r->rows <= 0 || r->options < 1) return 0;
  return grad_row_blocks(r->rows, r->options) * r->options * 4;
}

int ep_policy_evaluate_grad(const ep_policy_rows* r, const int32_t* action, const float* entropy, const float* stats,
                            const float* grad_log_prob, const float* grad_entropy, void* grad_logits, int64_t grad_logits_stride,
                            void* grad_bias, int64_t grad_bias_stride) {
  epp::Rows k;
  if (int rc = check_rows(r, &k)) return rc;
  if (r->rows > 0 && (!action || !entropy || !stats)) return fail(EP_ERR_INVALID, "action, entropy, stats: null pointer");
  if (!grad_logits && !grad_bias) return fail(EP_ERR_INVALID, "neither grad_logits nor grad_bias is wanted");
  if (grad_logits && r->rows > 1 && grad_logits_stride < r->options) return fail(EP_ERR_INVALID, "grad_logits_stride = %lld is less than options", (long long)grad_logits_stride);
  if ((uintptr_t)grad_logits % size_of(r->dtype)) return fail(EP_ERR_INVALID, "grad_logits: not aligned to its type");
  if (grad_bias && !r->bias) return fail(EP_ERR_INVALID, "grad_bias without a bias");
  const bool shared = grad_bias && r->bias_stride == 0;
  if (grad_bias && !shared && r->rows > 1 && grad_bias_stride < r->options)
    return fail(EP_ERR_INVALID, "grad_bias_stride = %lld is less than options", (long long)grad_bias_stride);
  if (grad_bias && (uintptr_t)grad_bias % size_of(r->bias_dtype)) return fail(EP_ERR_INVALID, "grad_bias: not aligned to its type");
  if (int rc = check_workspace(r, ep_policy_evaluate_grad_workspace(r, grad_bias != nullptr))) return rc;
  EP_ENTER_DEVICE(r->device_id);
  const hipStream_t stream = (hipStream_t)r->stream;
  const int64_t pieces = (r->options + epp::kPiece - 1) / epp::kPiece;
  const int64_t blocks = grad_row_blocks(r->rows, r->options);
  float* partial = shared ? (float*)r->workspace : nullptr;
  if (r->rows > 0) {
    epp::GradArgs g{action, entropy, stats, grad_log_prob, grad_entropy, grad_logits, grad_logits_stride, shared ? nullptr : grad_bias, grad_bias_stride,
                    partial, 0};
    g.vec_out = (uintptr_t)grad_logits % 16 == 0 && (r->rows <= 1 || (grad_logits_stride * (int64_t)size_of(r->dtype)) % 16 == 0);
    const int64_t per = (r->rows + blocks - 1) / blocks;
    with_type(r->dtype, [&](auto t) {
      hipLaunchKernelGGL(epp::evaluate_grad_piece<decltype(t)>, dim3((unsigned)pieces, (unsigned)blocks), dim3(epp::kThreads), 0, stream, k, g, per);
    });
    HIP_TRY(hipGetLastError());
  }
  if (shared) {
    with_type(r->bias_dtype, [&](auto t) {
      hipLaunchKernelGGL(epp::sum_partials<decltype(t)>, dim3((unsigned)((r->options + 15) / 16)), dim3(epp::kThreads), 0, stream, partial,
                         r->rows > 0 ? blocks : 0, r->options, (decltype(t)*)grad_bias);
    });
    HIP_TRY(hipGetLastError());
  }
  return EP_OK;
}

}  // extern "C"
