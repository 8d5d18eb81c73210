// policy.hip - ep_policy_choose / ep_policy_evaluate / ep_policy_evaluate_grad: checks and launches.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/envpool_amd_policy.h"
#include "common.hpp"
#include "policy_kernels.hpp"

namespace {

using epc::fail;
using epc::kMaxGroups256;

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
  k->inv_t_all = 1.0 / r->temperature_all, k->inv_t_all_32 = 1.f / (float)r->temperature_all;
  const auto rows16 = [&](const void* ptr, int64_t stride, size_t size) {
    return (uintptr_t)ptr % 16 == 0 && (r->rows <= 1 || (stride * (int64_t)size) % 16 == 0);
  };
  k->vec = rows16(r->logits, r->logits_stride, size_of(r->dtype)) &&
           (!r->bias || r->bias_dtype != EP_F32 || rows16(r->bias, r->bias_stride, 4)) &&
           (!r->mask || r->mask_dtype == EP_I32 || ((uintptr_t)r->mask % 8 == 0 && (r->rows <= 1 || r->mask_stride % 8 == 0)));
  return EP_OK;
}

// evaluate computes in 32 bits: a number for all rows that those do not hold would make every row BAD
int check_narrow(const ep_policy_rows* r) {
  const auto holds = [](double v) { return v < INFINITY && (float)v > 0.f && (float)v < INFINITY && 1.f / (float)v < INFINITY; };
  if (!r->temperature && !holds(r->temperature_all)) return fail(EP_ERR_INVALID, "temperature = %g: 32 bits do not hold it and its reciprocal", r->temperature_all);
  if (!r->history || r->history_len == 0) return EP_OK;
  if (!r->repetition && !holds(r->repetition_all)) return fail(EP_ERR_INVALID, "repetition = %g: 32 bits do not hold it and its reciprocal", r->repetition_all);
  if (!r->frequency && !std::isfinite((float)r->frequency_all)) return fail(EP_ERR_INVALID, "frequency = %g: 32 bits do not hold it", r->frequency_all);
  if (!r->presence && !std::isfinite((float)r->presence_all)) return fail(EP_ERR_INVALID, "presence = %g: 32 bits do not hold it", r->presence_all);
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
template <class F> void with_kernel(int32_t dtype, const epp::Rows& k, F f, bool vec_out = true) {
  const bool whole = k.vec && vec_out && k.options % epp::kPer == 0;
  with_type(dtype, [&](auto t) {
    if (k.history && whole) f(t, std::true_type{}, std::true_type{});
    else if (k.history) f(t, std::true_type{}, std::false_type{});
    else if (whole) f(t, std::false_type{}, std::true_type{});
    else f(t, std::false_type{}, std::false_type{});
  });
}

// How rows map to the chip. Up to 2048 options a row is held by 1 to 64 neighbouring lanes (8 options a lane and
// piece, 1 or 4 pieces): enough lanes for the options, and for a long history at least a lane per 16 entries
// of it. Longer rows are walked by workgroups, 2048 options at a time; with few rows each is cut into parts so
// that about kFill workgroups stand on the chip (eight a CU; kChooseFill: the choice walks down one part again to
// find its option, so shorter parts pay twice: 64 x 131072 bf16 takes 31 + 13 us in parts of 2048 options, 28 + 17
// in parts of 4096).
constexpr int64_t kGroupOptions = 64 * epp::kPer * 4;
constexpr int64_t kFill = 2048, kChooseFill = 2 * kFill;
constexpr int64_t kManyOctets = 262144;

struct Width {
  int log, pieces;
  unsigned blocks;  // workgroups for all rows
  size_t lds;
};
Width group_width(const epp::Rows& k, bool grad = false) {
  const int64_t octets = (k.options + epp::kPer - 1) / epp::kPer;
  // More pieces a lane mean fewer lanes a row and less work that every lane repeats (one lane for 16 options: no
  // exchange at all), at half the lanes in flight: for rows that fill the chip anyway (choose, 524288 x 16 bf16:
  // 18.1 us with two pieces a lane, 22.3 with one; evaluate, 524288 x 24: 15.4 and 20.5; but 4096 x 16 f32: 4.6
  // with two, 3.9 with one). Not for the
  // gradients, which keep a sum per option: 524288 x 24 bf16 takes 21 us with one piece a lane, 30 with two.
  Width w{0, octets > 128 ? 4 : octets > 64 || (!grad && octets > 1 && k.rows * octets >= kManyOctets) ? 2 : 1, 0, 0};
  const int64_t lanes = (octets + w.pieces - 1) / w.pieces;
  const int64_t want = std::max<int64_t>(lanes, k.history ? std::min<int64_t>(64, (k.history_len + 15) / 16) : 1);
  while ((1 << w.log) < want) ++w.log;
  const int64_t per = epp::kThreads >> w.log;
  w.blocks = (unsigned)((k.rows + per - 1) / per);
  w.lds = (size_t)epp::kThreads * epp::kPer * w.pieces * 4;
  return w;
}

struct Cut {
  int pieces, parts;  // pieces per part, parts per row
};
Cut cut_rows(int64_t rows, int64_t options, int64_t fill = kFill) {
  const int64_t all = (options + epp::kPiece - 1) / epp::kPiece;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(all, (fill + rows - 1) / std::max<int64_t>(rows, 1)));
  const int64_t pieces = (all + want - 1) / want;
  return {(int)pieces, (int)((all + pieces - 1) / pieces)};
}

// partial sums of a shared bias' gradient: one row of them per workgroup that walks down rows
int64_t grad_group_blocks(const Width& w) { return std::min<int64_t>(w.blocks, 256 * epp::grad_group_per_cu(w.pieces)); }
int64_t grad_row_blocks(int64_t rows, int64_t options) {
  const int64_t pieces = (options + epp::kPiece - 1) / epp::kPiece;
  const int64_t blocks = std::min<int64_t>(std::min<int64_t>(rows, 65535), std::max<int64_t>(1, 256 * epp::kGradPieceBlocks / pieces));
  const int64_t per = (rows + blocks - 1) / std::max<int64_t>(blocks, 1);
  return per > 0 ? (rows + per - 1) / per : 0;
}

// whether one launch can hold the workgroups of a pass over the rows
int check_groups(const ep_policy_rows* r, const epp::Rows& k, int64_t fill) {
  const int64_t groups = r->options <= kGroupOptions ? group_width(k).blocks : r->rows * cut_rows(r->rows, r->options, fill).parts;
  if (groups > kMaxGroups256) return fail(EP_ERR_TOO_LARGE, "%lld rows of %lld options", (long long)r->rows, (long long)r->options);
  return EP_OK;
}

}  // namespace

extern "C" {

int64_t ep_policy_choose_workspace(const ep_policy_rows* r) {
  if (!r || r->rows <= 0 || r->options <= kGroupOptions) return 0;
  return r->rows * cut_rows(r->rows, r->options, kChooseFill).parts * (int64_t)sizeof(epp::Stat<double>);
}

int ep_policy_choose(const ep_policy_rows* r, const void* u, int32_t u_dtype, int32_t* action, float* log_prob, float* entropy) {
  epp::Rows k;
  if (int rc = check_rows(r, &k)) return rc;
  if (u && u_dtype != EP_F32 && u_dtype != EP_F64) return fail(EP_ERR_INVALID, "u_dtype = %d is neither EP_F32 nor EP_F64", u_dtype);
  if (u && (uintptr_t)u % (u_dtype == EP_F64 ? 8 : 4)) return fail(EP_ERR_INVALID, "u: not aligned to its type");
  if (r->rows > 0 && (!action || !log_prob || !entropy)) return fail(EP_ERR_INVALID, "action, log_prob, entropy: null pointer");
  if (r->rows == 0) return EP_OK;
  if (int rc = check_groups(r, k, kChooseFill)) return rc;
  if (int rc = check_workspace(r, ep_policy_choose_workspace(r))) return rc;
  EP_ENTER_GPU(r->device_id);
  const hipStream_t stream = (hipStream_t)r->stream;
  const epp::ChooseOut out{action, log_prob, entropy};
  const int u_f64 = u_dtype == EP_F64;
  if (r->options <= kGroupOptions) {
    const Width w = group_width(k);
    const size_t lds = k.history ? w.lds : 0;
    with_kernel(r->dtype, k, [&](auto t, auto h, auto whole) {
      if (w.pieces == 1) hipLaunchKernelGGL((epp::choose_group<decltype(t), 1, h.value, whole.value>), dim3(w.blocks), dim3(epp::kThreads), lds, stream, k, w.log, u, u_f64, out);
      else if (w.pieces == 2) hipLaunchKernelGGL((epp::choose_group<decltype(t), 2, h.value, whole.value>), dim3(w.blocks), dim3(epp::kThreads), lds, stream, k, w.log, u, u_f64, out);
      else hipLaunchKernelGGL((epp::choose_group<decltype(t), 4, h.value, whole.value>), dim3(w.blocks), dim3(epp::kThreads), lds, stream, k, w.log, u, u_f64, out);
    });
  } else {
    const Cut cut = cut_rows(r->rows, r->options, kChooseFill);
    auto* parts = (epp::Stat<double>*)r->workspace;
    with_kernel(r->dtype, k, [&](auto t, auto h, auto whole) {
      const auto stats = u ? epp::choose_parts<decltype(t), h.value, whole.value, false> : epp::choose_parts<decltype(t), h.value, whole.value, true>;
      hipLaunchKernelGGL(stats, dim3((unsigned)(r->rows * cut.parts)), dim3(epp::kThreads), 0, stream, k, cut.pieces, cut.parts, parts);
      hipLaunchKernelGGL((epp::choose_join<decltype(t), h.value, whole.value>), dim3((unsigned)r->rows), dim3(epp::kThreads), 0, stream, k, cut.pieces, cut.parts, parts, u, u_f64, out);
    });
  }
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

int64_t ep_policy_evaluate_workspace(const ep_policy_rows* r) {
  if (!r || r->rows <= 0 || r->options <= kGroupOptions) return 0;
  const Cut cut = cut_rows(r->rows, r->options);
  return cut.parts == 1 ? 0 : r->rows * cut.parts * (int64_t)sizeof(epp::EvaluatePart);
}

int ep_policy_evaluate(const ep_policy_rows* r, const int32_t* action, float* log_prob, float* entropy, float* stats) {
  epp::Rows k;
  if (int rc = check_rows(r, &k)) return rc;
  if (int rc = check_narrow(r)) return rc;
  if (r->rows > 0 && (!action || !log_prob || !entropy || !stats)) return fail(EP_ERR_INVALID, "action, log_prob, entropy, stats: null pointer");
  if (r->rows == 0) return EP_OK;
  if (int rc = check_groups(r, k, kFill)) return rc;
  if (int rc = check_workspace(r, ep_policy_evaluate_workspace(r))) return rc;
  EP_ENTER_GPU(r->device_id);
  const hipStream_t stream = (hipStream_t)r->stream;
  const epp::EvaluateOut out{action, log_prob, entropy, stats};
  if (r->options <= kGroupOptions) {
    const Width w = group_width(k);
    const size_t lds = k.history ? w.lds : 0;
    with_kernel(r->dtype, k, [&](auto t, auto h, auto whole) {
      if (w.pieces == 1) hipLaunchKernelGGL((epp::evaluate_group<decltype(t), 1, h.value, whole.value>), dim3(w.blocks), dim3(epp::kThreads), lds, stream, k, w.log, out);
      else if (w.pieces == 2) hipLaunchKernelGGL((epp::evaluate_group<decltype(t), 2, h.value, whole.value>), dim3(w.blocks), dim3(epp::kThreads), lds, stream, k, w.log, out);
      else hipLaunchKernelGGL((epp::evaluate_group<decltype(t), 4, h.value, whole.value>), dim3(w.blocks), dim3(epp::kThreads), lds, stream, k, w.log, out);
    });
  } else {
    const Cut cut = cut_rows(r->rows, r->options);
    auto* parts = (epp::EvaluatePart*)r->workspace;
    with_kernel(r->dtype, k, [&](auto t, auto h, auto whole) {
      hipLaunchKernelGGL((epp::evaluate_parts<decltype(t), h.value, whole.value>), dim3((unsigned)(r->rows * cut.parts)), dim3(epp::kThreads), 0, stream, k, cut.pieces, cut.parts, parts, out);
    });
    if (cut.parts > 1)
      hipLaunchKernelGGL(epp::evaluate_join, dim3((unsigned)((r->rows + 3) / 4)), dim3(epp::kThreads), 0, stream, k, cut.parts, parts, out);
  }
  HIP_TRY(hipGetLastError());
  return EP_OK;
}

int64_t ep_policy_evaluate_grad_workspace(const ep_policy_rows* r, int32_t with_bias) {
  if (!r || !with_bias || !r->bias || r->bias_stride != 0 || r->rows <= 0 || r->options < 1) return 0;
  if (r->options > kGroupOptions) return grad_row_blocks(r->rows, r->options) * r->options * 4;
  epp::Rows k{};
  k.rows = r->rows, k.options = r->options, k.history = r->history_len > 0 ? r->history : nullptr, k.history_len = r->history_len;
  return grad_group_blocks(group_width(k, true)) * r->options * 4;
}

int ep_policy_evaluate_grad(const ep_policy_rows* r, const int32_t* action, const float* entropy, const float* stats,
                            const float* grad_log_prob, const float* grad_entropy, void* grad_logits, int64_t grad_logits_stride,
                            void* grad_bias, int64_t grad_bias_stride) {
  epp::Rows k;
  if (int rc = check_rows(r, &k)) return rc;
  if (int rc = check_narrow(r)) return rc;
  if (r->rows > 0 && (!action || !entropy || !stats)) return fail(EP_ERR_INVALID, "action, entropy, stats: null pointer");
  if (r->rows > 0 && !grad_logits && !grad_bias) return fail(EP_ERR_INVALID, "neither grad_logits nor grad_bias is wanted");
  if (grad_logits && r->rows > 1 && grad_logits_stride < r->options) return fail(EP_ERR_INVALID, "grad_logits_stride = %lld is less than options", (long long)grad_logits_stride);
  if ((uintptr_t)grad_logits % size_of(r->dtype)) return fail(EP_ERR_INVALID, "grad_logits: not aligned to its type");
  if (grad_bias && !r->bias) return fail(EP_ERR_INVALID, "grad_bias without a bias");
  const bool shared = grad_bias && r->bias_stride == 0;
  if (grad_bias && !shared && r->rows > 1 && grad_bias_stride < r->options)
    return fail(EP_ERR_INVALID, "grad_bias_stride = %lld is less than options", (long long)grad_bias_stride);
  if (grad_bias && (uintptr_t)grad_bias % size_of(r->bias_dtype)) return fail(EP_ERR_INVALID, "grad_bias: not aligned to its type");
  if (int rc = check_workspace(r, ep_policy_evaluate_grad_workspace(r, grad_bias != nullptr))) return rc;
  EP_ENTER_GPU(r->device_id);
  const hipStream_t stream = (hipStream_t)r->stream;
  const int64_t pieces = (r->options + epp::kPiece - 1) / epp::kPiece;
  const bool group = r->options <= kGroupOptions;
  const Width w = group ? group_width(k, true) : Width{};
  const int64_t blocks = group ? grad_group_blocks(w) : grad_row_blocks(r->rows, r->options);
  float* partial = shared ? (float*)r->workspace : nullptr;
  if (r->rows > 0) {
    epp::GradArgs g{action, entropy, stats, grad_log_prob, grad_entropy, grad_logits, grad_logits_stride, shared ? nullptr : grad_bias, grad_bias_stride,
                    partial, 0};
    g.vec_out = (uintptr_t)grad_logits % 16 == 0 && (r->rows <= 1 || (grad_logits_stride * (int64_t)size_of(r->dtype)) % 16 == 0);
    const int64_t per = (r->rows + blocks - 1) / blocks;
    with_kernel(r->dtype, k, [&](auto t, auto h, auto whole) {
      const size_t lds = k.history || shared ? w.lds : 0;
      if (group && w.pieces == 1)
        hipLaunchKernelGGL((epp::evaluate_grad_group<decltype(t), 1, h.value, whole.value>), dim3((unsigned)blocks), dim3(epp::kThreads), lds, stream, k, g, w.log, (int64_t)w.blocks);
      else if (group && w.pieces == 2)
        hipLaunchKernelGGL((epp::evaluate_grad_group<decltype(t), 2, h.value, whole.value>), dim3((unsigned)blocks), dim3(epp::kThreads), lds, stream, k, g, w.log, (int64_t)w.blocks);
      else if (group)
        hipLaunchKernelGGL((epp::evaluate_grad_group<decltype(t), 4, h.value, whole.value>), dim3((unsigned)blocks), dim3(epp::kThreads), lds, stream, k, g, w.log, (int64_t)w.blocks);
      else
        hipLaunchKernelGGL((epp::evaluate_grad_piece<decltype(t), h.value, whole.value>), dim3((unsigned)pieces, (unsigned)blocks), dim3(epp::kThreads), 0, stream, k, g, per);
    }, g.vec_out);
    HIP_TRY(hipGetLastError());
  }
  if (shared) {
    with_type(r->bias_dtype, [&](auto t) {
      // few columns: four a workgroup, so that 64 threads go down each; many: a cache line of them
      const int cols = r->options <= 1024 ? 4 : 32;
      const unsigned groups = (unsigned)std::min<int64_t>((r->options + cols - 1) / cols, 65536);
      const auto sum = cols == 4 ? epp::sum_partials<decltype(t), 4> : epp::sum_partials<decltype(t), 32>;
      hipLaunchKernelGGL(sum, dim3(groups), dim3(epp::kThreads), 0, stream, partial, r->rows > 0 ? blocks : 0, r->options, (decltype(t)*)grad_bias);
    });
    HIP_TRY(hipGetLastError());
  }
  return EP_OK;
}

}  // extern "C"
