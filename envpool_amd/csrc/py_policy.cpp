// py_policy.cpp - pybind11 module over include/envpool_amd_policy.h: addresses and sizes in, status out.
// envpool_amd/policy.py holds the checks of tensors; this file fills the structs, so that a call from
// Python costs one crossing.
#include "envpool_amd_policy.h"
#include "py_common.h"

namespace {

using u64 = uintptr_t;
template <class T> T* at(u64 p) { return reinterpret_cast<T*>(p); }

// (rows, options, logits, logits_stride), num_options, (mask, dtype, stride), (bias, dtype, stride),
// (history, len, stride), ((pointer, value) of repetition, frequency, presence, temperature)
struct Rows : ep_policy_rows {
  Rows(int device, int dtype, int64_t n, int64_t options, u64 logits, int64_t logits_stride, u64 num_options, u64 mask_, int mask_dtype_, int64_t mask_stride_,
       u64 bias_, int bias_dtype_, int64_t bias_stride_, u64 history_, int64_t history_len_, int64_t history_stride_, u64 rep, double rep_all, u64 freq,
       double freq_all, u64 pres, double pres_all, u64 temp, double temp_all, u64 stream_)
      : ep_policy_rows{} {
    device_id = device;
    this->dtype = dtype;
    rows = n, this->options = options;
    this->logits = at<void>(logits), this->logits_stride = logits_stride;
    this->num_options = at<const int32_t>(num_options);
    mask = at<void>(mask_), mask_dtype = mask_dtype_, mask_stride = mask_stride_;
    bias = at<void>(bias_), bias_dtype = bias_dtype_, bias_stride = bias_stride_;
    history = at<const int32_t>(history_), history_len = history_len_, history_stride = history_stride_;
    repetition = at<const float>(rep), repetition_all = rep_all;
    frequency = at<const float>(freq), frequency_all = freq_all;
    presence = at<const float>(pres), presence_all = pres_all;
    temperature = at<const float>(temp), temperature_all = temp_all;
    stream = at<void>(stream_);
  }
  // whether rows follow one another without gaps (or one serves all)
  bool dense() const {
    const int64_t words = mask_dtype == EP_I32 ? (options + 31) / 32 : options;
    const auto follows = [&](int64_t stride, int64_t width) { return rows <= 1 || stride == 0 || stride == width; };
    return (rows <= 1 || logits_stride == options) && (!mask || follows(mask_stride, words)) && (!bias || follows(bias_stride, options)) &&
           (!history || follows(history_stride, history_len));
  }
};

void choose(const Rows& rows, u64 u, int u_dtype, u64 action, u64 log_prob, u64 entropy, u64 workspace, int64_t workspace_bytes) {
  ep_policy_rows r = rows;
  r.workspace = at<void>(workspace), r.workspace_bytes = workspace_bytes;
  int rc;
  {
    py::gil_scoped_release rel;
    rc = ep_policy_choose(&r, at<void>(u), u_dtype, at<int32_t>(action), at<float>(log_prob), at<float>(entropy));
  }
  epy::check(rc);
}

void evaluate(const Rows& rows, u64 action, u64 log_prob, u64 entropy, u64 stats, u64 workspace, int64_t workspace_bytes) {
  ep_policy_rows r = rows;
  r.workspace = at<void>(workspace), r.workspace_bytes = workspace_bytes;
  int rc;
  {
    py::gil_scoped_release rel;
    rc = ep_policy_evaluate(&r, at<const int32_t>(action), at<float>(log_prob), at<float>(entropy), at<float>(stats));
  }
  epy::check(rc);
}

// `at_now`: where the forward pass' operands are now (logits, num_options, mask, bias, history, repetition, frequency, presence,
// temperature; then action, entropy, stats). The addresses in `rows` are not followed, those tensors may be gone.
void evaluate_grad(const Rows& rows, const std::array<u64, 12>& at_now, u64 g_lp, u64 g_h, u64 grad_logits, int64_t grad_logits_stride, u64 grad_bias,
                   int64_t grad_bias_stride, u64 workspace, int64_t workspace_bytes, u64 stream) {
  ep_policy_rows r = rows;
  r.workspace = at<void>(workspace), r.workspace_bytes = workspace_bytes;
  r.logits = at<void>(at_now[0]), r.num_options = at<const int32_t>(at_now[1]), r.mask = at<void>(at_now[2]), r.bias = at<void>(at_now[3]);
  r.history = at<const int32_t>(at_now[4]), r.repetition = at<const float>(at_now[5]), r.frequency = at<const float>(at_now[6]);
  r.presence = at<const float>(at_now[7]), r.temperature = at<const float>(at_now[8]);
  r.stream = at<void>(stream);  // (the backward pass may run on another stream than the forward pass)
  int rc;
  {
    py::gil_scoped_release rel;
    rc = ep_policy_evaluate_grad(&r, at<const int32_t>(at_now[9]), at<const float>(at_now[10]), at<const float>(at_now[11]), at<const float>(g_lp),
                                 at<const float>(g_h), at<void>(grad_logits), grad_logits_stride, at<void>(grad_bias), grad_bias_stride);
  }
  epy::check(rc);
}

// the fixed part of a memory's steps (sizes, state, decay), filled per call with the batch's tensors
struct Step {
  ep_memory_step_args a{};
  Step(int device, int64_t num_envs, int heads, int key_dim, int value_dim, u64 log_decay, u64 state, int env_id_offset, u64 error) {
    a.device_id = device, a.num_envs = num_envs, a.heads = heads, a.key_dim = key_dim, a.value_dim = value_dim;
    a.log_decay = at<const float>(log_decay), a.state = at<float>(state), a.env_id_offset = env_id_offset, a.error = at<int32_t>(error);
  }
  int64_t workspace(int64_t rows, bool with_ids) const {
    ep_memory_step_args b = a;
    b.rows = rows;
    b.env_id = with_ids ? reinterpret_cast<const int32_t*>(4) : nullptr;
    return ep_memory_step_workspace(&b);
  }
  void run(int dtype, int64_t rows, int kv_heads, u64 q, int64_t q0, int64_t q1, u64 k, int64_t k0, int64_t k1, u64 v, int64_t v0, int64_t v1, u64 out,
           int64_t o0, int64_t o1, u64 env_id, u64 fresh, int fresh_dtype, float scale, u64 workspace, int64_t workspace_bytes, u64 stream) const {
    ep_memory_step_args b = a;
    b.dtype = dtype, b.rows = rows, b.kv_heads = kv_heads;
    b.q = at<void>(q), b.q_stride[0] = q0, b.q_stride[1] = q1;
    b.k = at<void>(k), b.k_stride[0] = k0, b.k_stride[1] = k1;
    b.v = at<void>(v), b.v_stride[0] = v0, b.v_stride[1] = v1;
    b.out = at<void>(out), b.out_stride[0] = o0, b.out_stride[1] = o1;
    b.env_id = at<const int32_t>(env_id), b.fresh = at<void>(fresh), b.fresh_dtype = fresh_dtype;
    b.scale = scale, b.workspace = at<void>(workspace), b.workspace_bytes = workspace_bytes, b.stream = at<void>(stream);
    int rc;
    {
      py::gil_scoped_release rel;
      rc = ep_memory_step(&b);
    }
    epy::check(rc);
  }
  void reset(int64_t rows, u64 env_id, u64 stream) const {
    ep_memory_step_args b = a;
    b.rows = rows, b.env_id = at<const int32_t>(env_id), b.stream = at<void>(stream);
    int rc;
    {
      py::gil_scoped_release rel;
      rc = ep_memory_reset(&b);
    }
    epy::check(rc);
  }
};

using Stride3 = std::array<int64_t, 3>;
using Stride4 = std::array<int64_t, 4>;
struct Scan {
  ep_memory_scan_args a{};
  Scan(int device, int dtype, int64_t steps, int64_t rows, int heads, int key_dim, int value_dim, u64 log_decay, u64 fresh, int64_t f0, int64_t f1, u64 stream) {
    a.device_id = device, a.dtype = dtype, a.steps = steps, a.rows = rows, a.heads = heads, a.key_dim = key_dim, a.value_dim = value_dim;
    a.log_decay = at<const float>(log_decay), a.fresh = at<const uint8_t>(fresh), a.fresh_stride[0] = f0, a.fresh_stride[1] = f1;
    a.out_dtype = dtype, a.q_group = a.k_group = a.v_group = 1, a.inc_scale = a.out_scale = 1.f, a.stream = at<void>(stream);
  }
  void operands(u64 q, const Stride3& qs, int qg, u64 k, const Stride3& ks, int kg, u64 v, const Stride3& vs, int vg) {
    a.q = at<void>(q), a.k = at<void>(k), a.v = at<void>(v), a.q_group = qg, a.k_group = kg, a.v_group = vg;
    for (int i = 0; i < 3; ++i) a.q_stride[i] = qs[i], a.k_stride[i] = ks[i], a.v_stride[i] = vs[i];
  }
  void output(u64 out, const Stride3& os, int dtype) {
    a.out = at<void>(out), a.out_dtype = dtype;
    for (int i = 0; i < 3; ++i) a.out_stride[i] = os[i];
  }
  void states(u64 in, const Stride4& is, u64 out, const Stride4& os) {
    a.state_in = at<const float>(in), a.state_out = at<float>(out);
    for (int i = 0; i < 4; ++i) a.state_in_stride[i] = is[i], a.state_out_stride[i] = os[i];
  }
  int64_t workspace() const { return ep_memory_scan_workspace(&a); }
  void direction(float inc_scale, float out_scale, bool reverse) { a.inc_scale = inc_scale, a.out_scale = out_scale, a.reverse = reverse; }
  void run(u64 workspace, int64_t workspace_bytes) {
    a.workspace = at<void>(workspace), a.workspace_bytes = workspace_bytes;
    int rc;
    {
      py::gil_scoped_release rel;
      rc = ep_memory_scan(&a);
    }
    epy::check(rc);
  }
};

}  // namespace

PYBIND11_MODULE(policy_native, m) {
  m.attr("F32") = (int)EP_F32, m.attr("F64") = (int)EP_F64, m.attr("F16") = (int)EP_F16, m.attr("BF16") = (int)EP_BF16;
  m.attr("BOOL") = (int)EP_BOOL, m.attr("U8") = (int)EP_U8, m.attr("I32") = (int)EP_I32;
  py::class_<Rows>(m, "Rows")
      .def(py::init<int, int, int64_t, int64_t, u64, int64_t, u64, u64, int, int64_t, u64, int, int64_t, u64, int64_t, int64_t, u64, double, u64, double, u64,
                    double, u64, double, u64>())
      .def("choose_workspace", [](const Rows& r) { return ep_policy_choose_workspace(&r); })
      .def("evaluate_workspace", [](const Rows& r) { return ep_policy_evaluate_workspace(&r); })
      .def("grad_workspace", [](const Rows& r, bool with_bias) { return ep_policy_evaluate_grad_workspace(&r, with_bias); })
      .def("choose", &choose)
      .def("evaluate", &evaluate)
      .def("dense", &Rows::dense)
      .def("bias_per_row", [](const Rows& r) { return r.bias_stride != 0; })
      .def("evaluate_grad", &evaluate_grad);
  py::class_<Step>(m, "Step")
      .def(py::init<int, int64_t, int, int, int, u64, u64, int, u64>())
      .def("workspace", &Step::workspace)
      .def("run", &Step::run)
      .def("reset", &Step::reset);
  py::class_<Scan>(m, "Scan")
      .def(py::init<int, int, int64_t, int64_t, int, int, int, u64, u64, int64_t, int64_t, u64>())
      .def("operands", &Scan::operands)
      .def("output", &Scan::output)
      .def("states", &Scan::states)
      .def("direction", &Scan::direction)
      .def("workspace", &Scan::workspace)
      .def("run", &Scan::run);
  m.def("scan_pair_workspace", [](const Scan& x, const Scan& y) { return ep_memory_scan_pair_workspace(&x.a, &y.a); });
  m.def("scan_pair", [](Scan& x, Scan& y, u64 workspace, int64_t workspace_bytes) {
    x.a.workspace = y.a.workspace = at<void>(workspace), x.a.workspace_bytes = y.a.workspace_bytes = workspace_bytes;
    int rc;
    {
      py::gil_scoped_release rel;
      rc = ep_memory_scan_pair(&x.a, &y.a);
    }
    epy::check(rc);
  });
  m.def("sum_heads", [](int device, u64 src, int64_t n, int heads_out, int group, int dim, u64 out, int dtype, u64 stream) {
    int rc;
    {
      py::gil_scoped_release rel;
      rc = ep_memory_sum_heads(device, at<const float>(src), n, heads_out, group, dim, at<void>(out), dtype, at<void>(stream));
    }
    epy::check(rc);
  });
}
