"""ctypes binding of include/envpool_amd_policy.h (the policy-side operators' C ABI), as a foreign caller sees it.
envpool_amd/policy.py is the torch front-end (over a pybind11 module, one crossing per call)."""
import ctypes as C

from . import capi
from ._loader import load_library

EP_F16, EP_BF16 = 7, 8

_vp, _i32, _i64, _f32, _f64 = C.c_void_p, C.c_int32, C.c_int64, C.c_float, C.c_double


class PolicyRows(C.Structure):
  _fields_ = [("device_id", _i32), ("dtype", _i32), ("rows", _i64), ("options", _i64), ("logits", _vp), ("logits_stride", _i64),
              ("num_options", _vp), ("mask", _vp), ("mask_dtype", _i32), ("mask_stride", _i64), ("bias", _vp), ("bias_dtype", _i32),
              ("bias_stride", _i64), ("history", _vp), ("history_len", _i64), ("history_stride", _i64), ("repetition", _vp), ("frequency", _vp),
              ("presence", _vp), ("temperature", _vp), ("repetition_all", _f64), ("frequency_all", _f64), ("presence_all", _f64),
              ("temperature_all", _f64), ("workspace", _vp), ("workspace_bytes", _i64), ("stream", _vp)]


class MemoryStepArgs(C.Structure):
  _fields_ = [("device_id", _i32), ("dtype", _i32), ("num_envs", _i64), ("rows", _i64), ("heads", _i32), ("kv_heads", _i32), ("key_dim", _i32),
              ("value_dim", _i32), ("q", _vp), ("k", _vp), ("v", _vp), ("q_stride", _i64 * 2), ("k_stride", _i64 * 2), ("v_stride", _i64 * 2),
              ("out_stride", _i64 * 2), ("out", _vp), ("log_decay", _vp), ("state", _vp), ("env_id", _vp), ("env_id_offset", _i32), ("fresh", _vp),
              ("fresh_dtype", _i32), ("scale", _f32), ("error", _vp), ("workspace", _vp), ("workspace_bytes", _i64), ("stream", _vp)]


class MemoryScanArgs(C.Structure):
  _fields_ = [("device_id", _i32), ("dtype", _i32), ("steps", _i64), ("rows", _i64), ("heads", _i32), ("q_group", _i32), ("k_group", _i32),
              ("v_group", _i32), ("key_dim", _i32), ("value_dim", _i32), ("q", _vp), ("k", _vp), ("v", _vp), ("q_stride", _i64 * 3),
              ("k_stride", _i64 * 3), ("v_stride", _i64 * 3), ("out_stride", _i64 * 3), ("out", _vp), ("out_dtype", _i32), ("log_decay", _vp),
              ("fresh", _vp), ("fresh_stride", _i64 * 2), ("state_in", _vp), ("state_out", _vp), ("state_in_stride", _i64 * 4),
              ("state_out_stride", _i64 * 4), ("inc_scale", _f32), ("out_scale", _f32), ("reverse", _i32), ("workspace", _vp),
              ("workspace_bytes", _i64), ("stream", _vp)]


SYMBOLS = [
  "ep_policy_choose", "ep_policy_choose_workspace", "ep_policy_evaluate", "ep_policy_evaluate_workspace", "ep_policy_evaluate_grad",
  "ep_policy_evaluate_grad_workspace", "ep_memory_step", "ep_memory_step_workspace", "ep_memory_reset", "ep_memory_scan", "ep_memory_scan_workspace",
  "ep_memory_scan_pair", "ep_memory_scan_pair_workspace",
  "ep_memory_sum_heads",
]

_bound = None


def lib():
  global _bound
  if _bound is None:
    capi.lib()
    L = load_library()
    rows, step, scan = C.POINTER(PolicyRows), C.POINTER(MemoryStepArgs), C.POINTER(MemoryScanArgs)
    L.ep_policy_choose.argtypes = [rows, _vp, _i32, _vp, _vp, _vp]
    L.ep_policy_evaluate.argtypes = [rows, _vp, _vp, _vp, _vp]
    L.ep_policy_evaluate_grad.argtypes = [rows, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _i64]
    L.ep_memory_step.argtypes = [step]
    L.ep_memory_reset.argtypes = [step]
    L.ep_memory_scan.argtypes = [scan]
    L.ep_memory_scan_pair.argtypes = [scan, scan]
    L.ep_memory_sum_heads.argtypes = [_i32, _vp, _i64, _i32, _i32, _i32, _vp, _i32, _vp]
    for name, args in (("ep_policy_choose_workspace", [rows]), ("ep_policy_evaluate_workspace", [rows]),
                       ("ep_policy_evaluate_grad_workspace", [rows, _i32]), ("ep_memory_step_workspace", [step]),
                       ("ep_memory_scan_workspace", [scan]), ("ep_memory_scan_pair_workspace", [scan, scan])):
      getattr(L, name).argtypes = args
      getattr(L, name).restype = _i64
    _bound = L
  return _bound
