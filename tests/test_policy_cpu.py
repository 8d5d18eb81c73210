"""CPU: what the policy-side operators refuse, at the C ABI and in Python, before anything touches a device; the
header as C and C++; the 64-bit definitions the GPU tests rely on, against differences."""
import ctypes as C
import math
import os
import shutil
import subprocess

import pytest
import torch

from envpool_amd import capi, capi_policy as cp
from tests import policy_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 4096  # an address that is never followed: every call here is refused first


def test_header_is_plain_c_and_cxx_and_bound_completely(tmp_path):
  src = tmp_path / "hdr.c"
  src.write_text('#include "envpool_amd_policy.h"\nint main(void) { return (int)sizeof(ep_policy_rows) + EP_BF16; }\n')
  for cc, std, extra in (("gcc", "-std=c99", []), ("g++", "-std=c++11", ["-x", "c++"])):
    if not shutil.which(cc):
      continue
    r = subprocess.run([cc, std, "-Wall", "-Wextra", "-pedantic", "-Werror", "-I", os.path.join(ROOT, "include")] + extra +
                       ["-c", str(src), "-o", str(tmp_path / "hdr.o")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
  # the ctypes structs have the header's layout
  probe = tmp_path / "size.c"
  probe.write_text('#include <stdio.h>\n#include "envpool_amd_policy.h"\nint main(void) { printf("%d %d %d %d %d\\n", (int)sizeof(ep_policy_rows), '
                   '(int)sizeof(ep_memory_step_args), (int)sizeof(ep_memory_scan_args), (int)offsetof(ep_memory_scan_args, state_out_stride), '
                   '(int)offsetof(ep_policy_rows, workspace)); return 0; }\n')
  exe = tmp_path / "size"
  subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(probe), "-o", str(exe)])
  got = [int(x) for x in subprocess.check_output([str(exe)], text=True).split()]
  assert got == [C.sizeof(cp.PolicyRows), C.sizeof(cp.MemoryStepArgs), C.sizeof(cp.MemoryScanArgs), cp.MemoryScanArgs.state_out_stride.offset,
                 cp.PolicyRows.workspace.offset]
  L = cp.lib()
  assert all(hasattr(L, s) for s in cp.SYMBOLS)


def _rows(**kw):
  r = cp.PolicyRows(device_id=0, dtype=capi.EP_F32, rows=4, options=10, logits=PTR, logits_stride=10, repetition_all=1.0, temperature_all=1.0)
  for k, v in kw.items():
    setattr(r, k, v)
  return r


def _refused(rc, *words):
  text = cp.lib().ep_last_error().decode()
  assert rc == capi.EP_ERR_INVALID, (rc, text)
  assert all(w in text for w in words), text


BAD_ROWS = [
  (dict(dtype=capi.EP_F64), "dtype"), (dict(rows=-1), "rows"), (dict(rows=2**31), "rows"), (dict(options=0), "options"), (dict(options=2**30 + 1), "options"),
  (dict(logits=0), "logits"), (dict(logits=PTR + 2), "logits"), (dict(logits_stride=9), "logits_stride"), (dict(mask=PTR, mask_dtype=capi.EP_F32), "mask_dtype"),
  (dict(mask=PTR, mask_dtype=capi.EP_BOOL, mask_stride=9), "mask_stride"), (dict(mask=PTR + 1, mask_dtype=capi.EP_I32), "mask"),
  (dict(bias=PTR, bias_dtype=cp.EP_BF16), "bias_dtype"), (dict(bias=PTR, bias_dtype=capi.EP_F32, bias_stride=3), "bias_stride"),
  (dict(bias=PTR + 2, bias_dtype=capi.EP_F32), "bias"), (dict(history=PTR, history_len=-1), "history_len"),
  (dict(history=PTR, history_len=5, history_stride=4), "history_stride"), (dict(temperature_all=0.0), "temperature"), (dict(temperature_all=-1.0), "temperature"),
  (dict(temperature_all=math.inf), "temperature"), (dict(temperature_all=math.nan), "temperature"), (dict(repetition_all=0.0), "repetition"),
  (dict(frequency_all=math.inf), "frequency"), (dict(presence_all=math.nan), "presence"), (dict(num_options=PTR + 1), "aligned"),
]


@pytest.mark.parametrize("rows,options", [(2**25, 4096), (2**27, 2048), (2**27, 1024)])
def test_rows_that_one_launch_cannot_hold(rows, options):
  """A launch counts its threads in 32 bits."""
  L = cp.lib()
  r = C.byref(_rows(rows=rows, options=options, logits_stride=options, num_options=0, workspace=PTR, workspace_bytes=2**62))
  for rc in (L.ep_policy_choose(r, None, 0, PTR, PTR, PTR), L.ep_policy_evaluate(r, PTR, PTR, PTR, PTR)):
    assert rc == capi.EP_ERR_TOO_LARGE and f"{rows} rows" in L.ep_last_error().decode()


@pytest.mark.parametrize("bad,word", BAD_ROWS, ids=lambda x: str(x))
def test_rows_that_are_refused(bad, word):
  L = cp.lib()
  r = C.byref(_rows(**bad))
  _refused(L.ep_policy_choose(r, None, 0, PTR, PTR, PTR), word)
  _refused(L.ep_policy_evaluate(r, PTR, PTR, PTR, PTR), word)
  _refused(L.ep_policy_evaluate_grad(r, PTR, PTR, PTR, PTR, PTR, PTR, 10, None, 0), word)


def test_other_refusals_of_the_logits_calls():
  L = cp.lib()
  r = C.byref(_rows())
  _refused(L.ep_policy_choose(None, None, 0, PTR, PTR, PTR), "null")
  _refused(L.ep_policy_choose(r, PTR, capi.EP_I32, PTR, PTR, PTR), "u_dtype")
  _refused(L.ep_policy_choose(r, PTR + 4, capi.EP_F64, PTR, PTR, PTR), "u:")
  _refused(L.ep_policy_choose(r, None, 0, None, PTR, PTR), "action")
  _refused(L.ep_policy_evaluate(r, None, PTR, PTR, PTR), "action")
  _refused(L.ep_policy_evaluate_grad(r, PTR, None, PTR, PTR, PTR, PTR, 10, None, 0), "entropy")
  _refused(L.ep_policy_evaluate_grad(r, PTR, PTR, PTR, PTR, PTR, None, 10, None, 0), "neither")
  _refused(L.ep_policy_evaluate_grad(r, PTR, PTR, PTR, PTR, PTR, PTR, 9, None, 0), "grad_logits_stride")
  _refused(L.ep_policy_evaluate_grad(r, PTR, PTR, PTR, PTR, PTR, PTR, 10, PTR, 10), "without a bias")
  b = _rows(bias=PTR, bias_dtype=capi.EP_F32, bias_stride=10)
  _refused(L.ep_policy_evaluate_grad(C.byref(b), PTR, PTR, PTR, PTR, PTR, PTR, 10, PTR, 4), "grad_bias_stride")
  # long rows need scratch memory, and say how much
  long = _rows(options=100000, logits_stride=100000)
  need = L.ep_policy_choose_workspace(C.byref(long))
  assert need > 0 and need % 8 == 0
  _refused(L.ep_policy_choose(C.byref(long), None, 0, PTR, PTR, PTR), "workspace", str(need))
  long.workspace, long.workspace_bytes = PTR, need - 1
  _refused(L.ep_policy_choose(C.byref(long), None, 0, PTR, PTR, PTR), "workspace", str(need))
  long.workspace, long.workspace_bytes = PTR + 8, need
  _refused(L.ep_policy_choose(C.byref(long), None, 0, PTR, PTR, PTR), "16 bytes")
  # no rows: nothing to do, whatever the pointers
  none = _rows(rows=0, logits=0)
  assert L.ep_policy_choose(C.byref(none), None, 0, None, None, None) == capi.EP_OK
  assert L.ep_policy_evaluate(C.byref(none), None, None, None, None) == capi.EP_OK


def _step(**kw):
  a = cp.MemoryStepArgs(device_id=0, dtype=capi.EP_F32, num_envs=8, rows=4, heads=4, kv_heads=2, key_dim=16, value_dim=16, q=PTR, k=PTR, v=PTR, out=PTR,
                        log_decay=PTR, state=PTR, scale=1.0)
  for k, v in kw.items():
    setattr(a, k, v)
  return a


def _scan(**kw):
  a = cp.MemoryScanArgs(device_id=0, dtype=capi.EP_F32, steps=5, rows=2, heads=4, q_group=1, k_group=2, v_group=2, key_dim=16, value_dim=16, q=PTR, k=PTR,
                        v=PTR, out=PTR, out_dtype=capi.EP_F32, log_decay=PTR, inc_scale=1.0, out_scale=1.0)
  for k, v in kw.items():
    setattr(a, k, v)
  return a


@pytest.mark.parametrize("bad,word", [
  (dict(dtype=capi.EP_I32), "dtype"), (dict(num_envs=0), "num_envs"), (dict(rows=-1), "rows"), (dict(heads=0), "heads"), (dict(kv_heads=3), "kv_heads"),
  (dict(kv_heads=0), "kv_heads"), (dict(key_dim=0), "key_dim"), (dict(key_dim=257), "key_dim"), (dict(value_dim=257), "value_dim"),
  (dict(rows=9), "without env_id"), (dict(q=0), "null"), (dict(state=0), "null"), (dict(out=PTR + 1), "aligned"), (dict(state=PTR + 2), "aligned"),
  (dict(fresh=PTR, fresh_dtype=capi.EP_F32), "fresh_dtype"), (dict(scale=math.nan), "scale"),
  (dict(env_id=PTR, rows=5000), "workspace"),
], ids=lambda x: str(x))
def test_memory_steps_that_are_refused(bad, word):
  _refused(cp.lib().ep_memory_step(C.byref(_step(**bad))), word)


@pytest.mark.parametrize("bad,word", [
  (dict(dtype=capi.EP_I32), "dtype"), (dict(out_dtype=cp.EP_F16), "out_dtype"), (dict(steps=-1), "steps"), (dict(rows=-1), "rows"), (dict(heads=0), "heads"),
  (dict(k_group=3), "group"), (dict(q_group=0), "group"), (dict(key_dim=129), "key_dim"), (dict(value_dim=0), "value_dim"), (dict(log_decay=0), "log_decay"),
  (dict(q=0), "null"), (dict(out=0), "neither"), (dict(inc_scale=math.inf), "scale"), (dict(q=PTR + 2), "aligned"), (dict(out=PTR + 2), "aligned"),
  (dict(state_in=PTR + 2), "aligned"), (dict(steps=10000), "workspace"),
], ids=lambda x: str(x))
def test_scans_that_are_refused(bad, word):
  _refused(cp.lib().ep_memory_scan(C.byref(_scan(**bad))), word)


def test_null_arguments_and_empty_calls():
  L = cp.lib()
  _refused(L.ep_memory_step(None), "null")
  _refused(L.ep_memory_scan(None), "null")
  assert L.ep_memory_step(C.byref(_step(rows=0, q=0, state=0))) == capi.EP_OK
  assert L.ep_memory_scan(C.byref(_scan(rows=0, q=0, log_decay=0))) == capi.EP_OK
  _refused(L.ep_memory_sum_heads(0, PTR, 4, 2, 0, 8, PTR, capi.EP_F32, None), "group")
  _refused(L.ep_memory_sum_heads(0, PTR, 4, 2, 2, 8, PTR, capi.EP_I32, None), "dtype")
  _refused(L.ep_memory_sum_heads(0, None, 4, 2, 2, 8, PTR, capi.EP_F32, None), "null")
  assert L.ep_memory_sum_heads(0, None, 0, 2, 2, 8, None, capi.EP_F32, None) == capi.EP_OK


def test_states_that_one_launch_cannot_hold():
  L = cp.lib()
  for rc in (L.ep_memory_scan(C.byref(_scan(rows=2**24))), L.ep_memory_step(C.byref(_step(rows=2**27, num_envs=2**27)))):
    assert rc == capi.EP_ERR_TOO_LARGE and "heads" in L.ep_last_error().decode()


def test_pairs_of_scans_that_are_refused():
  L = cp.lib()
  pair = lambda a, b: L.ep_memory_scan_pair(C.byref(_scan(**a)), C.byref(_scan(**b)))  # noqa: E731
  _refused(L.ep_memory_scan_pair(None, C.byref(_scan())), "null")
  _refused(L.ep_memory_scan_pair(C.byref(_scan()), None), "null")
  _refused(pair({}, dict(key_dim=0)), "key_dim")
  _refused(pair(dict(heads=0), {}), "heads")
  _refused(pair({}, dict(device_id=1)), "one device")
  _refused(pair(dict(stream=PTR), {}), "stream")
  _refused(pair(dict(workspace=PTR), {}), "one workspace")
  _refused(pair({}, dict(steps=10000)), "workspace")
  assert L.ep_memory_scan_pair(C.byref(_scan(rows=0)), C.byref(_scan(rows=0))) == capi.EP_OK
  size = L.ep_memory_scan_pair_workspace(C.byref(_scan()), C.byref(_scan(steps=10000)))
  assert size == L.ep_memory_scan_workspace(C.byref(_scan(steps=10000))) > 0
  # many states leave time in one piece, so that the pair needs none
  assert L.ep_memory_scan_pair_workspace(C.byref(_scan(rows=4096)), C.byref(_scan(rows=4096))) == 0


def test_without_a_gpu_the_calls_fail_loudly():
  L = cp.lib()
  if L.ep_device_count() > 0:
    pytest.skip("a GPU is visible")
  for rc in (L.ep_policy_choose(C.byref(_rows()), None, 0, PTR, PTR, PTR), L.ep_memory_step(C.byref(_step())), L.ep_memory_scan(C.byref(_scan()))):
    assert rc == capi.EP_ERR_NO_DEVICE and "no CPU fallback" in L.ep_last_error().decode()


def test_python_refusals():
  from envpool_amd import policy
  x = torch.zeros(4, 10)
  i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
  cases = [
    (lambda: policy.choose(x.double()), "logits"), (lambda: policy.choose(x[0]), "logits"), (lambda: policy.choose(x[:, :0]), "logits"),
    (lambda: policy.choose(x, num_options=i32(4).long()), "num_options"), (lambda: policy.choose(x, num_options=i32(3)), "num_options"),
    (lambda: policy.choose(x, mask=torch.zeros(4, 10)), "mask"), (lambda: policy.choose(x, mask=torch.zeros(4, 9, dtype=torch.bool)), "mask"),
    (lambda: policy.choose(x, mask=i32(4, 2)), "mask"), (lambda: policy.choose(x, mask=torch.zeros(3, 10, dtype=torch.bool)), "mask"),
    (lambda: policy.choose(x, bias=torch.zeros(10, dtype=torch.float16)), "bias"), (lambda: policy.choose(x, bias=torch.zeros(11)), "bias"),
    (lambda: policy.choose(x, history=torch.zeros(4, 3)), "history"), (lambda: policy.choose(x, history=i32(2, 3)), "history"),
    (lambda: policy.choose(x, temperature=0.0), "temperature"), (lambda: policy.choose(x, temperature=torch.ones(3)), "temperature"),
    (lambda: policy.choose(x, repetition=-1.0), "repetition"), (lambda: policy.choose(x, presence=math.inf), "presence"),
    (lambda: policy.choose(x, frequency=torch.ones(4, dtype=torch.float64)), "frequency"),
    (lambda: policy.evaluate(x, i32(4)), "GPU"), (lambda: policy.choose(x), "GPU"),
    (lambda: policy.EnvMemory(0, 1, 4, 4, torch.zeros(1)), "num_envs"), (lambda: policy.EnvMemory(4, 1, 300, 4, torch.zeros(1)), "key_dim"),
    (lambda: policy.EnvMemory(4, 2, 4, 4, torch.zeros(1)), "log_decay"), (lambda: policy.EnvMemory(4, 1, 4, 4, torch.zeros(1), state=torch.zeros(4, 1, 4, 5)), "state"),
    (lambda: policy.EnvMemory(4, 1, 4, 4, torch.zeros(1)), "GPU"),
  ]
  q, k, v, d = torch.zeros(5, 2, 4, 8), torch.zeros(5, 2, 2, 8), torch.zeros(5, 2, 2, 6), torch.zeros(4)
  cases += [
    (lambda: policy.memory_scan(q.half(), k, v, d), "one type"), (lambda: policy.memory_scan(q[0], k, v, d), "q must"),
    (lambda: policy.memory_scan(q, k[:4], v, d), "k, v"), (lambda: policy.memory_scan(q, k, v[:, :, :1], d), "k, v"),
    (lambda: policy.memory_scan(q, torch.zeros(5, 2, 3, 8), torch.zeros(5, 2, 3, 6), d), "kv_heads"),
    (lambda: policy.memory_scan(torch.zeros(5, 2, 4, 200), torch.zeros(5, 2, 4, 200), torch.zeros(5, 2, 4, 6), d), "key_dim"),
    (lambda: policy.memory_scan(q, k, v, d[:3]), "log_decay"), (lambda: policy.memory_scan(q, k, v, d.clone().requires_grad_()), "log_decay"),
    (lambda: policy.memory_scan(q, k, v, d, fresh=torch.zeros(5, 3, dtype=torch.bool)), "fresh"),
    (lambda: policy.memory_scan(q, k, v, d, fresh=torch.zeros(5, 2)), "fresh"), (lambda: policy.memory_scan(q, k, v, d, state=torch.zeros(2, 4, 6, 8)), "state"),
    (lambda: policy.memory_scan(q, k, v, d), "GPU"),
  ]
  for i, (call, word) in enumerate(cases):
    with pytest.raises(ValueError, match=word):
      call()
      raise AssertionError(f"case {i} was not refused")


def test_front_ends_without_a_device_mask_refuse():
  from envpool_amd.python.pool import EnvPoolFrontEnd
  from envpool_amd.python.sharded import ShardedTorchMixin

  class Bare(EnvPoolFrontEnd):
    def __init__(self):
      pass

  with pytest.raises(RuntimeError, match="choose_torch"):
    Bare().choose_torch(torch.zeros(1, 2))
  with pytest.raises(RuntimeError, match="send_choice"):
    Bare().send_choice(None)
  for name in ("memory_torch", "choose_torch", "send_choice"):
    with pytest.raises(RuntimeError, match="several GPUs"):
      getattr(ShardedTorchMixin, name)(None)


# ---- the definitions themselves -------------------------------------------------------------------
def test_evaluate_definition_against_differences():
  g = torch.Generator().manual_seed(0)
  n, a = 3, 7
  x, b = torch.randn(n, a, generator=g).double(), torch.randn(a, generator=g).double()
  act = torch.tensor([2, 0, -1], dtype=torch.int32)
  kw = dict(history=torch.randint(0, a, (n, 4), generator=g, dtype=torch.int32), repetition=1.3, frequency=0.2, presence=0.1, temperature=0.8,
            num_options=torch.tensor([7, 4, 5], dtype=torch.int32))
  g1, g2 = torch.randn(n, generator=g), torch.randn(n, generator=g)

  def value(xx, bb):
    r = ref.evaluate(xx, act, g1, g2, bias=bb, **kw)
    return float((r["log_prob"] * g1.double() + r["entropy"] * g2.double()).sum())

  r = ref.evaluate(x, act, g1, g2, bias=b, **kw)
  eps = 1e-6
  for _ in range(5):
    dx, db = torch.randn(n, a, generator=g).double(), torch.randn(a, generator=g).double()
    num = (value(x + eps * dx, b + eps * db) - value(x - eps * dx, b - eps * db)) / (2 * eps)
    ana = float((r["grad_logits"] * dx).sum() + (r["grad_bias"].sum(0) * db).sum())
    assert abs(num - ana) < 1e-6 * (1 + abs(num))


def test_scan_definition_against_differences():
  g = torch.Generator().manual_seed(1)
  t, n, h, hk, dk, dv = 6, 2, 4, 2, 3, 5
  q, k, v = (torch.randn(t, n, x, d, generator=g).double() for x, d in ((h, dk), (hk, dk), (hk, dv)))
  s0, ds = torch.randn(n, h, dk, dv, generator=g).double(), torch.randn(n, h, dk, dv, generator=g).double()
  do = torch.randn(t, n, h, dv, generator=g).double()
  decay = -torch.rand(h, generator=g)
  fresh = torch.rand(t, n, generator=g) < 0.3
  kw = dict(fresh=fresh, scale=0.7)

  def value(q, k, v, s):
    r = ref.scan(q, k, v, decay, state=s, **kw)
    return float((r["out"] * do).sum() + (r["final"] * ds).sum())

  r = ref.scan(q, k, v, decay, state=s0, grad_out=do, reverse_from=ds, **kw)
  eps = 1e-6
  for _ in range(4):
    d = [torch.randn(x.shape, generator=g).double() for x in (q, k, v, s0)]
    up = value(*[x + eps * y for x, y in zip((q, k, v, s0), d)])
    down = value(*[x - eps * y for x, y in zip((q, k, v, s0), d)])
    ana = sum(float((r["grad_" + name] * y).sum()) for name, y in zip(("q", "k", "v", "state"), d))
    assert abs((up - down) / (2 * eps) - ana) < 1e-6 * (1 + abs(ana))
