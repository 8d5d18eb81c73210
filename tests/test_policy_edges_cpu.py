"""CPU: edges of the policy-side operators that show without a GPU - what a stand-in for the native module is handed, what
Python refuses before anything touches a device."""
import types

import pytest
import torch


class _FakeRows:
  """Takes the native struct's place: notes the addresses that a call would follow."""
  calls = []

  def __init__(self, dev, dtype, rows, options, logits, logits_stride, num_options, mask, mask_dtype, mask_stride, bias, bias_dtype, bias_stride, history,
               history_len, history_stride, rep, rep_all, freq, freq_all, pres, pres_all, temp, temp_all, stream):
    self.at = {"logits": logits, "num_options": num_options, "mask": mask, "bias": bias, "history": history, "repetition": rep, "frequency": freq,
               "presence": pres, "temperature": temp}
    self.strides = {"logits": logits_stride, "mask": mask_stride, "bias": bias_stride, "history": history_stride}
    self.is_dense = logits_stride == options and mask_stride in (0, options) and bias_stride in (0, options) and history_stride in (0, history_len)

  def evaluate_workspace(self):
    return 0

  def grad_workspace(self, with_bias):
    return 0

  def evaluate(self, *args):
    pass

  def dense(self):
    return self.is_dense

  def bias_per_row(self):
    return self.strides["bias"] != 0

  def evaluate_grad(self, at_now, *rest):
    names = ("logits", "num_options", "mask", "bias", "history", "repetition", "frequency", "presence", "temperature", "action", "entropy", "stats")
    _FakeRows.calls.append((dict(zip(names, at_now)), self.strides))


@pytest.fixture
def stand_in(monkeypatch):
  from envpool_amd import policy
  monkeypatch.setattr(policy, "_same_device", lambda dev, **tensors: None)
  monkeypatch.setattr(policy, "current_stream_handle", lambda dev: 0)
  _FakeRows.guard = staticmethod(policy._guard_capture)
  monkeypatch.setattr(policy, "_guard_capture", lambda *inputs: ())
  monkeypatch.setattr(policy, "_native", types.SimpleNamespace(Rows=_FakeRows))
  _FakeRows.calls = []
  return policy


def _operands(n, a):
  g = torch.Generator().manual_seed(0)
  return dict(num_options=torch.full((n,), a, dtype=torch.int32), mask=torch.ones(n, a, dtype=torch.bool), bias=torch.randn(n, a, generator=g).requires_grad_(),
              history=torch.randint(0, a, (n, 4), generator=g, dtype=torch.int32), repetition=torch.full((n,), 1.2), frequency=torch.zeros(n),
              presence=torch.zeros(n), temperature=torch.ones(n))


@pytest.mark.parametrize("layout", ["dense", "columns"])
def test_the_backward_pass_of_evaluate_reads_what_autograd_hands_back(stand_in, layout):
  """Under a hook for saved tensors (checkpoints and offloading are such hooks) the forward pass' own tensors may be gone:
  every address that the backward pass follows is that of a tensor that the hook gave back."""
  n, a = 3, 10
  kw = _operands(n, a)
  leaf = torch.randn(n, a).requires_grad_()
  logits = leaf if layout == "dense" else torch.randn(a, n).requires_grad_().t()
  given = []

  def unpack(packed):
    given.append(packed.clone())
    return given[-1]

  with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
    lp, ent = stand_in.evaluate(logits, torch.zeros(n, dtype=torch.int32), **kw)
  (lp.sum() + ent.sum()).backward()
  (at, strides), = _FakeRows.calls
  alive = {t.data_ptr() for t in given}
  assert all(ptr in alive for ptr in at.values()), {k: ptr in alive for k, ptr in at.items()}
  assert strides == {"logits": a, "mask": a, "bias": a, "history": 4}


def test_a_hook_may_hand_back_another_layout(stand_in):
  n, a = 3, 10
  kw = _operands(n, a)
  logits = torch.randn(n, a).requires_grad_()
  kw["mask"] = kw["mask"][:1].expand(n, a)  # one mask for all rows: comes back as a row each

  def unpack(packed):
    return packed.t().contiguous().t() if packed.dim() == 2 else packed.clone()

  with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
    lp, ent = stand_in.evaluate(logits, torch.zeros(n, dtype=torch.int32), **kw)
  (lp.sum() + ent.sum()).backward()
  (_, strides), = _FakeRows.calls
  assert strides == {"logits": a, "mask": a, "bias": a, "history": 4}
  # rows with gaps come back without them
  kw["mask"] = torch.ones(n, a + 6, dtype=torch.bool)[:, 2:a + 2]
  with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t.clone()):
    lp, ent = stand_in.evaluate(logits, torch.zeros(n, dtype=torch.int32), **kw)
  (lp.sum() + ent.sum()).backward()
  assert _FakeRows.calls[1][1] == {"logits": a, "mask": a, "bias": a, "history": 4}
  assert logits.grad.shape == (n, a) and kw["bias"].grad.shape == (n, a)


def test_dual_numbers_are_refused(stand_in):
  """Forward-mode derivatives: refused, where they were lost without a word (nothing here requires a gradient)."""
  import torch.autograd.forward_ad as fw
  x, act = torch.randn(3, 4), torch.zeros(3, dtype=torch.int32)
  with fw.dual_level():
    dual = lambda *shape: fw.make_dual(torch.randn(*shape), torch.randn(*shape))  # noqa: E731
    for kw in (dict(logits=dual(3, 4)), dict(logits=x, bias=dual(4)), dict(logits=x, temperature=dual(3)), dict(logits=dual(3, 4).requires_grad_())):
      with pytest.raises(ValueError, match="forward-mode"):
        stand_in.evaluate(action=act, **kw)
    stand_in.evaluate(x, act)
    q = torch.randn(5, 2, 1, 4)
    for i in range(3):
      qkv = [dual(5, 2, 1, 4) if i == j else q for j in range(3)]
      with pytest.raises(ValueError, match="forward-mode"):
        stand_in.memory_scan(*qkv, torch.zeros(1))
    with pytest.raises(ValueError, match="forward-mode.*state"):
      stand_in.memory_scan(q, q, q, torch.zeros(1), state=dual(2, 1, 4, 4))
    with pytest.raises(ValueError, match="forward-mode.*log_decay"):
      stand_in.memory_scan(q, q, q, dual(1))


@pytest.mark.parametrize("name", ["repetition", "frequency", "presence", "temperature"])
def test_per_row_numbers_that_require_a_gradient_are_refused(stand_in, name):
  """A learned temperature would be left without its gradient, in silence."""
  x, act = torch.randn(3, 4).requires_grad_(), torch.zeros(3, dtype=torch.int32)
  number = torch.ones(3).requires_grad_()
  with pytest.raises(ValueError, match=f"{name} is not differentiated"):
    stand_in.evaluate(x, act, **{name: number})
  stand_in.evaluate(x, act, **{name: number.detach()})
  with torch.no_grad():
    stand_in.evaluate(x, act, **{name: number})


def test_send_choice_tells_rows_without_options_from_rows_without_a_distribution():
  """-1 with log_prob 0 is an ended duel and sends 0; -1 with a NaN is a policy that has diverged, and sends nothing."""
  import numpy as np

  from envpool_amd.policy import Choice
  from envpool_amd.python.pool import EnvPoolFrontEnd

  class Pool(EnvPoolFrontEnd):
    last_env_ids = np.array([7, 3, 5], np.int32)

    def __init__(self):
      self.sent = []

    def send(self, action, env_id=None):
      self.sent.append((np.asarray(action).tolist(), np.asarray(env_id).tolist()))

  pool = Pool()
  action = torch.tensor([2, -1, 4], dtype=torch.int32)
  pool.send_choice(Choice(action, torch.tensor([-0.5, 0.0, -1.0]), torch.zeros(3)))
  assert pool.sent == [([2, 0, 4], [7, 3, 5])]
  with pytest.raises(RuntimeError, match="1 rows.*row 1, env 3"):
    pool.send_choice(Choice(action, torch.tensor([-0.5, float("nan"), -1.0]), torch.zeros(3)))
  assert len(pool.sent) == 1


def test_reset_leaves_envs_alone_that_it_was_not_asked_for(monkeypatch):
  """An id below the memory's first is not its last env; what 32 bits do not hold is not what they wrap to."""
  from envpool_amd import policy
  monkeypatch.setattr(policy, "_same_device", lambda dev, **tensors: None)
  monkeypatch.setattr(policy, "current_stream_handle", lambda dev: 0)
  seen = []

  class Native:
    def reset(self, rows, env_id, stream):
      import ctypes
      seen.append(list((ctypes.c_int32 * rows).from_address(env_id)) if rows else [])

  memory = object.__new__(policy.EnvMemory)
  memory.num_envs, memory.env_id_offset, memory.device, memory._native = 4, 10, torch.device("cpu"), Native()
  memory.state = torch.ones(4, 1, 2, 2)
  memory.reset(torch.tensor([9, 11], dtype=torch.int32))
  memory.reset(torch.tensor([2**32 + 11, 12, -2**40, 13]))
  memory.reset(torch.zeros(0, dtype=torch.int64))
  assert torch.equal(memory.state, torch.ones(4, 1, 2, 2))  # (the stand-in zeroes nothing)
  assert seen == [[9, 11], [14, 12, 9, 13], []]
  for bad in (torch.tensor([True, False]), torch.tensor([1.0]), torch.zeros(2, 2, dtype=torch.int32)):
    with pytest.raises(ValueError, match="whole numbers"):
      memory.reset(bad)
  memory.reset()
  assert not memory.state.any()


def test_resets_that_are_refused():
  import ctypes as C

  from envpool_amd import capi, capi_policy as cp
  L = cp.lib()
  ptr = 4096  # (never followed)

  def args(**kw):
    a = dict(device_id=0, num_envs=8, rows=4, heads=2, key_dim=16, value_dim=16, state=ptr, env_id=ptr)
    return cp.MemoryStepArgs(**dict(a, **kw))

  for bad, word in ((dict(num_envs=0), "num_envs"), (dict(rows=-1), "rows"), (dict(heads=0), "heads"), (dict(key_dim=257), "key_dim"), (dict(value_dim=0), "value_dim"),
                    (dict(rows=9, env_id=None), "without env_id"), (dict(state=None), "state"), (dict(env_id=ptr + 2), "aligned")):
    assert L.ep_memory_reset(C.byref(args(**bad))) == capi.EP_ERR_INVALID and word in L.ep_last_error().decode(), bad
  assert L.ep_memory_reset(None) == capi.EP_ERR_INVALID
  assert L.ep_memory_reset(C.byref(args(rows=0, state=None))) == capi.EP_OK
  if L.ep_device_count() == 0:
    assert L.ep_memory_reset(C.byref(args())) == capi.EP_ERR_NO_DEVICE


@pytest.mark.parametrize("name,bad", [("temperature", 1e39), ("temperature", 1e-39), ("temperature", 1e-300), ("repetition", 1e-46), ("repetition", 1e300),
                                      ("frequency", 1e39), ("presence", -1e39)])
def test_numbers_that_32_bits_do_not_hold_are_refused_by_evaluate(name, bad):
  """They would make every row one without a distribution. choose computes in 64 bits and takes them."""
  import ctypes as C

  from envpool_amd import capi, capi_policy as cp
  L, ptr = cp.lib(), 4096  # (never followed)
  rows = cp.PolicyRows(dtype=capi.EP_F32, rows=4, options=10, logits=ptr, logits_stride=10, repetition_all=1.0, temperature_all=1.0, history=ptr, history_len=3,
                       history_stride=3)
  setattr(rows, name + "_all", bad)
  r = C.byref(rows)
  for rc in (L.ep_policy_evaluate(r, ptr, ptr, ptr, ptr), L.ep_policy_evaluate_grad(r, ptr, ptr, ptr, ptr, ptr, ptr, 10, None, 0)):
    assert rc == capi.EP_ERR_INVALID and name in L.ep_last_error().decode()
  rows.rows = 0
  assert L.ep_policy_choose(r, None, 0, None, None, None) == capi.EP_OK
  setattr(rows, name, ptr)  # (one per row is on the device)
  assert L.ep_policy_evaluate(r, None, None, None, None) == capi.EP_OK


def test_the_guard_of_captures_sees_the_leaves_themselves(stand_in, monkeypatch):
  """Not the copies that are made of those whose rows have gaps: behind a copy the leaf's node would go unnoticed."""

  class Seen(Exception):
    pass

  def guard(*inputs):
    raise Seen(inputs)

  monkeypatch.setattr(stand_in, "_guard_capture", guard)
  leaf = torch.randn(5, 2, 4, 3).requires_grad_()
  state = torch.randn(2, 3, 4, 4)
  with pytest.raises(Seen) as e:
    stand_in.memory_scan(leaf.detach().transpose(2, 3).requires_grad_(), *(torch.randn(5, 2, 3, 4) for _ in range(2)), torch.zeros(3), state=state)
  assert all(t.is_leaf for t in e.value.args[0])
  logits, bias = torch.randn(6, 3).t().requires_grad_(), torch.randn(1, 6).expand(3, 6).requires_grad_()
  with pytest.raises(Seen) as e:
    stand_in.evaluate(logits, torch.zeros(3, dtype=torch.int32), bias=bias)
  assert e.value.args[0][0] is logits and e.value.args[0][1] is bias


def test_an_eager_call_in_another_thread_is_no_business_of_a_capture(monkeypatch):
  """Two calls over one leaf in one capture, while another thread works without one."""
  import threading

  from envpool_amd import policy
  capturing = threading.local()
  monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: getattr(capturing, "yes", False))
  leaf, other = torch.zeros(3).requires_grad_(), torch.zeros(3).requires_grad_()
  capturing.yes = True
  first = policy._guard_capture(leaf)
  recorded = leaf * 2  # (the first call's graph holds the leaf's node)
  thread = threading.Thread(target=lambda: policy._guard_capture(other))
  thread.start()
  thread.join()
  policy._guard_capture(leaf)
  del first, recorded
  # a graph recorded outside the capture is still found
  capturing.yes = False
  policy._guard_capture(leaf)
  living = leaf * 2
  capturing.yes = True
  with pytest.raises(RuntimeError, match="recorded outside this capture"):
    policy._guard_capture(leaf)
  del living
  assert len(policy._guard_capture(leaf)) == 1


def test_copies_of_a_call_do_not_count_as_holders_of_its_leaves(stand_in, monkeypatch):
  """Inside a capture: leaves whose rows have gaps, or are one row expanded, and no graph outside."""
  monkeypatch.setattr(stand_in, "_guard_capture", _FakeRows.guard)
  monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
  act = torch.zeros(3, dtype=torch.int32)
  for bias in (None, torch.randn(1, 6).expand(3, 6), torch.randn(6, 3).t(), torch.randn(12)[::2]):
    stand_in._capture.token = None
    logits = torch.randn(6, 3).t().requires_grad_()
    bias = None if bias is None else bias.requires_grad_()
    lp, ent = stand_in.evaluate(logits, act, bias=bias)
    (lp.sum() + ent.sum()).backward()
    assert logits.grad.shape == (3, 6) and (bias is None or bias.grad.shape == bias.shape)
  stand_in._capture.token = None


@pytest.mark.parametrize("where", ["last", "decay"])
def test_the_backward_pass_of_a_scan_takes_any_layout(stand_in, monkeypatch, where):
  """The kernels read rows whose last dimension is dense, and a dense log_decay: whatever a hook hands back."""
  scans = []

  class Scan:
    def __init__(self, dev, dtype, steps, rows, heads, key_dim, value_dim, log_decay, *rest):
      self.decay, self.seen = log_decay, {}
      scans.append(self)

    def operands(self, q, qs, qg, k, ks, kg, v, vs, vg):
      self.seen = {q: qs, k: ks, v: vs}

    def workspace(self):
      return 0

    output = states = direction = run = lambda self, *args: None

  monkeypatch.setattr(stand_in, "_native", types.SimpleNamespace(Scan=Scan, scan_pair_workspace=lambda x, y: 0, scan_pair=lambda x, y, ws, n: None))
  q, k, v = (torch.randn(5, 2, 3, 4).requires_grad_() for _ in range(3))
  handed = []

  def unpack(t):
    if where == "last" and t.dim() == 4:
      t = t.transpose(2, 3).contiguous().transpose(2, 3)
    if where == "decay" and t.dim() == 1:
      t = torch.stack([t, t], 1)[:, 0]
    handed.append(t)
    return t

  with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
    out, final = stand_in.memory_scan(q, k, v, torch.zeros(3))
  del scans[:]
  (out.sum() + final.sum()).backward()
  gaps = {t.data_ptr() for t in handed if t.stride(-1) != 1}
  assert gaps and len(scans) == 3
  for s in scans:
    assert s.decay not in gaps and not gaps & set(s.seen), where
