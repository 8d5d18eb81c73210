"""What a policy on the GPU needs next to the pools, as torch calls over include/envpool_amd_policy.h:

* `choose` / `evaluate`: the action to send back, from logits under the pool's legal-action mask
  (`info["num_options"]`, `info["action_mask"]`), with biases and penalties for what was chosen before; and
  for training the log-probability and entropy of stored actions, differentiable in the logits and biases.
* `EnvMemory` / `memory_scan`: a linear-attention memory with one decay per head whose state belongs to an
  env. `EnvMemory.step` moves the rows of a batch one step on (by `env_id`, in whatever order the batch
  has), `memory_scan` runs a whole rollout segment `[T, B, ...]` with episode boundaries inside and is
  differentiable.

Everything is enqueued on torch's current stream of the tensors' device; nothing is copied to the host or
waited for, and the calls can be captured into a graph. Tensors that are views of a pool's ring are
overwritten when the ring comes round: clone what a later backward pass needs.

The reference has no counterpart (its policies see numpy arrays, envpool2/python/envpool.py:135-142)."""
import math
import threading
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from ._loader import load_library

load_library()  # fail loudly before the extension tries to resolve its symbols

from . import policy_native as _native  # noqa: E402
from .python.streamstep import current_stream_handle  # noqa: E402

_FLOATS = {torch.float32: _native.F32, torch.float16: _native.F16, torch.bfloat16: _native.BF16}
_MASKS = {torch.bool: _native.BOOL, torch.uint8: _native.U8, torch.int32: _native.I32}


class Choice(NamedTuple):
  """`action` int32 `[B]` (-1: nothing to choose), `log_prob` and `entropy` float32 `[B]`."""
  action: torch.Tensor
  log_prob: torch.Tensor
  entropy: torch.Tensor


def _same_device(dev, **tensors):
  if dev.type != "cuda":
    raise ValueError(f"the tensors must be on a GPU, not on {dev}")
  for name, t in tensors.items():
    if t is not None and t.device != dev:
      raise ValueError(f"{name} is on {t.device}, the others on {dev}")


def _no_tangents(call, **tensors):
  """Forward-mode derivatives have no formula here: a dual number is refused rather than stripped of its tangent."""
  if forward_ad._current_level < 0:
    return
  for name, t in tensors.items():
    if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
      raise ValueError(f"{call} has no forward-mode derivative: {name} is a dual number")


def _row_operand(t, name, rows, cols):
  """A `[cols]`, `[1, cols]` or `[rows, cols]` tensor -> (tensor, stride from row to row, 0: shared)."""
  if t.dim() == 1 and t.shape[0] == cols:
    return (t if t.stride(0) == 1 or cols == 1 else t.detach().contiguous()), 0
  if t.dim() != 2 or t.shape[1] != cols or t.shape[0] not in (1, rows):
    raise ValueError(f"{name} must be [{cols}] or [{rows}, {cols}], got {list(t.shape)}")
  if (cols > 1 and t.stride(1) != 1) or 0 < t.stride(0) < cols:
    t = t.detach().contiguous()
  return t, 0 if t.shape[0] == 1 and rows != 1 else t.stride(0)


def _penalty(v, name, rows):
  """A number, or a float32 `[rows]` tensor -> (tensor or None, the number)."""
  if isinstance(v, torch.Tensor):
    if v.dtype != torch.float32 or v.shape != (rows,):
      raise ValueError(f"{name} must be a number or a float32 tensor [{rows}], got {v.dtype} {list(v.shape)}")
    if v.requires_grad and torch.is_grad_enabled():
      raise ValueError(f"{name} is not differentiated: pass {name}.detach()")
    return v, 1.0
  return None, float(v)


class _Prepared:
  """The checked operands of one call: tensors as the kernels read them, the numbers beside them, and the native struct."""
  __slots__ = ("tensors", "numbers", "native", "dev", "n")


# the operands in `_Prepared.tensors`: logits, num_options, mask, bias, history, repetition, frequency, presence, temperature
_BIAS, _SLOTS = 3, 9


def _dense(t):
  return t if t is None or t.is_contiguous() else t.contiguous()


def _bind(p):
  """Lays `p.tensors` (of checked types and shapes) out as the kernels read them and fills `p.native` with where they are
  now. The backward pass does it anew where what autograd hands back is laid out otherwise than what was saved. (Copies
  are no part of the graph: the gradients are those of the originals, and _guard_capture must not find a leaf held by them.)"""
  logits, num_options, mask, bias, history, *per_row = p.tensors
  n, a = logits.shape
  if (a > 1 and logits.stride(1) != 1) or (n > 1 and logits.stride(0) < a):
    logits = logits.detach().contiguous()
  if num_options is not None and not num_options.is_contiguous():
    num_options = num_options.contiguous()
  mask_ptr = mask_dt = mask_stride = bias_ptr = bias_dt = bias_stride = hist_ptr = hist_len = hist_stride = 0
  if mask is not None:
    mask, mask_stride = _row_operand(mask, "mask", n, (a + 31) // 32 if mask.dtype == torch.int32 else a)
    mask_ptr, mask_dt = mask.data_ptr(), _MASKS[mask.dtype]
  if bias is not None:
    bias, bias_stride = _row_operand(bias, "bias", n, a)
    bias_ptr, bias_dt = bias.data_ptr(), _FLOATS[bias.dtype]
  if history is not None:
    hist_len = history.shape[-1]
    if hist_len > 0:
      history, hist_stride = _row_operand(history, "history", n, hist_len)
      hist_ptr = history.data_ptr()
  rep, freq, pres, temp = per_row = [t if t is None or t.is_contiguous() else t.contiguous() for t in per_row]
  _same_device(p.dev, num_options=num_options, mask=mask, bias=bias, history=history, repetition=rep, frequency=freq, presence=pres, temperature=temp)
  rep_all, freq_all, pres_all, temp_all = p.numbers
  p.tensors = (logits, num_options, mask, bias, history, *per_row)
  p.native = _native.Rows(p.dev.index, _FLOATS[logits.dtype], n, a, logits.data_ptr(), logits.stride(0), 0 if num_options is None else num_options.data_ptr(),
                          mask_ptr, mask_dt, mask_stride, bias_ptr, bias_dt, bias_stride, hist_ptr, hist_len, hist_stride, 0 if rep is None else rep.data_ptr(),
                          rep_all, 0 if freq is None else freq.data_ptr(), freq_all, 0 if pres is None else pres.data_ptr(), pres_all,
                          0 if temp is None else temp.data_ptr(), temp_all, current_stream_handle(p.dev))


def _prepare(logits, num_options, mask, bias, history, repetition, frequency, presence, temperature):
  if logits.dim() != 2 or logits.dtype not in _FLOATS or logits.shape[1] < 1:
    raise ValueError(f"logits must be float32, float16 or bfloat16 [rows, options >= 1], got {logits.dtype} {list(logits.shape)}")
  n, dev = logits.shape[0], logits.device
  if num_options is not None and (num_options.dtype != torch.int32 or num_options.shape != (n,)):
    raise ValueError(f"num_options must be int32 [{n}], got {num_options.dtype} {list(num_options.shape)}")
  if mask is not None and mask.dtype not in _MASKS:
    raise ValueError(f"mask must be bool or uint8 (one per option) or int32 (32 options a word), got {mask.dtype}")
  if bias is not None and bias.dtype != torch.float32 and bias.dtype != logits.dtype:
    raise ValueError(f"bias must be float32 or of the logits' type, got {bias.dtype}")
  if history is not None and (history.dtype != torch.int32 or history.dim() not in (1, 2)):
    raise ValueError(f"history must be int32 [{n}, length] or [length], got {history.dtype} {list(history.shape)}")
  rep, rep_all = _penalty(repetition, "repetition", n)
  freq, freq_all = _penalty(frequency, "frequency", n)
  pres, pres_all = _penalty(presence, "presence", n)
  temp, temp_all = _penalty(temperature, "temperature", n)
  for name, t, v, low in (("temperature", temp, temp_all, 0.0), ("repetition", rep, rep_all, 0.0), ("frequency", freq, freq_all, -math.inf),
                          ("presence", pres, pres_all, -math.inf)):
    if t is None and not low < v < math.inf:
      raise ValueError(f"{name} = {v} is not a {'positive ' if low == 0.0 else ''}number")
  p = _Prepared()
  p.dev, p.n = dev, n
  p.tensors = (logits, num_options, mask, bias, history, rep, freq, pres, temp)
  p.numbers = (rep_all, freq_all, pres_all, temp_all)
  _bind(p)
  return p


def _scratch(nbytes, dev):
  """-> (tensor that holds the memory, address, bytes) of a call's workspace."""
  if nbytes == 0:
    return None, 0, 0
  t = torch.empty(nbytes, dtype=torch.uint8, device=dev)
  return t, t.data_ptr(), nbytes


def choose(logits, u=None, *, num_options=None, mask=None, bias=None, history=None, repetition=1.0, frequency=0.0, presence=0.0,
           temperature=1.0) -> Choice:
  """The action of every row from its `logits` `[B, A]` (float32, float16 or bfloat16).

  Legal are the options below `num_options` (int32 `[B]`, e.g. `info["num_options"]`) that `mask` allows:
  bool / uint8 `[B, A]` (e.g. `info["action_mask"]`) or int32 words of 32 options `[B, ceil(A / 32)]`; either may
  be None, and a mask of one row serves all. `history` int32 `[B, L]` holds options chosen before (-1: none): one
  that stands there c > 0 times has its logit divided by `repetition` (multiplied, if it is not positive) and
  lowered by `frequency * c + presence`. `bias` (`[A]` or `[B, A]`, float32 or the logits' type) is added, then all
  is divided by `temperature`. The four numbers may be float32 tensors `[B]`.

  `u` (`[B]`, float32 or float64, in [0, 1)): the option where the cumulated probability first exceeds it.
  None: the most probable option, the lowest of equals. Returns a `Choice` (no gradients: `evaluate` has them); a row
  without a legal option gets action -1, log_prob 0 and entropy 0, a row with a NaN or +inf among its legal options -1,
  NaN and NaN."""
  with torch.no_grad():
    p = _prepare(logits, num_options, mask, bias, history, repetition, frequency, presence, temperature)
    u_ptr = u_dt = 0
    if u is not None:
      if u.dtype not in (torch.float32, torch.float64) or u.shape != (p.n,):
        raise ValueError(f"u must be float32 or float64 [{p.n}], got {u.dtype} {list(u.shape)}")
      _same_device(p.dev, u=u)
      if not u.is_contiguous():
        u = u.contiguous()
      u_ptr, u_dt = u.data_ptr(), _native.F64 if u.dtype == torch.float64 else _native.F32
    action = torch.empty(p.n, dtype=torch.int32, device=p.dev)
    log_prob = torch.empty(p.n, dtype=torch.float32, device=p.dev)
    entropy = torch.empty(p.n, dtype=torch.float32, device=p.dev)
    ws, ws_ptr, ws_bytes = _scratch(p.native.choose_workspace(), p.dev)
    p.native.choose(u_ptr, u_dt, action.data_ptr(), log_prob.data_ptr(), entropy.data_ptr(), ws_ptr, ws_bytes)
    return Choice(action, log_prob, entropy)


_capture = threading.local()  # .token: lasts from a capture's first differentiable call to the thread's next eager one


def _guard_capture(*inputs):
  """Refuses a differentiable call inside a graph capture where a leaf among its inputs is still part of a graph
  recorded outside it: torch would make that graph's stream wait inside the capture, which ends the process
  when the capture ends. (Whether somebody holds a leaf's accumulation node shows in a mark left on it: with no
  other holder the node goes, and the mark with it. Any holder counts: a wrapper that keeps the nodes of a module's
  parameters, to reduce their gradients, has them refused as well, since on which stream a node was made cannot be asked.)
  Returns the nodes, to be held until the call is recorded."""
  if not torch.cuda.is_current_stream_capturing():
    _capture.token = None
    return ()
  token = getattr(_capture, "token", None)
  if token is None:
    token = _capture.token = object()
  nodes = []
  for t in inputs:
    if t is None or not t.requires_grad or not t.is_leaf:
      continue
    node = torch.autograd.graph.get_gradient_edge(t).node
    if node.metadata.get("envpool_amd_capture") is token:
      continue
    node.metadata["envpool_amd_probe"] = True
    del node
    node = torch.autograd.graph.get_gradient_edge(t).node
    if "envpool_amd_probe" in node.metadata:
      del node.metadata["envpool_amd_probe"]
      raise RuntimeError("graph capture: a leaf input still belongs to an autograd graph recorded outside this capture; "
                         "drop that graph (its outputs), or what else holds the leaf's accumulation node, before capturing, or capture over other leaves")
    node.metadata["envpool_amd_capture"] = token
    nodes.append(node)
  return nodes


def _run_backward(plain, once, ctx, *grads):
  """A backward pass whose results are not differentiable again: torch's wrapper that says so costs more than
  a small pass and is only needed where a graph of the backward pass is asked for."""
  return once(ctx, *grads) if torch.is_grad_enabled() else plain(ctx, *grads)


def _evaluate_forward(p, action):
  log_prob = torch.empty(p.n, dtype=torch.float32, device=p.dev)
  entropy = torch.empty(p.n, dtype=torch.float32, device=p.dev)
  stats = torch.empty(2 * p.n, dtype=torch.float32, device=p.dev)
  ws, ws_ptr, ws_bytes = _scratch(p.native.evaluate_workspace(), p.dev)
  p.native.evaluate(action.data_ptr(), log_prob.data_ptr(), entropy.data_ptr(), stats.data_ptr(), ws_ptr, ws_bytes)
  return log_prob, entropy, stats


def _evaluate_backward(ctx, g_lp, g_h):
  saved = ctx.saved_tensors
  want_x, want_b = ctx.needs_input_grad[:2]
  if g_lp is None and g_h is None:
    return None, None, None, None
  native, dev, where, bias_like, numbers = ctx.call
  at, same = [], native.dense()
  for t in saved:
    if t is None:
      at.append(0)
      continue
    at.append(t.data_ptr())
    if t.get_device() != where:
      raise ValueError(f"a saved tensor came back on {t.device}, the others on {dev}")
    same = same and t.is_contiguous()
  if not same:  # rows with gaps, or a hook handed back another layout
    p = _Prepared()
    p.tensors, p.numbers, p.dev = list(saved[:_SLOTS]), numbers, dev
    if want_b and len(bias_like[0]) == 2 and bias_like[0][0] > 1:  # its gradient is one per row
      p.tensors[_BIAS] = _dense(p.tensors[_BIAS])
    _bind(p)
    native, saved = p.native, (*p.tensors, *(_dense(t) for t in saved[_SLOTS:]))
    at = [0 if t is None else t.data_ptr() for t in saved]
  logits = saved[0]
  n, a = logits.shape
  if g_lp is not None and not g_lp.is_contiguous():
    g_lp = g_lp.contiguous()
  if g_h is not None and not g_h.is_contiguous():
    g_h = g_h.contiguous()
  grad_x = torch.empty((n, a), dtype=logits.dtype, device=dev) if want_x else None
  grad_b, stride = None, 0
  if want_b:
    stride = a if native.bias_per_row() else 0
    grad_b = torch.empty((n, a) if stride else (a,), dtype=bias_like[1], device=dev)
  ws, ws_ptr, ws_bytes = _scratch(native.grad_workspace(want_b), dev)
  native.evaluate_grad(at, 0 if g_lp is None else g_lp.data_ptr(), 0 if g_h is None else g_h.data_ptr(), 0 if grad_x is None else grad_x.data_ptr(), a,
                       0 if grad_b is None else grad_b.data_ptr(), stride, ws_ptr, ws_bytes, current_stream_handle(dev))
  return grad_x, None if grad_b is None else grad_b.view(bias_like[0]), None, None


_evaluate_backward_once = torch.autograd.function.once_differentiable(_evaluate_backward)


class _Evaluate(torch.autograd.Function):

  @staticmethod
  def forward(ctx, logits, bias, action, p):
    log_prob, entropy, stats = _evaluate_forward(p, action)
    ctx.set_materialize_grads(False)
    # every tensor that the backward pass reads is saved, so that torch notices one that was changed in place, hands it
    # to its hooks (offloading, checkpoints) and frees it after. The native struct stays for its sizes; the backward
    # pass puts the addresses of what it is handed in place of the forward pass'
    ctx.save_for_backward(*p.tensors, action, entropy, stats)
    ctx.call = (p.native, p.dev, action.get_device(), None if bias is None else (bias.shape, bias.dtype), p.numbers)
    return log_prob, entropy

  @staticmethod
  def backward(ctx, g_lp, g_h):
    return _run_backward(_evaluate_backward, _evaluate_backward_once, ctx, g_lp, g_h)


def evaluate(logits, action, *, num_options=None, mask=None, bias=None, history=None, repetition=1.0, frequency=0.0, presence=0.0, temperature=1.0):
  """(log_prob, entropy), float32 `[B]` each, of stored actions under the distribution that `choose`
  describes, differentiable in `logits` and `bias` (once, backwards: dual numbers are refused, and so are per-row
  numbers that require a gradient).

  `action` int32 `[B]`: -1 (what `choose` gives a row with nothing to choose) has log_prob 0 and no gradient, an
  illegal option -inf, a value outside [-1, A) NaN. The statistics of a row and the gradients' sums are kept in
  32 bits; gradients come in the type of the tensor they belong to."""
  _no_tangents("evaluate", logits=logits, bias=bias, repetition=repetition, frequency=frequency, presence=presence, temperature=temperature)
  differentiable = torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad))
  p = _prepare(logits, num_options, mask, bias, history, repetition, frequency, presence, temperature)
  if action.dtype != torch.int32 or action.shape != (p.n,):
    raise ValueError(f"action must be int32 [{p.n}], got {action.dtype} {list(action.shape)}")
  _same_device(p.dev, action=action)
  if not action.is_contiguous():
    action = action.contiguous()
  if differentiable:
    nodes = _guard_capture(logits, bias)  # noqa: F841
    if bias is not None and bias.requires_grad and bias.dim() == 2 and bias.shape[0] > 1 and bias.stride(0) == 0:
      bias = _dense(bias)  # one row of biases expanded by the caller: its gradient is one per row
      p.tensors = (*p.tensors[:_BIAS], bias, *p.tensors[_BIAS + 1:])
      _bind(p)
    return _Evaluate.apply(logits, bias, action, p)
  return _evaluate_forward(p, action)[:2]


# ---- memory --------------------------------------------------------------------------------------
def _dense_last(t):
  return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


_error_pages, _error_lock = [], threading.Lock()


def _error_word():
  """A pinned word for a memory's kernels to flag an error in. Never freed: a step that is still under way when its memory
  is dropped must not write into what somebody else has been given meanwhile."""
  with _error_lock:
    if not _error_pages or _error_pages[-1][1] == 1024:
      _error_pages.append([torch.zeros(1024, dtype=torch.int32, pin_memory=True), 0])
    page, used = _error_pages[-1]
    _error_pages[-1][1] += 1
  return page[used:used + 1]


class EnvMemory:
  """The memory of a policy over the envs of a pool: per env and head a state `[key_dim, value_dim]` in
  float32, S <- exp(log_decay[head]) S + k^T v, out = scale * q S, zeroed where an episode starts.

  `log_decay` float32 `[num_heads]` on the GPU, values <= 0 (not differentiated). `state`: an existing
  `[num_envs, num_heads, key_dim, value_dim]` float32 tensor to work on (dense); made, all zero, when None.
  Dimensions 1 to 256 (`memory_scan`, and so training, 1 to 128). Steps of one memory are ordered by the caller (one
  stream). A step changes `state` in place, and autograd is told so: a `memory_scan` that starts from it and is
  differentiated after another step needs a copy (`memory.state.clone()`), without one its backward pass raises.
  (Replays of a captured step go unnoticed.)"""

  def __init__(self, num_envs: int, num_heads: int, key_dim: int, value_dim: int, log_decay: torch.Tensor, *, state: Optional[torch.Tensor] = None,
               env_id_offset: int = 0):
    if num_envs < 1 or num_heads < 1:
      raise ValueError(f"num_envs = {num_envs}, num_heads = {num_heads}")
    if not (1 <= key_dim <= 256 and 1 <= value_dim <= 256):
      raise ValueError(f"key_dim = {key_dim}, value_dim = {value_dim}: not both in [1, 256]")
    if log_decay.dtype != torch.float32 or log_decay.shape != (num_heads,):
      raise ValueError(f"log_decay must be float32 [{num_heads}], got {log_decay.dtype} {list(log_decay.shape)}")
    shape = (num_envs, num_heads, key_dim, value_dim)
    if state is not None and (state.dtype != torch.float32 or tuple(state.shape) != shape or not state.is_contiguous()):
      raise ValueError(f"state must be a contiguous float32 tensor {list(shape)}, got {state.dtype} {list(state.shape)}")
    dev = log_decay.device
    _same_device(dev, state=state)
    self.num_envs, self.num_heads, self.key_dim, self.value_dim = shape
    self.env_id_offset, self.device = env_id_offset, dev
    self.log_decay = log_decay.detach().contiguous()
    self.state = torch.zeros(shape, dtype=torch.float32, device=dev) if state is None else state.detach()
    self._error = _error_word()  # set by a kernel: an env id out of range
    self._error_np = self._error.numpy()
    self._native = _native.Step(dev.index, num_envs, num_heads, key_dim, value_dim, self.log_decay.data_ptr(), self.state.data_ptr(), env_id_offset,
                                self._error.data_ptr())

  def poll_errors(self) -> None:
    """Raises if a step or a reset so far named an env that is not in the memory. Never waits: what a running kernel has
    yet to flag is seen by a later call (every `step` polls first)."""
    if self._error_np[0]:
      self._error_np[0] = 0
      raise RuntimeError(f"EnvMemory: an earlier step or reset named an env id outside [{self.env_id_offset}, {self.env_id_offset + self.num_envs})")

  def reset(self, env_id: Optional[torch.Tensor] = None) -> None:
    """Zeroes the state of the envs in `env_id` (whole numbers `[n]`; all envs if None). An id outside the memory touches
    nothing and is reported by a later step, as a step's own are."""
    if env_id is None:
      self.state.zero_()
      return
    if env_id.dim() > 1 or env_id.dtype == torch.bool or env_id.is_floating_point() or env_id.is_complex():
      raise ValueError(f"env_id must be whole numbers [n], got {env_id.dtype} {list(env_id.shape)}")
    _same_device(self.device, env_id=env_id)
    with torch.no_grad():
      if env_id.dtype != torch.int32:  # (what 32 bits do not hold is outside)
        env_id = env_id.long().clamp(self.env_id_offset - 1, self.env_id_offset + self.num_envs).int()
      env_id = _dense(env_id)
      self._native.reset(env_id.numel(), env_id.data_ptr(), current_stream_handle(self.device))
      torch.autograd.graph.increment_version(self.state)

  def step(self, q, k, v, *, env_id=None, fresh=None, elapsed_step=None, scale: Optional[float] = None) -> torch.Tensor:
    """One step of the rows of a batch: `q` `[B, num_heads, key_dim]`, `k` `[B, kv_heads, key_dim]`, `v`
    `[B, kv_heads, value_dim]` (one float type; `kv_heads` divides `num_heads`) -> `[B, num_heads, value_dim]`.

    `env_id` int32 `[B]`: the env of each row (`info["env_id"]`); None: row i is env i. An env named several times
    is stepped several times, in row order; an id outside the memory gives NaN and an error at a later call.
    `elapsed_step` int32 `[B]` (`info["elapsed_step"]`): rows where it is 0 start from an empty state; or say so with
    `fresh` bool / uint8 `[B]`. `scale` defaults to key_dim ** -0.5. No gradient: training runs `memory_scan`."""
    self.poll_errors()
    dt = _FLOATS.get(q.dtype)
    if dt is None or k.dtype != q.dtype or v.dtype != q.dtype:
      raise ValueError(f"q, k, v must be of one type, float32, float16 or bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.dim() != 3 or q.shape[1] != self.num_heads or q.shape[2] != self.key_dim:
      raise ValueError(f"q must be [rows, {self.num_heads}, {self.key_dim}], got {list(q.shape)}")
    n = q.shape[0]
    if k.dim() != 3 or v.dim() != 3 or k.shape[0] != n or v.shape[:2] != k.shape[:2] or k.shape[2] != self.key_dim or v.shape[2] != self.value_dim:
      raise ValueError(f"k, v must be [{n}, kv_heads, {self.key_dim}] and [{n}, kv_heads, {self.value_dim}], got {list(k.shape)} and {list(v.shape)}")
    if k.shape[1] < 1 or self.num_heads % k.shape[1]:
      raise ValueError(f"kv_heads = {k.shape[1]} does not divide num_heads = {self.num_heads}")
    if env_id is None:
      if n > self.num_envs:
        raise ValueError(f"{n} rows for {self.num_envs} envs without env_id")
    elif env_id.dtype != torch.int32 or env_id.shape != (n,):
      raise ValueError(f"env_id must be int32 [{n}], got {env_id.dtype} {list(env_id.shape)}")
    if fresh is not None and elapsed_step is not None:
      raise ValueError("give fresh or elapsed_step, not both")
    if fresh is not None and (fresh.dtype not in (torch.bool, torch.uint8) or fresh.shape != (n,)):
      raise ValueError(f"fresh must be bool or uint8 [{n}], got {fresh.dtype} {list(fresh.shape)}")
    if elapsed_step is not None and (elapsed_step.dtype != torch.int32 or elapsed_step.shape != (n,)):
      raise ValueError(f"elapsed_step must be int32 [{n}], got {elapsed_step.dtype} {list(elapsed_step.shape)}")
    first = fresh if fresh is not None else elapsed_step
    dev = self.device
    _same_device(dev, q=q, k=k, v=v, env_id=env_id, fresh=first)
    with torch.no_grad():
      q, k, v = _dense_last(q), _dense_last(k), _dense_last(v)
      if env_id is not None and not env_id.is_contiguous():
        env_id = env_id.contiguous()
      if first is not None and not first.is_contiguous():
        first = first.contiguous()
      out = torch.empty(n, self.num_heads, self.value_dim, dtype=q.dtype, device=dev)
      ws, ws_ptr, ws_bytes = _scratch(self._native.workspace(n, env_id is not None), dev)
      self._native.run(dt, n, k.shape[1], q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                       v.stride(1), out.data_ptr(), out.stride(0), out.stride(1), 0 if env_id is None else env_id.data_ptr(),
                       0 if first is None else first.data_ptr(), _MASKS[first.dtype] if first is not None else 0,
                       self.key_dim ** -0.5 if scale is None else float(scale), ws_ptr, ws_bytes, current_stream_handle(dev))
      torch.autograd.graph.increment_version(self.state)  # (the kernel's writes are an in-place operation)
    return out


_NO_STRIDE = (0, 0, 0, 0)


def _turned(stride):
  return (stride[0], stride[1], stride[3], stride[2])


def _scan_args(dims, log_decay, fresh, q, q_group, k, k_group, v, v_group, out, state_in, state_out, inc_scale, out_scale, reverse, turn):
  """The arguments of one ep_memory_scan. `dims` (steps, rows, heads, key_dim, value_dim); `turn`: the states are stored as
  [value_dim, key_dim] of this call."""
  dev = log_decay.device
  f = (0, 0, 0) if fresh is None else (fresh.data_ptr(), *fresh.stride())
  s = _native.Scan(dev.index, _FLOATS[q.dtype], *dims, log_decay.data_ptr(), *f, current_stream_handle(dev))
  s.operands(q.data_ptr(), q.stride()[:3], q_group, k.data_ptr(), k.stride()[:3], k_group, v.data_ptr(), v.stride()[:3], v_group)
  if out is not None:
    s.output(out.data_ptr(), out.stride()[:3], _FLOATS[out.dtype])
  stride_of = lambda t: _NO_STRIDE if t is None else _turned(t.stride()) if turn else t.stride()  # noqa: E731
  s.states(0 if state_in is None else state_in.data_ptr(), stride_of(state_in), 0 if state_out is None else state_out.data_ptr(), stride_of(state_out))
  s.direction(inc_scale, out_scale, reverse)
  return s


def _scan_call(*args):
  s = _scan_args(*args)
  ws, ws_ptr, ws_bytes = _scratch(s.workspace(), args[1].device)
  s.run(ws_ptr, ws_bytes)


def _scan_forward(q, k, v, state, log_decay, fresh, scale):
  t, n, h, dk = q.shape
  dv, group = v.shape[3], h // k.shape[2]
  out = torch.empty(t, n, h, dv, dtype=q.dtype, device=q.device)
  final = torch.empty(n, h, dk, dv, dtype=torch.float32, device=q.device)
  _scan_call((t, n, h, dk, dv), log_decay, fresh, q, 1, k, group, v, group, out, state, final, 1.0, scale, False, False)
  return out, final


def _scan_backward(ctx, g_out, g_final):
  q, k, v, state, log_decay, fresh = ctx.saved_tensors
  # (a hook for saved tensors may hand back another layout)
  q, k, v, log_decay = _dense_last(q), _dense_last(k), _dense_last(v), _dense(log_decay)
  _same_device(ctx.dev, q=q, k=k, v=v, state=state, log_decay=log_decay, fresh=fresh)
  t, n, h, dk = q.shape
  dv, hk = v.shape[3], k.shape[2]
  group, scale = h // hk, ctx.scale
  if g_out is None and g_final is None:
    return (None,) * 7
  g_out = torch.zeros(t, n, h, dv, dtype=q.dtype, device=q.device) if g_out is None else _dense_last(g_out)
  want_q, want_k, want_v, want_s = ctx.needs_input_grad[:4]
  grad_q = grad_k = grad_v = grad_s = None
  if want_q:
    grad_q = torch.empty(t, n, h, dk, dtype=q.dtype, device=q.device)
    _scan_call((t, n, h, dv, dk), log_decay, fresh, g_out, 1, v, group, k, group, grad_q, state, None, 1.0, scale, False, True)

  def per_head(dim):  # heads that share keys and values: their gradients in 32 bits first, then summed
    return torch.empty(t, n, h, dim, dtype=q.dtype if group == 1 else torch.float32, device=q.device)

  def summed(x, dim):
    if group == 1:
      return x
    y = torch.empty(t, n, hk, dim, dtype=q.dtype, device=q.device)
    _native.sum_heads(q.device.index, x.data_ptr(), t * n, hk, group, dim, y.data_ptr(), _FLOATS[q.dtype], current_stream_handle(q.device))
    return y

  for_k = for_v = None
  if want_k:
    grad_k = per_head(dk)
    for_k = ((t, n, h, dv, dk), log_decay, fresh, v, group, g_out, 1, q, 1, grad_k, g_final, None, scale, 1.0, True, True)
  if want_v or want_s:
    grad_v = per_head(dv) if want_v else None
    grad_s = torch.empty(n, h, dk, dv, dtype=torch.float32, device=q.device) if want_s else None
    for_v = ((t, n, h, dk, dv), log_decay, fresh, k, group, q, 1, g_out, 1, grad_v, g_final, grad_s, scale, 1.0, True, False)
  if for_k and for_v:
    x, y = _scan_args(*for_v), _scan_args(*for_k)
    ws, ws_ptr, ws_bytes = _scratch(_native.scan_pair_workspace(x, y), q.device)
    _native.scan_pair(x, y, ws_ptr, ws_bytes)
  elif for_k or for_v:
    _scan_call(*(for_k or for_v))
  grad_k = summed(grad_k, dk) if want_k else None
  grad_v = summed(grad_v, dv) if want_v else None
  return grad_q, grad_k, grad_v, grad_s, None, None, None


_scan_backward_once = torch.autograd.function.once_differentiable(_scan_backward)


class _MemoryScan(torch.autograd.Function):

  @staticmethod
  def forward(ctx, q, k, v, state, log_decay, fresh, scale):
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(q, k, v, state, log_decay, fresh)
    ctx.scale, ctx.dev = scale, q.device
    return _scan_forward(q, k, v, state, log_decay, fresh, scale)

  @staticmethod
  def backward(ctx, g_out, g_final):
    return _run_backward(_scan_backward, _scan_backward_once, ctx, g_out, g_final)


def memory_scan(q, k, v, log_decay, *, fresh=None, state=None, scale: Optional[float] = None):
  """`EnvMemory.step` over a whole segment: `q` `[T, B, H, key_dim]`, `k` `[T, B, kv_heads, key_dim]`, `v`
  `[T, B, kv_heads, value_dim]` of one float type, time first as a rollout has it (any strides) -> (out
  `[T, B, H, value_dim]`, final state float32 `[B, H, key_dim, value_dim]`).

  `log_decay` float32 `[H]`, values <= 0, not differentiated. `fresh` bool / uint8 `[T, B]`: steps at which an
  episode starts, so that nothing from before reaches them (None: no such step). `state` float32
  `[B, H, key_dim, value_dim]`: where the rows start (None: zero). Dimensions 1 to 128 (`EnvMemory` acts with up to
  256). What is not finite goes where the recurrence takes it: to later steps of its episode, in the gradients to earlier.
  Differentiable (once, backwards: dual numbers are refused) in q, k, v and state; gradients come in the type of the tensor they belong to. States and sums
  are kept in 32 bits. As operands of 16-bit products the states and the scores of a chunk enter as two pieces of the type
  (16 bits together in bfloat16, 22 in float16), so that outputs and gradients are in effect rounded once, at the end;
  those of heads that share keys and values are summed in 32 bits before."""
  _no_tangents("memory_scan", q=q, k=k, v=v, log_decay=log_decay, state=state)
  if q.dtype not in _FLOATS or k.dtype != q.dtype or v.dtype != q.dtype:
    raise ValueError(f"q, k, v must be of one type, float32, float16 or bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
  if q.dim() != 4 or q.shape[2] < 1:
    raise ValueError(f"q must be [steps, rows, heads, key_dim], got {list(q.shape)}")
  t, n, h, dk = q.shape
  if k.dim() != 4 or v.dim() != 4 or k.shape[:2] != (t, n) or k.shape[3] != dk or v.shape[:3] != k.shape[:3]:
    raise ValueError(f"k, v must be [{t}, {n}, kv_heads, {dk}] and [{t}, {n}, kv_heads, value_dim], got {list(k.shape)} and {list(v.shape)}")
  dv = v.shape[3]
  if k.shape[2] < 1 or h % k.shape[2]:
    raise ValueError(f"kv_heads = {k.shape[2]} does not divide heads = {h}")
  if not (1 <= dk <= 128 and 1 <= dv <= 128):
    raise ValueError(f"key_dim = {dk}, value_dim = {dv}: not both in [1, 128]")
  if log_decay.dtype != torch.float32 or log_decay.shape != (h,):
    raise ValueError(f"log_decay must be float32 [{h}], got {log_decay.dtype} {list(log_decay.shape)}")
  if log_decay.requires_grad and torch.is_grad_enabled():
    raise ValueError("log_decay is not differentiated: pass log_decay.detach()")
  if fresh is not None and (fresh.dtype not in (torch.bool, torch.uint8) or fresh.shape != (t, n)):
    raise ValueError(f"fresh must be bool or uint8 [{t}, {n}], got {fresh.dtype} {list(fresh.shape)}")
  if state is not None and (state.dtype != torch.float32 or state.shape != (n, h, dk, dv)):
    raise ValueError(f"state must be float32 [{n}, {h}, {dk}, {dv}], got {state.dtype} {list(state.shape)}")
  _same_device(q.device, k=k, v=v, log_decay=log_decay, fresh=fresh, state=state)
  scale = dk ** -0.5 if scale is None else float(scale)
  differentiable = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, state))
  nodes = _guard_capture(q, k, v, state) if differentiable else ()  # noqa: F841 (before copies take the leaves' place)
  q, k, v, log_decay = _dense_last(q), _dense_last(k), _dense_last(v), log_decay.contiguous()
  if differentiable:
    return _MemoryScan.apply(q, k, v, state, log_decay, fresh, scale)
  return _scan_forward(q, k, v, state, log_decay, fresh, scale)
