"""envpool_amd.policy at its edges on the GPU, against the definitions in 64 bits (tests/policy_ref.py): how many bits
results keep, values that are not finite, hooks and checkpoints of autograd, in-place changes."""
import math

import pytest
import torch

from tests import policy_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"
H32 = ref.HALF[torch.float32]


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _decay(h):
  return torch.log1p(-torch.exp2(-2.0 - 6.0 * torch.arange(h).double() / h)).float()


def _scan_problem(t, n, h, hk, dk, dv, p_fresh, dtype):
  g = _gen(7 * t + dk)
  q, k, v = torch.randn(t, n, h, dk, generator=g), torch.randn(t, n, hk, dk, generator=g) * dk**-0.5, torch.randn(t, n, hk, dv, generator=g)
  fresh = torch.rand(t, n, generator=g) < p_fresh
  state, ds = torch.randn(n, h, dk, dv, generator=g), torch.randn(n, h, dk, dv, generator=g)
  do = torch.randn(t, n, h, dv, generator=g)
  return q.to(dtype), k.to(dtype), v.to(dtype), _decay(h), fresh, state, do.to(dtype), ds


def _scan_all(q, k, v, decay, fresh, state, do, ds):
  """Outputs and all gradients of one scan on the GPU, by name, on the CPU."""
  from envpool_amd import policy
  leaves = [x.to(DEV).requires_grad_() for x in (q, k, v, state)]
  out, final = policy.memory_scan(*leaves[:3], decay.to(DEV), fresh=None if fresh is None else fresh.to(DEV), state=leaves[3])
  grads = torch.autograd.grad([out, final], leaves, [do.to(DEV), ds.to(DEV)])
  names = ("out", "final", "grad_q", "grad_k", "grad_v", "grad_state")
  return {name: x.detach().cpu() for name, x in zip(names, (out, final, *grads))}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [(130, 5, 4, 4, 64, 64, 0.02), (130, 3, 4, 1, 48, 64, 0.02), (300, 2, 2, 2, 64, 128, 0.01), (200, 2, 2, 1, 128, 64, 0.01),
                                  (700, 1, 3, 3, 128, 128, 0.004), (260, 520, 2, 2, 64, 32, 0.01), (150, 2, 2, 2, 33, 21, 0.02)],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_results_in_16_bits_are_rounded_once(case, dtype):
  """Chunks, several of them, split time, the pair of gradients: an output is its value in 32 bits, rounded to its type.
  Before that rounding a term (a score times a value, or a query's product with the state) is off by what two pieces of the
  type leave out, half a step squared; in float16 what is below 2^-36 of a row's largest score or state is lost. The
  rest is 32-bit arithmetic: products and sums over 64 steps and `dim` entries twice, powers of the decay (their
  exponents off by 2^-24 of at most 27 octaves, twice), a rounding of the state per chunk, the sum of shared heads."""
  t, n, h, hk, dk, dv, _ = case
  q, k, v, decay, fresh, state, do, ds = _scan_problem(*case, dtype)
  got = _scan_all(q, k, v, decay, fresh, state, do, ds)
  rows = torch.arange(min(n, 6))  # (many rows choose the kernel; a few are looked at)
  part = lambda x, dim: x.index_select(dim, rows)  # noqa: E731
  args = dict(fresh=part(fresh, 1), state=part(state, 0), scale=dk**-0.5, grad_out=part(do, 1), reverse_from=part(ds, 0))
  want = ref.scan(part(q, 1), part(k, 1), part(v, 1), decay, **args)
  size = ref.scan(part(q, 1), part(k, 1), part(v, 1), decay, absolute=True, **args)
  half = ref.HALF[dtype]
  for name in ("out", "grad_q", "grad_k", "grad_v"):
    x, w, s = part(got[name], 1).double(), want[name], size[name]
    inner = 1.01 * half**2 + H32 * (2 * max(dk, dv) + 2 * 64 + 2 * 27 + 4 * (t / 64 + 1) + h // hk + 8)
    tol = s * inner + half * (w.abs() + s * inner) + ref.TINY[dtype] + 2.0**-34 * float(s.max())
    err = (x - w).abs()
    assert got[name].dtype == dtype and (err <= tol).all(), (name, float((err - tol).max()), float((err > tol).double().mean()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(130, 5, 4, 4, 64, 64, 0.02), (700, 1, 3, 3, 128, 128, 0.004), (700, 1, 2, 1, 24, 80, 0.0), (400, 300, 2, 2, 32, 64, 0.01)],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_states_keep_32_bits_over_many_chunks(case, dtype):
  """Carried from chunk to chunk, joined over split time. In half steps of 32 bits and of the sum of magnitudes: 4 for a
  term's two pieces, 2 * 27 ln 2 for its power of the decay, a rounding per step's sum, 3 per chunk that carries it. And of
  the whole in the 2-norm, where t independent roundings of partial sums add up as sqrt(t): 32 for up to 700."""
  t, n, h, hk, dk, dv, _ = case
  q, k, v, decay, fresh, state, do, ds = _scan_problem(*case, dtype)
  got = _scan_all(q, k, v, decay, fresh, state, do, ds)
  rows = torch.arange(min(n, 6))
  part = lambda x, dim: x.index_select(dim, rows)  # noqa: E731
  args = dict(fresh=part(fresh, 1), state=part(state, 0), scale=dk**-0.5, grad_out=part(do, 1), reverse_from=part(ds, 0))
  want = ref.scan(part(q, 1), part(k, 1), part(v, 1), decay, **args)
  size = ref.scan(part(q, 1), part(k, 1), part(v, 1), decay, absolute=True, **args)
  for name in ("final", "grad_state"):
    x, w = part(got[name], 0).double(), want[name]
    err = (x - w).abs()
    tol = size[name] * H32 * (4 + 38 + t + 3 * (t / 32 + 1) + 4) + 2.0**-30
    assert (err <= tol).all(), (name, float((err - tol).max()))
    assert float((x - w).norm()) <= 32 * H32 * float(w.norm()), (name, float((x - w).norm() / w.norm()))


# ---- what autograd may do between the forward and the backward pass ---------------------------------
def _clone_hooks():
  return torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t.clone())


def _checkpointed(call):
  from torch.utils.checkpoint import checkpoint
  return checkpoint(call, use_reentrant=False)


HOOKS = {
  "clone": lambda call: _under(_clone_hooks(), call),
  "save_on_cpu": lambda call: _under(torch.autograd.graph.save_on_cpu(), call),
  "checkpoint": _checkpointed,
}


def _under(context, call):
  with context:
    return call()


def _spoil():
  """Fills the allocator's free memory, so that what was freed no longer holds what it held."""
  spoiled = [torch.full((1 << 16,), 7, dtype=torch.int32, device=DEV) for _ in range(24)] + [torch.full((2048,), 7, dtype=torch.int32, device=DEV) for _ in range(64)]
  torch.cuda.synchronize()
  del spoiled


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("a", [24, 5000])
def test_gradients_under_hooks_for_saved_tensors(a, hook, dtype):
  """Everything the backward pass reads comes from what was saved: the same bits as without the hook."""
  from envpool_amd import policy
  g = _gen(a)
  n = 40
  x = torch.randn(n, a, generator=g).to(dtype).to(DEV).requires_grad_()
  b = torch.randn(n, a, generator=g).to(DEV).requires_grad_()
  mask = torch.rand(n, a, generator=g) < 0.6
  hist = torch.randint(0, a, (n, 9), generator=g, dtype=torch.int32)
  rows = [(0.5 + torch.rand(n, generator=g)).to(DEV) for _ in range(4)]
  action = mask.int().argmax(1).int()
  g1, g2 = torch.randn(n, generator=g).to(DEV), torch.randn(n, generator=g).to(DEV)

  def call():  # (operands that live only as long as the call: the saved ones are the last)
    kw = dict(mask=mask.to(DEV), num_options=torch.full((n,), a - 1, dtype=torch.int32, device=DEV), history=hist.to(DEV), bias=b * 1.0,
              repetition=rows[0].clone(), frequency=rows[1].clone(), presence=rows[2].clone(), temperature=rows[3].clone())
    return policy.evaluate(x * 1.0, action.to(DEV), **kw)

  def run(through):
    lp, ent = through(call)
    _spoil()
    return [lp.detach(), ent.detach(), *torch.autograd.grad([lp, ent], [x, b], [g1, g2])]

  want = run(lambda c: c())
  got = run(HOOKS[hook])
  assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("hook", list(HOOKS))
def test_gradients_of_a_scan_under_hooks_for_saved_tensors(hook):
  from envpool_amd import policy
  q, k, v, decay, fresh, state, do, ds = (x.to(DEV) for x in _scan_problem(130, 3, 4, 2, 32, 48, 0.02, torch.bfloat16))
  leaves = [x.requires_grad_() for x in (q, k, v, state)]

  def call():
    return policy.memory_scan(*(x * 1.0 for x in leaves[:3]), decay.clone(), fresh=fresh.clone(), state=leaves[3] * 1.0)

  def run(through):
    out, final = through(call)
    _spoil()
    return [out.detach(), final.detach(), *torch.autograd.grad([out, final], leaves, [do, ds])]

  want = run(lambda c: c())
  assert all(torch.equal(p, w) for p, w in zip(run(HOOKS[hook]), want))


def test_a_step_between_a_scan_and_its_backward_pass_is_noticed():
  """The state that a scan started from has moved on: an error, not the gradients of another start."""
  from envpool_amd import policy
  g = _gen(3)
  q, k, v = (torch.randn(20, 3, 2, 8, generator=g).to(DEV) for _ in range(3))
  decay = torch.tensor([-0.1, -0.2], device=DEV)
  table = torch.randn(3, 2, 8, 8, generator=g).to(DEV)
  for start in ("memory", "caller"):  # the memory's own view of it, and the tensor that the caller made the memory from
    memory = policy.EnvMemory(3, 2, 8, 8, decay, state=table)
    leaf = q.clone().requires_grad_()
    before = table.clone()
    out, _ = policy.memory_scan(leaf, k, v, decay, state=memory.state if start == "memory" else table)
    kept, _ = policy.memory_scan(leaf, k, v, decay, state=before)
    memory.step(q[0], k[0], v[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
      out.sum().backward()
    kept.sum().backward()
    assert torch.isfinite(leaf.grad).all()
  with torch.inference_mode():
    memory = policy.EnvMemory(3, 2, 8, 8, decay)
    memory.step(q[0], k[0], v[0])
  memory.step(q[0], k[0], v[0])


# ---- values that are not finite ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("filler", [math.inf, math.nan])
@pytest.mark.parametrize("case", [(150, 4, 2, 2, 64, 64), (150, 4, 2, 1, 33, 21), (140, 530, 2, 2, 64, 48), (700, 4, 2, 2, 128, 128), (16, 4, 2, 2, 32, 32)],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_what_is_not_finite_goes_where_the_recurrence_takes_it(case, filler, dtype):
  """A query, key, value or gradient that is not finite, in a row each: later steps of its episode have it in their state,
  earlier ones do not (and the other way round in the gradients), whatever shares a chunk with it. Everything else is
  within the bound of test_results_in_16_bits_are_rounded_once; in 32 bits the same without its pieces."""
  t, n, h, hk, dk, dv = case
  q, k, v, decay, _, state, do, ds = _scan_problem(*case, 0.0, dtype)
  fresh = torch.zeros(t, n, dtype=torch.bool)
  at = 5 * t // 8  # inside a chunk of 32 and of 64
  for row in range(4):
    fresh[[at - 3, t - 2], row] = row % 2 == 0  # an episode that starts soon before and one that starts after, or neither
    (q, k, v, do)[row][at, row, :, :] = filler
  if t > 100:
    v[at + 1, 1, 0, 0] = k[at + 30, 1, -1, -1] = filler  # several, a step and most of a chunk apart
  got = _scan_all(q, k, v, decay, fresh, state, do, ds)
  rows = torch.arange(4)
  part = lambda x, dim: x.index_select(dim, rows)  # noqa: E731
  args = dict(fresh=part(fresh, 1), state=part(state, 0), scale=dk**-0.5, grad_out=part(do, 1), reverse_from=part(ds, 0))
  want = ref.scan(part(q, 1), part(k, 1), part(v, 1), decay, **args)
  size = ref.scan(part(q, 1), part(k, 1), part(v, 1), decay, absolute=True, **args)
  for name, x in got.items():
    x, w, s = part(x, 0 if name in ("final", "grad_state") else 1).double(), want[name], size[name]
    there = torch.isfinite(w)
    assert torch.equal(torch.isfinite(x), there), (name, [sorted(set((torch.isfinite(x) != there).nonzero()[:, 0].tolist()))][:1])
    half = ref.HALF[got[name].dtype]
    inner = 1.01 * ref.HALF[dtype]**2 + H32 * (2 * max(dk, dv) + 2 * 64 + 2 * 27 + t + 4 * (t / 32 + 1) + h // hk + 8)
    tol = s * inner + half * (w.abs() + s * inner) + ref.TINY[dtype] + 2.0**-34 * float(s[there].max())
    assert ((x - w).abs() <= tol)[there].all(), (name, float((x - w).abs()[there].max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,d", [(12, 3, 16), (130, 3, 40), (300, 520, 64), (700, 1, 128)])
def test_a_decay_that_is_nan_shows(t, n, d, dtype):
  """In steps, in short segments and in chunks alike: its head is NaN, the others are as they were."""
  from envpool_amd import policy
  q, k, v, _, _, state, do, ds = (x.to(DEV) for x in _scan_problem(t, n, 2, 2, d, d, 0.0, dtype))
  decay = torch.tensor([math.nan, -0.1], device=DEV)

  def run(decay):
    leaves = [x.detach().requires_grad_() for x in (q, k, v, state)]
    out, final = policy.memory_scan(*leaves[:3], decay, state=leaves[3])
    return [x.detach() for x in (out, final, *torch.autograd.grad([out, final], leaves, [do, ds]))]

  got, plain = run(decay), run(torch.tensor([-0.1, -0.1], device=DEV))
  for i, (x, w) in enumerate(zip(got, plain)):
    h = 1 if i in (1, 5) else 2
    sick, well = x.select(h, 0), x.select(h, 1)
    if i in (3, 4):  # (the last step's gradients of k and v do not pass a decay in the recurrence)
      sick = sick[:-1]
    assert torch.isnan(sick).all() and torch.equal(well, w.select(h, 1)), i
  memory = policy.EnvMemory(n, 2, d, d, decay, state=state.clone())
  out = memory.step(q[0], k[0], v[0])
  assert torch.isnan(out[:, 0]).all() and torch.isfinite(out[:, 1]).all()


@pytest.mark.parametrize("shape", [(6, 1, 1, 1), (9, 3, 5, 7), (40, 4, 64, 64), (3, 8, 256, 256)])
def test_reset_by_id(shape):
  from envpool_amd import policy
  g = _gen(1)
  table = torch.randn(*shape, generator=g).to(DEV)
  n = shape[0]
  memory = policy.EnvMemory(*shape, torch.zeros(shape[1], device=DEV), state=table.clone(), env_id_offset=100)
  memory.reset(torch.tensor([101, 99, 101, 100 + n, 100], dtype=torch.int32, device=DEV))  # twice, and outside on both ends
  assert not memory.state[:2].any() and torch.equal(memory.state[2:], table[2:])
  torch.cuda.synchronize()
  with pytest.raises(RuntimeError, match="outside"):
    memory.poll_errors()
  memory.reset(torch.tensor([2**32 + 102, 102], device=DEV)[1:])
  memory.reset(torch.arange(100, 100 + n, device=DEV)[::2])  # (strided, 64 bits)
  torch.cuda.synchronize()
  memory.poll_errors()
  assert not memory.state[::2].any() and torch.equal(memory.state[3::2], table[3::2])
  memory.reset(torch.tensor([2**32 + 103], device=DEV))
  assert torch.equal(memory.state[3::2], table[3::2])
  torch.cuda.synchronize()
  with pytest.raises(RuntimeError, match="outside"):
    memory.poll_errors()


# ---- logits at the ends of the type's range ---------------------------------------------------------
def _evaluate_all(x, action, g1, g2, **kw):
  from envpool_amd import policy
  leaf = x.to(DEV).requires_grad_()
  lp, ent = policy.evaluate(leaf, action.to(DEV), **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
  gx, = torch.autograd.grad([lp, ent], leaf, [g1.to(DEV), g2.to(DEV)])
  return lp.detach().cpu().double(), ent.detach().cpu().double(), gx.cpu().double()


def _agrees(got, want, size, tol):
  """Within tol of the magnitude `size` (infinite and too large values have to be the same)."""
  top = float(torch.finfo(torch.float32).max)
  want = torch.where(want.abs() > top * (1 + H32), want.sign() * math.inf, want)
  same = (got == want) | ((got - want).abs() <= tol * size)
  return bool(same.all())


@pytest.mark.parametrize("a", [6, 40, 300, 5000])
def test_sums_beyond_32_bits(a):
  """Finite logits and biases whose sum leaves the range: its end stands for them, forward and in the gradients."""
  top = 3e38
  x = torch.randn(3, a, generator=_gen(a))
  b = torch.zeros(3, a)
  x[0, [1, 4]], b[0, [1, 4]] = top, top    # two above everything: a half each
  x[1], b[1] = -top, -top                  # nothing but sums below the range: uniform
  x[2, 3], b[2, 3] = top, top              # one above everything
  action = torch.tensor([1, 2, 3], dtype=torch.int32)
  g1, g2 = torch.ones(3), torch.full((3,), 0.5)
  want = ref.evaluate(x, action, g1, g2, bias=b)
  lp, ent, gx = _evaluate_all(x, action, g1, g2, bias=b)
  tol = 64 * H32
  assert _agrees(lp, want["log_prob"], 1 + want["log_prob"].abs(), tol) and _agrees(ent, want["entropy"], 1 + want["entropy"].abs(), tol)
  assert ((gx - want["grad_logits"]).abs() <= 4 * 12 * tol * (want["grad_logits"].abs() + 1e-3 / a)).all(), (gx - want["grad_logits"]).abs().max(1)


def test_sums_below_32_bits_beside_nothing():
  """A row of nothing but sums below the range and logits of -inf: forward the sums share it; the gradients cannot tell the
  two apart and say so, NaN."""
  x = torch.full((3, 12), -3e38)
  b = torch.full((12,), -3e38)
  x[0, 4] = x[1, 0] = -math.inf
  action = torch.tensor([1, 1, 1], dtype=torch.int32)
  mask = torch.ones(3, 12, dtype=torch.bool)
  mask[1, 0] = False  # (not legal: not looked at)
  lp, ent, gx = _evaluate_all(x, action, torch.ones(3), torch.ones(3), bias=b, mask=mask)
  assert torch.allclose(lp, -torch.log(torch.tensor([11.0, 11.0, 12.0]).double()), atol=1e-6) and torch.allclose(ent, -lp, atol=1e-6)
  assert torch.isnan(gx[0]).all() and torch.isfinite(gx[1:]).all() and gx[1, 0] == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("a", [6, 40, 300, 5000])
def test_rows_masked_with_the_lowest_value(a, dtype):
  """Options masked by the type's lowest value instead of by a mask: among others they keep their tiny probability (a
  log-probability of the value's size, not -inf), and a row of nothing else is uniform, its gradients too. The sums have up
  to 5000 equal terms in 32 bits: (5000 / 2048 * 8 + 20) half steps of their 1."""
  low = torch.finfo(dtype).min
  x = torch.randn(5, a, generator=_gen(a)).to(dtype)
  x[0] = low
  x[1] = low
  x[1, a - 1] = -math.inf  # no probability at all: the others are uniform
  x[2, ::2] = low          # action there
  x[3, 1::2] = low         # action not there
  x[4] = low
  x[4, 2] = 1.0
  action = torch.tensor([3, 2, 4, 4, 2], dtype=torch.int32)
  g1, g2 = torch.tensor([1.0, -2.0, 0.5, 1.5, 1.0]), torch.tensor([0.3, 1.0, -1.0, 0.5, 0.1])
  for kw in (dict(), dict(temperature=2.5), dict(num_options=torch.full((5,), a - 1, dtype=torch.int32)), dict(mask=torch.arange(a)[None].expand(5, a) != 5)):
    want = ref.evaluate(x, action, g1, g2, **kw)
    lp, ent, gx = _evaluate_all(x, action, g1, g2, **kw)
    tol = 64 * H32
    assert _agrees(lp, want["log_prob"], 1 + want["log_prob"].abs().nan_to_num(0, 0, 0), tol), (lp, want["log_prob"])
    assert _agrees(ent, want["entropy"], 1 + want["entropy"].abs(), tol), (ent, want["entropy"])
    # dy = g1 (one - p) - g2 p (ln p + H). p is off by r: the sum's 64 half steps, and (y - m) / T, of magnitudes up to 10,
    # in the exponent, 5 roundings; H by what was allowed above; ln p by r and its own two roundings. One rounding each of the sums
    y = ref.processed(x, **kw)[0]
    m, w, total, _, _ = ref.distribution(y)
    p = w / total[:, None]
    logp = torch.where(w > 0, y - m - torch.log(total)[:, None], 0.0)
    r, h = (64 + 50) * H32, want["entropy"][:, None]
    g_1, g_2 = g1.double().abs()[:, None], g2.double().abs()[:, None]
    bound = g_1 * (p * r + 4 * H32) + g_2 * p * ((logp + h).abs() * (r + 4 * H32) + (1 + h) * tol + r + 2 * H32 * logp.abs())
    slack = bound / kw.get("temperature", 1.0) + (4 * H32 + ref.HALF[dtype]) * want["grad_logits"].abs() + ref.TINY[dtype]
    assert ((gx - want["grad_logits"]).abs() <= slack).all(), ((gx - want["grad_logits"]).abs() - slack).max(1)


@pytest.mark.parametrize("a", [6, 40, 5000])
@pytest.mark.parametrize("per_row", [False, True])
def test_temperatures_at_the_end_of_the_range(a, per_row):
  """However hot, an option that is not legal has no probability."""
  from envpool_amd import policy
  x = torch.randn(4, a, generator=_gen(a))
  count = torch.tensor([2, a // 2, a, 1], dtype=torch.int32)
  action = torch.zeros(4, dtype=torch.int32)
  g = torch.ones(4)
  for t in (1e30, 1e37, 3.4e38):
    temp = torch.full((4,), t) if per_row else t
    kw = dict(num_options=count, temperature=temp)
    want = ref.evaluate(x, action, g, g, **kw)
    lp, ent, gx = _evaluate_all(x, action, g, g, **kw)
    tol = 64 * H32
    assert _agrees(lp, want["log_prob"], 1 + want["log_prob"].abs(), tol) and _agrees(ent, want["entropy"], 1 + want["entropy"].abs(), tol), (t, lp, ent)
    c = policy.choose(x.to(DEV), torch.full((4,), 0.999, device=DEV), num_options=count.to(DEV), temperature=temp.to(DEV) if per_row else t)
    assert torch.equal(c.action.cpu().long(), ref.choose(x, torch.full((4,), 0.999), **kw)[0])
  if not per_row:
    c = policy.choose(x.to(DEV), torch.full((4,), 0.999, device=DEV), num_options=count.to(DEV), temperature=1e307)
    assert (c.action.cpu() < count).all() and torch.allclose(c.entropy.cpu(), torch.log(count.float()), atol=1e-6)


def test_repetitions_of_a_row_that_are_no_numbers():
  from envpool_amd import policy
  x = torch.randn(4, 9, generator=_gen(0)).to(DEV).requires_grad_()
  kw = dict(history=torch.full((4, 2), 3, dtype=torch.int32, device=DEV), repetition=torch.tensor([1.2, math.inf, 1e-40, math.nan], device=DEV))
  lp, ent = policy.evaluate(x, torch.zeros(4, dtype=torch.int32, device=DEV), **kw)
  gx, = torch.autograd.grad(lp.sum() + ent.sum(), x)
  c = policy.choose(x, **kw)
  for t in (lp, ent, gx[:, 0]):
    assert torch.isfinite(t[0]) and torch.isnan(t[1:]).all()
  assert c.action[0] >= 0 and c.action[[1, 3]].tolist() == [-1, -1]  # (64 bits hold 1e-40 and its reciprocal)
  # without a history there is nothing to repeat
  lp, _ = policy.evaluate(x, torch.zeros(4, dtype=torch.int32, device=DEV), repetition=1e300)
  assert torch.isfinite(lp).all()


def test_captured_over_leaves_with_gaps():
  """Transposed and expanded leaves in a captured forward and backward pass: every replay against the eager result."""
  from envpool_amd import policy
  g = _gen(4)
  n, a, t = 5, 12, 130
  logits = torch.randn(a, n, generator=g).to(DEV).t().requires_grad_()
  bias = torch.randn(1, a, generator=g).to(DEV).expand(n, a).requires_grad_()
  q = torch.randn(t, 3, 8, 2, generator=g).to(DEV).transpose(2, 3).requires_grad_()
  k, v = (torch.randn(t, 3, 2, 8, generator=g).to(DEV).requires_grad_() for _ in range(2))
  action = torch.arange(n, dtype=torch.int32, device=DEV)
  decay = torch.tensor([-0.1, -0.2], device=DEV)

  def work():
    lp, ent = policy.evaluate(logits, action, bias=bias)
    out, final = policy.memory_scan(q, k, v, decay)
    outs = [lp, ent, out, final]
    return [x.detach() for x in outs] + list(torch.autograd.grad(outs, [logits, bias, q, k, v], [torch.ones_like(x) for x in outs]))

  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    work()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = work()
  for _ in range(3):
    with torch.no_grad():
      logits.copy_(torch.randn(n, a, generator=g).to(DEV))
      k.copy_(torch.randn(t, 3, 2, 8, generator=g).to(DEV))
    graph.replay()
    got = [x.clone() for x in captured]
    torch.cuda.synchronize()
    want = work()
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for x, w in zip(got, want))


def test_the_error_word_of_a_dropped_memory_is_nobody_elses():
  """A step under way may still flag an error when its memory is gone: not in memory that has a new owner."""
  from envpool_amd import policy
  words = []
  for _ in range(3):
    memory = policy.EnvMemory(2, 1, 4, 4, torch.zeros(1, device=DEV))
    words.append(memory._error.data_ptr())
    del memory
    new = [torch.zeros(1, dtype=torch.int32, pin_memory=True) for _ in range(8)]
    assert not any(t.data_ptr() <= w < t.data_ptr() + 4 for t in new for w in words)
  assert len(set(words)) == 3
  memories = [policy.EnvMemory(2, 1, 4, 4, torch.zeros(1, device=DEV)) for _ in range(1100)]
  assert len({m._error.data_ptr() for m in memories}) == 1100
  one = torch.ones(1, 1, 4, device=DEV)
  memories[700].step(one, one, one, env_id=torch.tensor([5], dtype=torch.int32, device=DEV))
  torch.cuda.synchronize()
  for i in (0, 699, 701, 1099):
    memories[i].poll_errors()
  with pytest.raises(RuntimeError, match="outside"):
    memories[700].poll_errors()


def test_gradients_of_segments_without_steps_or_rows():
  """No steps: the first state is the last one, gradient included. No rows: empty gradients."""
  from envpool_amd import policy
  g = _gen(1)
  for t, n in ((0, 3), (7, 0), (130, 0), (0, 0)):
    q, k, v = (torch.randn(t, n, h, 8, generator=g).to(DEV).requires_grad_() for h in (4, 2, 2))
    state = torch.randn(n, 4, 8, 8, generator=g).to(DEV).requires_grad_()
    out, final = policy.memory_scan(q, k, v, torch.full((4,), -0.5, device=DEV), state=state)
    ds = torch.randn(n, 4, 8, 8, generator=g).to(DEV)
    grads = torch.autograd.grad([out, final], [q, k, v, state], [torch.ones_like(out), ds])
    assert [x.shape for x in grads] == [x.shape for x in (q, k, v, state)]
    assert torch.equal(grads[3], ds) and torch.equal(final, state)


@pytest.mark.parametrize("a", [24, 5000])
@pytest.mark.parametrize("rows", [0, 1, 37])
def test_the_gradient_of_a_bias_alone(a, rows):
  """Logits that require none, a bias for all rows and one for each."""
  from envpool_amd import policy
  g = _gen(a)
  x = torch.randn(rows, a, generator=g).to(DEV)
  action = torch.randint(0, a, (rows,), generator=g, dtype=torch.int32).to(DEV)
  for b in (torch.randn(a, generator=g), torch.randn(1, a, generator=g), torch.randn(rows, a, generator=g)):
    alone, both = b.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()
    leaf = x.clone().requires_grad_()
    lp, ent = policy.evaluate(x, action, bias=alone)
    one, = torch.autograd.grad(lp.sum() + ent.sum(), alone)
    lp, ent = policy.evaluate(leaf, action, bias=both)
    _, two = torch.autograd.grad(lp.sum() + ent.sum(), [leaf, both])
    assert one.shape == b.shape and torch.equal(one, two) and (rows or not one.any())
  lp, ent = policy.evaluate(leaf, action)
  assert torch.autograd.grad(lp.sum() + ent.sum(), leaf)[0].shape == (rows, a)
