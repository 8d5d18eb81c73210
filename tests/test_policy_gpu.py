"""envpool_amd.policy on the GPU against the definitions in 64 bits (tests/policy_ref.py)."""
import math

import pytest
import torch

from tests import policy_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _bits(legal):
  n, a = legal.shape
  words = torch.zeros(n, (a + 31) // 32, dtype=torch.int64)
  for i in range(32):
    col = legal[:, i::32].long()
    words[:, :col.shape[1]] |= col << i
  words = torch.where(words >= 2**31, words - 2**32, words)
  return words.to(torch.int32)


def _problem(n, a, dtype, mask, bias, hist, per_row, seed):
  """-> (logits, options for choose / evaluate, legal actions), with empty rows and garbage in masked places."""
  g = _gen(seed)
  logits = (3 * torch.randn(n, a, generator=g)).to(dtype)
  legal = torch.ones(n, a, dtype=torch.bool)
  kw = {"temperature": 0.7}
  if mask in ("count", "both"):
    count = torch.randint(0, a + 1, (n,), generator=g, dtype=torch.int32)
    legal &= torch.arange(a)[None] < count[:, None]
    kw["num_options"] = count
  if mask in ("bytes", "bits", "both", "one"):
    m = torch.rand(1 if mask == "one" else n, a, generator=g) < 0.5
    if mask != "one":
      m[::5] = False
    else:
      m[0, a // 2] = True
    legal &= m
    kw["mask"] = _bits(m) if mask == "bits" else m
  logits[~legal] = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max], dtype=dtype)[
      torch.randint(0, 4, (int((~legal).sum()),), generator=g)]
  if bias:
    kw["bias"] = torch.randn(a if bias == "shared" else (n, a), generator=g).to(dtype if bias == "typed" else torch.float32)
  if hist:
    h = (torch.rand(n, hist, generator=g)**2 * (a + 2)).int() - 1  # outside on both ends too
    kw.update(history=h, repetition=1.3, frequency=0.2, presence=0.4)
  if per_row:
    kw["temperature"] = 0.5 + torch.rand(n, generator=g)
    if hist:
      kw.update(repetition=1 + torch.rand(n, generator=g), frequency=torch.rand(n, generator=g), presence=torch.rand(n, generator=g))
  action = torch.where(legal.any(1), (torch.rand(n, a, generator=g) * legal).argmax(1), -1).int()
  return logits, kw, action


def _to(kw):
  return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}


CASES = [
  # rows, options, mask, bias, history, per-row numbers
  (1, 1, "none", "", 0, False), (3, 1, "count", "", 0, False), (5, 2, "both", "shared", 0, False), (64, 7, "bytes", "rows", 3, True),
  (1030, 16, "count", "", 0, False), (257, 16, "bytes", "shared", 0, True), (33, 24, "both", "typed", 5, False), (19, 64, "bits", "", 64, True),
  (9, 65, "one", "shared", 0, False), (7, 255, "bits", "rows", 0, False), (6, 256, "none", "", 9, False), (5, 1000, "count", "typed", 0, True),
  (5, 1024, "bits", "shared", 700, True), (4, 1025, "both", "", 0, False), (3, 2048, "bytes", "", 0, False), (3, 2049, "none", "rows", 31, False),
  (2, 9973, "bits", "shared", 300, True), (2, 70001, "count", "", 100, False), (1, 131072, "bits", "rows", 0, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
@pytest.mark.parametrize("greedy", [False, True])
def test_choose(case, dtype, greedy):
  from envpool_amd import policy
  n, a = case[:2]
  logits, kw, _ = _problem(n, a, dtype, *case[2:], seed=n * 7 + a)
  u = None if greedy else torch.rand(n, generator=_gen(a), dtype=torch.float64 if n % 2 else torch.float32)
  want = ref.choose(logits, u, **kw)
  got = policy.choose(logits.to(DEV), None if u is None else u.to(DEV), **_to(kw))
  assert got.action.dtype == torch.int32 and torch.equal(got.action.cpu().long(), want[0])
  for x, w in zip(got[1:], want[1:]):  # computed in 64 bits, rounded once
    x, w = x.cpu().double(), w
    assert x.shape == w.shape and torch.equal(torch.isnan(x), torch.isnan(w))
    assert ((x - w).abs() <= ref.HALF[torch.float32] * w.abs() + 1e-9).all(), (x - w).abs().max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_evaluate_and_its_gradients(case, dtype):
  from envpool_amd import policy
  n, a = case[:2]
  logits, kw, action = _problem(n, a, dtype, *case[2:], seed=n + a)
  g = _gen(3)
  g1, g2 = torch.randn(n, generator=g), torch.randn(n, generator=g)
  want = ref.evaluate(logits, action, g1, g2, **kw)
  dkw = _to(kw)
  leaves = [logits.to(DEV).requires_grad_()]
  if "bias" in dkw:
    dkw["bias"].requires_grad_()
    leaves.append(dkw["bias"])
  lp, ent = policy.evaluate(leaves[0], action.to(DEV), **dkw)
  grads = torch.autograd.grad([lp, ent], leaves, [g1.to(DEV), g2.to(DEV)])
  assert ((lp.detach().cpu().double() - want["log_prob"]).abs() <= want["tol_log_prob"]).all()
  assert ((ent.detach().cpu().double() - want["entropy"]).abs() <= want["tol_entropy"]).all()
  gx = grads[0].cpu().double()
  assert grads[0].dtype == dtype and grads[0].shape == logits.shape
  tiny = ref.TINY[dtype]
  assert ((gx - want["grad_logits"]).abs() <= want["tol_logits"] + ref.HALF[dtype] * want["grad_logits"].abs() + tiny).all()
  if "bias" in kw:
    b = kw["bias"]
    gb, wb, tb = grads[1].cpu().double(), want["grad_bias"], want["tol_bias"]
    assert grads[1].dtype == b.dtype and grads[1].shape == b.shape
    if b.dim() == 1:
      tb = tb.sum(0) + (n / 2 + 20) * ref.HALF[torch.float32] * wb.abs().sum(0)
      wb = wb.sum(0)
    assert ((gb - wb).abs() <= tb + ref.HALF[b.dtype] * wb.abs() + ref.TINY[b.dtype]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1700, 2056, "bits", "shared", 0, False), (1600, 2051, "none", "rows", 5, False), (1600, 2056, "bytes", "typed", 40, True),
                                  (150000, 24, "bytes", "shared", 0, False), (140000, 13, "count", "typed", 3, False), (1200, 1500, "count", "shared", 0, True)],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_more_rows_than_the_chip_holds_at_once(case, dtype):
  """Workgroups that walk down several rows, each way of reading them."""
  test_evaluate_and_its_gradients(case, dtype)
  test_choose(case, dtype, False)


@pytest.mark.parametrize("a", [6, 40, 300, 5000])
def test_rows_without_a_distribution(a):
  """Nothing legal, nothing but -inf, NaN or +inf among the legal, the type's lowest value everywhere."""
  from envpool_amd import policy
  x = torch.zeros(8, a)
  x[1] = -math.inf
  x[2, a // 2] = math.nan
  x[3, a - 1] = math.inf
  x[4] = torch.finfo(torch.float32).min
  x[5] = torch.finfo(torch.float32).min
  x[5, 3] = 2.0
  x[6, 4:] = -math.inf
  temp = torch.ones(8)
  temp[7] = 0.0  # not a temperature
  count = torch.full((8,), a, dtype=torch.int32)
  count[0] = 0
  for u in (None, torch.full((8,), 0.5, device=DEV)):
    c = policy.choose(x.to(DEV), u, num_options=count.to(DEV), temperature=temp.to(DEV))
    act, lp, ent = (t.cpu() for t in c)
    assert act[:4].tolist() == [-1] * 4 and act[7] == -1
    assert lp[:2].tolist() == [0.0] * 2 and ent[:2].tolist() == [0.0] * 2
    assert torch.isnan(lp[[2, 3, 7]]).all() and torch.isnan(ent[[2, 3, 7]]).all()
    assert int(act[4]) == (0 if u is None else a // 2) and int(act[5]) == 3
    assert abs(float(lp[4]) + math.log(a)) < 1e-5 and float(lp[5]) == 0.0 and float(ent[5]) == 0.0
    assert 0 <= int(act[6]) < 4 and abs(float(ent[6]) - math.log(4)) < 1e-6
  leaf = x.to(DEV).requires_grad_()
  action = torch.tensor([-1, -1, 0, 0, 1, 3, 5, 0], dtype=torch.int32, device=DEV)
  lp, ent = policy.evaluate(leaf, action, num_options=count.to(DEV), temperature=temp.to(DEV))
  gx, = torch.autograd.grad([lp, ent], leaf, [torch.ones(8, device=DEV), torch.ones(8, device=DEV)])
  lp, ent, gx = lp.detach().cpu(), ent.detach().cpu(), gx.cpu()
  assert lp[:2].tolist() == [0.0, 0.0] and ent[:2].tolist() == [0.0, 0.0] and (gx[:2] == 0).all()
  assert torch.isnan(lp[[2, 3, 7]]).all() and torch.isnan(gx[2, 0]) and torch.isnan(gx[3, 0])
  assert abs(float(lp[4]) + math.log(a)) < 1e-4 and float(lp[5]) == 0.0 and (gx[5] == 0).all()
  assert float(lp[6]) == -math.inf and torch.isfinite(gx[6]).all()
  # values outside the options
  lp, _ = policy.evaluate(torch.zeros(3, a, device=DEV), torch.tensor([-2, a, -1], dtype=torch.int32, device=DEV))
  assert torch.isnan(lp[:2]).all() and float(lp[2]) == 0.0


def test_ends_of_the_uniform_range():
  from envpool_amd import policy
  for a in (5, 70, 3001, 40000):
    x = torch.randn(4, a, generator=_gen(a))
    legal = torch.rand(4, a, generator=_gen(1)) < 0.3
    legal[:, [1, a - 2]] = True
    legal[:, [0, a - 1]] = False
    u = torch.tensor([0.0, math.nextafter(1.0, 0.0), 1.0, 0.0], dtype=torch.float64)
    c = policy.choose(x.to(DEV), u.to(DEV), mask=legal.to(DEV))
    lowest, highest = legal.int().argmax(1), a - 1 - legal.flip(1).int().argmax(1)
    assert c.action.cpu().tolist() == [int(lowest[0]), int(highest[1]), int(highest[2]), int(lowest[3])]


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_odd_alignment(dtype):
  from envpool_amd import policy
  for a in (13, 16, 257, 2056):
    big = torch.randn(9, 2 * a + 5, generator=_gen(a)).to(dtype).to(DEV)
    mask = (torch.rand(9, a + 3, generator=_gen(2)) < 0.6).to(DEV)
    u = torch.rand(9, 2, generator=_gen(4)).to(DEV)[:, 1]
    for view in (big[:, 1:1 + a], big[:, ::2][:, :a], big[::2][:, :a].repeat(2, 1)[:9], big[:1, :a].expand(9, a)):
      want = policy.choose(view.clone(), u.clone(), mask=mask[:, 1:1 + a].clone())
      got = policy.choose(view, u, mask=mask[:, 1:1 + a])
      assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gradient_against_differences():
  from envpool_amd import policy
  g = _gen(11)
  n, a = 4, 21
  x = torch.randn(n, a, generator=g)
  hist = torch.randint(0, a, (n, 6), generator=g, dtype=torch.int32)
  b = torch.randn(a, generator=g)
  action = torch.randint(0, a, (n,), generator=g, dtype=torch.int32)
  kw = dict(history=hist, repetition=1.4, frequency=0.1, presence=0.2, temperature=1.7)
  g1, g2 = torch.randn(n, generator=g), torch.randn(n, generator=g)

  def value(xx, bb):
    r = ref.evaluate(xx, action, g1, g2, bias=bb, **kw)
    return float((r["log_prob"] * g1.double() + r["entropy"] * g2.double()).sum())

  lx, lb = x.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()
  lp, ent = policy.evaluate(lx, action.to(DEV), bias=lb, **_to(kw))
  ((lp * g1.to(DEV)).sum() + (ent * g2.to(DEV)).sum()).backward()
  for _ in range(5):
    dx, db = torch.randn(n, a, generator=g).double(), torch.randn(a, generator=g).double()
    eps = 1e-5
    num = (value(x.double() + eps * dx, b.double() + eps * db) - value(x.double() - eps * dx, b.double() - eps * db)) / (2 * eps)
    ana = float((lx.grad.cpu().double() * dx).sum() + (lb.grad.cpu().double() * db).sum())
    assert abs(num - ana) < 1e-4 * (1 + abs(num))


# ---- memory --------------------------------------------------------------------------------------
def _decay(h):
  return torch.log1p(-torch.exp2(-2.0 - 6.0 * torch.arange(h).double() / h)).float()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,hk,dk,dv", [(1, 1, 1, 1, 1), (8, 4, 4, 64, 64), (5, 6, 2, 33, 17), (3, 2, 1, 128, 256), (2, 3, 3, 256, 40), (1500, 2, 2, 16, 32),
                                          (7, 5, 5, 20, 100), (4, 2, 2, 96, 6)])
def test_memory_step(dtype, n, h, hk, dk, dv):
  from envpool_amd.policy import EnvMemory
  g = _gen(n + dk)
  envs = n + 3
  state = torch.randn(envs, h, dk, dv, generator=g)
  decay = _decay(h)
  mem = EnvMemory(envs, h, dk, dv, decay.to(DEV), state=state.to(DEV), env_id_offset=10)
  ids = torch.randperm(envs, generator=g)[:n]
  h32 = ref.HALF[torch.float32]
  for step in range(2):
    q, k, v = (torch.randn(n, x, d, generator=g).to(dtype) for x, d in ((h, dk), (hk, dk), (hk, dv)))
    elapsed = torch.randint(0, 3, (n,), generator=g, dtype=torch.int32)
    before = mem.state.cpu().double()
    if step:
      out = mem.step(q.to(DEV), k.to(DEV), v.to(DEV), env_id=(ids + 10).int().to(DEV), fresh=(elapsed == 0).to(DEV))
    else:
      out = mem.step(q.to(DEV), k.to(DEV), v.to(DEV), env_id=(ids + 10).int().to(DEV), elapsed_step=elapsed.to(DEV))
    want = ref.scan(q[None], k[None], v[None], decay, fresh=(elapsed == 0)[None], state=before[ids], scale=dk**-0.5)
    size = ref.scan(q[None], k[None], v[None], decay, fresh=(elapsed == 0)[None], state=before[ids], scale=dk**-0.5, absolute=True)
    after = mem.state.cpu().double()
    others = torch.ones(envs, dtype=torch.bool)
    others[ids] = False
    assert torch.equal(after[others], before[others])
    # state: decay rounded (twice: exp), two products, a sum
    assert ((after[ids] - want["final"]).abs() <= 6 * h32 * size["final"]).all()
    # out: the state's 6, dk products and sums, the scale, the result's type
    tol = (dk + 10) * h32 * size["out"][0] + ref.HALF[dtype] * want["out"][0].abs() + ref.TINY[dtype]
    assert out.dtype == dtype and ((out.cpu().double() - want["out"][0]).abs() <= tol).all()


@pytest.mark.parametrize("n,h,hk,dk,dv", [(40, 3, 1, 101, 66), (6, 2, 2, 33, 67), (5, 2, 1, 64, 130), (4, 1, 1, 31, 201), (3, 2, 2, 16, 255), (3, 1, 1, 5, 254)])
def test_memory_step_of_uneven_widths(n, h, hk, dk, dv):
  """Rows of the state that are not made of 16-byte pieces: 8 bytes or 4 a lane, once, twice or four times."""
  for dtype in DTYPES:
    test_memory_step(dtype, n, h, hk, dk, dv)


@pytest.mark.parametrize("n", [9, 1300])
def test_memory_step_envs_named_twice_and_out_of_range(n):
  """Rows of one env are stepped in row order; a foreign id touches nothing, gives NaN and an error later."""
  from envpool_amd.policy import EnvMemory
  g = _gen(5)
  h, dk, dv, envs = 2, 16, 8, n
  decay = _decay(h)
  state = torch.randn(envs, h, dk, dv, generator=g)
  ids = torch.randperm(envs, generator=g).int()
  ids[5] = ids[2]
  ids[7] = ids[2]
  ids[n - 1] = ids[0]
  q, k, v = (torch.randn(n, h, d, generator=g) for d in (dk, dk, dv))
  fresh = torch.rand(n, generator=g) < 0.2
  fresh[5] = False
  mem = EnvMemory(envs, h, dk, dv, decay.to(DEV), state=state.clone().to(DEV))
  out = mem.step(q.to(DEV), k.to(DEV), v.to(DEV), env_id=ids.to(DEV), fresh=fresh.to(DEV)).cpu()
  one = EnvMemory(envs, h, dk, dv, decay.to(DEV), state=state.clone().to(DEV))
  for i in range(n) if n < 100 else []:
    row = one.step(q[i:i + 1].to(DEV), k[i:i + 1].to(DEV), v[i:i + 1].to(DEV), env_id=ids[i:i + 1].to(DEV), fresh=fresh[i:i + 1].to(DEV))
    assert torch.equal(row[0].cpu(), out[i])
  if n < 100:
    assert torch.equal(one.state, mem.state)
  else:
    s = state[ids[2].item()].double()
    lam = torch.exp(decay.double())[:, None, None]
    for i in (2, 5, 7):
      s = (s * 0 if fresh[i] else s * lam) + k[i].double()[..., :, None] * v[i].double()[..., None, :]
      want = dk**-0.5 * (q[i].double()[..., None] * s).sum(1)
      assert (out[i].double() - want).abs().max() < 1e-5
    assert (mem.state[ids[2].item()].cpu().double() - s).abs().max() < 1e-5
  before = mem.state.clone()
  bad = ids.clone()
  bad[1], bad[3] = envs, -1
  keep = torch.ones(n, dtype=torch.bool)
  keep[[1, 3]] = False
  out = mem.step(q.to(DEV), k.to(DEV), v.to(DEV), env_id=bad.to(DEV))
  torch.cuda.synchronize()
  assert torch.isnan(out.cpu()[~keep]).all() and torch.isfinite(out.cpu()[keep]).all()
  untouched = sorted(set(range(envs)) - set(bad[keep].tolist()))
  assert torch.equal(mem.state[untouched], before[untouched])
  with pytest.raises(RuntimeError, match="outside"):
    mem.step(q.to(DEV), k.to(DEV), v.to(DEV), env_id=ids.to(DEV))
  mem.poll_errors()  # reported once


def test_memory_step_without_ids_and_reset():
  from envpool_amd.policy import EnvMemory
  g = _gen(8)
  mem = EnvMemory(6, 2, 8, 12, _decay(2).to(DEV))
  ids = torch.arange(6, dtype=torch.int32, device=DEV)
  other = EnvMemory(6, 2, 8, 12, _decay(2).to(DEV))
  for _ in range(3):
    q, k, v = (torch.randn(6, 2, d, generator=g).to(DEV) for d in (8, 8, 12))
    assert torch.equal(mem.step(q, k, v), other.step(q, k, v, env_id=ids))
  q0 = torch.zeros(0, 2, 8, device=DEV)
  assert mem.step(q0, q0, torch.zeros(0, 2, 12, device=DEV)).shape == (0, 2, 12)
  # infinities in a state that is dropped do not come through
  mem.state[1] = math.inf
  fresh = torch.tensor([0, 1, 0, 0, 0, 0], dtype=torch.uint8, device=DEV)
  assert torch.isfinite(mem.step(q, k, v, fresh=fresh)).all() and torch.isfinite(mem.state).all()
  mem.reset(torch.tensor([2, 4], device=DEV))
  assert (mem.state[[2, 4]] == 0).all() and (mem.state[3] != 0).any()
  mem.reset()
  assert (mem.state == 0).all()


SCANS = [
  # steps, rows, heads, kv heads, key dim, value dim, fresh, state
  (1, 1, 1, 1, 1, 1, 0.0, False), (1, 5, 2, 2, 64, 64, 0.5, True), (7, 3, 2, 1, 16, 24, 0.3, True), (63, 2, 1, 1, 32, 32, 0.0, True),
  (64, 2, 2, 2, 64, 64, 0.02, True), (65, 2, 3, 3, 40, 72, 0.05, False), (130, 3, 4, 2, 64, 128, 0.02, True), (200, 1, 2, 2, 128, 128, 0.0, True),
  (257, 2, 3, 1, 80, 112, 0.01, True), (700, 3, 2, 2, 72, 16, 0.004, True), (700, 2, 2, 1, 100, 60, 0.004, True), (96, 1, 1, 1, 128, 5, 0.9, True), (1000, 1, 2, 2, 33, 64, 0.003, True),
]


def _scan_problem(case, dtype, seed=0):
  t, n, h, hk, dk, dv, p, with_state = case
  g = _gen(t + dk + seed)
  q = torch.randn(t, n, h, dk, generator=g).to(dtype)
  k = (torch.randn(t, n, hk, dk, generator=g) * dk**-0.5).to(dtype)
  v = torch.randn(t, n, hk, dv, generator=g).to(dtype)
  fresh = torch.rand(t, n, generator=g) < p
  state = torch.randn(n, h, dk, dv, generator=g) if with_state else None
  do = torch.randn(t, n, h, dv, generator=g).to(dtype)
  ds = torch.randn(n, h, dk, dv, generator=g) if with_state else None
  return q, k, v, _decay(h), fresh, state, do, ds


def _tol(size, value, dtype, steps, dim, extra=0):
  """An output of the chunked form. Inside, in a 16-bit type: the weighted scores, the weighted values and the
  state are each rounded once before a product (3 half steps of the sums of magnitudes). In 32 bits: products and
  sums over up to 64 steps and `dim` entries twice, decays as powers (one 2^-24 of the exponent, at most 64 * 2 ln
  2 of it), one rounding of the carried state per chunk. Then one rounding of the result."""
  h32 = ref.HALF[torch.float32]
  inner = 3 * ref.HALF[dtype] if dtype != torch.float32 else 0.0
  return size * (inner * 1.01 + h32 * (2 * dim + 2 * 64 + 100 + 4 * (steps / 64 + 1) + extra)) + ref.HALF[dtype] * value.abs() + \
      ref.TINY[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SCANS, ids=lambda c: "-".join(str(x) for x in c))
def test_memory_scan_and_its_gradients(case, dtype):
  from envpool_amd import policy
  t, n, h, hk, dk, dv, _, with_state = case
  q, k, v, decay, fresh, state, do, ds = _scan_problem(case, dtype)
  args = dict(fresh=fresh, state=state, scale=dk**-0.5, grad_out=do, reverse_from=ds)
  want = ref.scan(q, k, v, decay, **args)
  size = ref.scan(q, k, v, decay, absolute=True, **args)
  leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
  s_leaf = None if state is None else state.to(DEV).requires_grad_()
  out, final = policy.memory_scan(*leaves, decay.to(DEV), fresh=fresh.to(DEV), state=s_leaf)
  gets = leaves + ([s_leaf] if with_state else [])
  grads = torch.autograd.grad([out, final] if with_state else [out], gets, [do.to(DEV), ds.to(DEV)] if with_state else [do.to(DEV)])
  group = h // hk
  got = {"out": out.detach(), "final": final.detach(), "grad_q": grads[0], "grad_k": grads[1], "grad_v": grads[2]}
  if with_state:
    got["grad_state"] = grads[3]
  for name, x in got.items():
    w, s = want[name], size[name]
    assert x.shape == w.shape, name
    assert x.dtype == (torch.float32 if name in ("final", "grad_state") else dtype)
    if x.dtype == torch.float32 and dtype != torch.float32:  # a state: its increments are rounded, it is not
      tol = _tol(s, w * 0, dtype, t, max(dk, dv)) + ref.HALF[torch.float32] * w.abs()
    else:
      tol = _tol(s, w, dtype, t, max(dk, dv), extra=group)
    err = (x.cpu().double() - w).abs()
    assert (err <= tol).all(), (name, float((err - tol).max()), float(err.max()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_memory_scan_keeps_what_is_not_finite_inside_its_episode(dtype):
  """An env whose keys or values overflowed: the next episode, and the one before in the gradients, are as if
  those steps had been zero."""
  from envpool_amd import policy
  t, n, h, dk, dv = 150, 4, 2, 40, 24
  q, k, v, decay, _, state, do, ds = _scan_problem((t, n, h, h, dk, dv, 0.0, True), dtype)
  fresh = torch.zeros(t, n, dtype=torch.bool)
  fresh[[0, 20, 33, 70, 140], 0] = True   # several episodes inside a chunk
  fresh[[63, 64, 65], 1] = True
  fresh[100, 2] = True
  bad = torch.zeros(t, n, dtype=torch.bool)
  bad[25, 0] = bad[64, 1] = bad[99, 2] = True
  ep = fresh.int().cumsum(0)
  sick = torch.zeros(t, n, dtype=torch.bool)  # steps of an episode with a bad step
  for b in range(n):
    for e in ep[bad[:, b], b].tolist():
      sick[:, b] |= ep[:, b] == e

  def run(filler):
    kk, vv, dd = k.clone(), v.clone(), do.clone()
    kk[bad], vv[bad], dd[bad] = filler, filler, filler
    leaves = [x.to(DEV).requires_grad_() for x in (q, kk, vv, state)]
    out, final = policy.memory_scan(*leaves[:3], decay.to(DEV), fresh=fresh.to(DEV), state=leaves[3])
    grads = torch.autograd.grad([out, final], leaves, [dd.to(DEV), ds.to(DEV)])
    return [x.detach().cpu() for x in (out, final, *grads)]

  clean = run(0.0)
  for filler in (math.inf, math.nan):
    got = run(filler)
    for name, x, w in zip(("out", "grad_q", "grad_k", "grad_v"), (got[0], *got[2:5]), (clean[0], *clean[2:5])):
      ok = ~sick
      # the same values, chunks cut differently: two results of one formula, each within the bound of the other tests
      assert torch.isfinite(x[ok]).all(), name
      assert torch.allclose(x[ok].float(), w[ok].float(), rtol=16 * ref.HALF[dtype], atol=16 * ref.HALF[dtype] * float(w.abs().max())), name
    live = [b for b in range(n) if not sick[t - 1, b]]
    assert torch.isfinite(got[1][live]).all()
    assert torch.isfinite(got[5][[1, 3]]).all()


FEW = [
  # steps, rows, heads, kv heads, key dim, value dim, P(fresh), states
  (1, 5, 2, 2, 32, 32, 0.0, True), (2, 3, 2, 1, 7, 5, 0.3, True), (8, 70, 2, 1, 32, 32, 0.2, True), (16, 33, 1, 1, 16, 16, 0.1, False), (16, 9, 3, 3, 29, 31, 0.1, True),
  (8, 6, 2, 2, 64, 64, 0.1, True), (5, 4, 2, 2, 64, 3, 0.2, True), (16, 7, 2, 1, 3, 64, 0.2, True), (15, 5, 2, 1, 33, 12, 0.3, True), (17, 5, 2, 1, 33, 12, 0.3, True),
  (16, 8, 1, 1, 1, 1, 0.2, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", FEW, ids=lambda c: "-".join(str(x) for x in c))
def test_segments_of_few_steps(case, dtype):
  test_memory_scan_and_its_gradients(case, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_steps_keep_what_is_not_finite_inside_its_episode(dtype):
  from envpool_amd import policy
  t, n, h, dk, dv = 12, 3, 2, 32, 16
  q, k, v, decay, _, state, do, ds = _scan_problem((t, n, h, h, dk, dv, 0.0, True), dtype)
  fresh = torch.zeros(t, n, dtype=torch.bool)
  fresh[[3, 7], 0] = True
  fresh[5, 1] = True

  def run(filler):
    kk, vv, dd = k.clone(), v.clone(), do.clone()
    for x in (kk, vv, dd):
      x[4, 0] = x[2, 1] = filler
    leaves = [x.to(DEV).requires_grad_() for x in (q, kk, vv, state)]
    out, final = policy.memory_scan(*leaves[:3], decay.to(DEV), fresh=fresh.to(DEV), state=leaves[3])
    return [x.detach().cpu() for x in (out, final, *torch.autograd.grad([out, final], leaves, [dd.to(DEV), ds.to(DEV)]))]

  well = torch.ones(t, n, dtype=torch.bool)
  well[3:7, 0] = False
  well[:5, 1] = False
  clean, sick = run(0.0), run(math.inf)
  for x, w in zip((sick[0], *sick[2:5]), (clean[0], *clean[2:5])):
    assert torch.equal(x[well], w[well])
  assert torch.equal(sick[1], clean[1]) and torch.equal(sick[5][[0, 2]], clean[5][[0, 2]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,h,dk,dv", [(16, 4, 12, 64, 64), (32, 40, 4, 16, 16), (30, 3, 2, 128, 128), (17, 5, 3, 20, 19)])
def test_states_keep_32_bits(t, n, h, dk, dv, dtype):
  """The final state and the first state's gradient of one chunk, whatever the type of what goes in: a term is off by
  at most 2^-22 (two pieces of 11 bits), the decay's power by 2 half steps of its exponent (at most 32 * 0.42 octaves,
  each worth ln 2: 19 half steps of 32 bits) and 2 of its own, the sum by one per term."""
  from envpool_amd import policy
  q, k, v, decay, fresh, state, do, ds = _scan_problem((t, n, h, h, dk, dv, 0.02, True), dtype)
  args = dict(fresh=fresh, state=state, scale=1.0, grad_out=do, reverse_from=ds)
  want, size = ref.scan(q, k, v, decay, **args), ref.scan(q, k, v, decay, absolute=True, **args)
  leaf = state.to(DEV).requires_grad_()
  out, final = policy.memory_scan(q.to(DEV), k.to(DEV), v.to(DEV), decay.to(DEV), fresh=fresh.to(DEV), state=leaf, scale=1.0)
  grad, = torch.autograd.grad([out, final], leaf, [do.to(DEV), ds.to(DEV)])
  h32 = ref.HALF[torch.float32]
  for name, x in (("final", final.detach()), ("grad_state", grad)):
    err = (x.cpu().double() - want[name]).abs()
    tol = size[name] * (4 + 19 + 2 + t + 2) * h32 + h32 * want[name].abs() + 2.0**-30
    assert (err <= tol).all(), (name, float((err - tol).max()), float((err / size[name].clamp_min(1e-30)).max()))


def test_memory_scan_layouts_and_missing_pieces():
  """Batch-major views, expanded heads, no fresh, no state, no steps, nothing wanted from one of the outputs."""
  from envpool_amd import policy
  g = _gen(2)
  t, n, h, dk, dv = 90, 3, 2, 24, 40
  q = torch.randn(n, t, h, dk, generator=g).to(DEV).transpose(0, 1)
  k = torch.randn(h, n, t, dk, generator=g).to(DEV).permute(2, 1, 0, 3)
  v = torch.randn(t, n, 1, dv, generator=g).to(DEV).expand(t, n, h, dv)
  state = torch.randn(n, h, dv, dk, generator=g).to(DEV).transpose(2, 3)
  fresh = (torch.rand(n, t, generator=g) < 0.05).to(DEV).t()
  decay = _decay(h).to(DEV)
  a = policy.memory_scan(q, k, v, decay, fresh=fresh, state=state)
  b = policy.memory_scan(q.contiguous(), k.contiguous(), v.contiguous(), decay, fresh=fresh.contiguous().to(torch.uint8), state=state.contiguous())
  assert all(torch.equal(x, y) for x, y in zip(a, b))
  # in two parts, the state handed on
  o1, s1 = policy.memory_scan(q[:37], k[:37], v[:37], decay, fresh=fresh[:37], state=state)
  o2, s2 = policy.memory_scan(q[37:], k[37:], v[37:], decay, fresh=fresh[37:], state=s1)
  assert torch.allclose(torch.cat([o1, o2]), a[0], atol=1e-4, rtol=1e-4) and torch.allclose(s2, a[1], atol=1e-4, rtol=1e-4)
  o, s = policy.memory_scan(q[:0], k[:0], v[:0], decay, state=state)
  assert o.shape == (0, n, h, dv) and torch.equal(s, state)
  o, s = policy.memory_scan(q[:, :0], k[:, :0], v[:, :0], decay)
  assert o.shape == (t, 0, h, dv) and s.shape == (0, h, dk, dv)
  z = torch.zeros(n, h, dk, dv, device=DEV)
  none, zero = policy.memory_scan(q, k, v, decay), policy.memory_scan(q, k, v, decay, fresh=torch.zeros_like(fresh), state=z)
  assert all(torch.equal(x, y) for x, y in zip(none, zero))
  leaf = k.detach().requires_grad_()
  out, final = policy.memory_scan(q, leaf, v, decay, state=state)
  both, = torch.autograd.grad([out.sum(), final.sum()], leaf, [torch.ones((), device=DEV)] * 2, retain_graph=True)
  first, = torch.autograd.grad(out.sum(), leaf, retain_graph=True)
  second, = torch.autograd.grad(final.sum(), leaf)
  assert torch.allclose(first + second, both, atol=1e-4, rtol=1e-4)


@pytest.mark.parametrize("t,n,dk,dv,dtype", [(300, 260, 64, 48, torch.bfloat16), (130, 600, 16, 64, torch.float16), (1, 3, 8, 8, torch.float16)])
def test_gradients_of_keys_and_values_together_and_alone(t, n, dk, dv, dtype):
  """Many envs: one walk serves both gradients; each is what its own walk gives."""
  from envpool_amd import policy
  q, k, v, decay, fresh, state, do, ds = (x.to(DEV) for x in _scan_problem((t, n, 2, 1, dk, dv, 0.01, True), dtype))

  def run(wanted, start):
    leaves = [x.detach().requires_grad_(i in wanted) for i, x in enumerate((q, k, v, state))]
    out, final = policy.memory_scan(*leaves[:3], decay, fresh=fresh, state=leaves[3] if start else None)
    return torch.autograd.grad([out, final], [leaves[i] for i in wanted], [do, ds])

  for start in (True, False):
    together = run((1, 2), start)
    assert torch.equal(together[0], run((1,), start)[0]) and torch.equal(together[1], run((2,), start)[0])
  keys, first = run((1, 3), True)
  assert torch.equal(keys, run((1,), True)[0]) and torch.equal(first, run((3,), True)[0])


@pytest.mark.parametrize("t,dk,dv", [(70, 24, 40), (300, 128, 128), (33, 7, 5)])
def test_memory_scan_only_what_is_asked_for(t, dk, dv):
  """Each gradient alone (the others are not computed) is what it is among the others."""
  from envpool_amd import policy
  q, k, v, decay, fresh, state, do, ds = (x.to(DEV) for x in _scan_problem((t, 2, 2, 1, dk, dv, 0.02, True), torch.bfloat16))

  def run(wanted):
    leaves = [x.detach().requires_grad_(i in wanted) for i, x in enumerate((q, k, v, state))]
    out, final = policy.memory_scan(*leaves[:3], decay, fresh=fresh, state=leaves[3])
    return torch.autograd.grad([out, final], [leaves[i] for i in wanted], [do, ds])

  every = run((0, 1, 2, 3))
  for i in range(4):
    assert torch.equal(run((i,))[0], every[i])


def test_memory_scan_agrees_with_steps():
  """The acting path and the learning path are one memory: T steps of EnvMemory against one scan."""
  from envpool_amd import policy
  g = _gen(21)
  t, n, h, hk, dk, dv = 70, 5, 4, 2, 32, 48
  q, k, v = (torch.randn(t, n, x, d, generator=g).to(DEV) for x, d in ((h, dk), (hk, dk), (hk, dv)))
  fresh = (torch.rand(t, n, generator=g) < 0.1).to(DEV)
  decay = _decay(h).to(DEV)
  mem = policy.EnvMemory(n, h, dk, dv, decay)
  outs = torch.stack([mem.step(q[i], k[i], v[i], fresh=fresh[i]) for i in range(t)])
  out, final = policy.memory_scan(q, k, v, decay, fresh=fresh)
  size = float(out.abs().max())
  assert (outs - out).abs().max() <= 1e-5 * size and (mem.state - final).abs().max() <= 1e-5 * float(final.abs().max())
