"""The policy-side operators from their definitions, in 64 bits on the CPU, one row or step at a time where that
is the plainest way to say it. Test infrastructure."""
import math

import torch

HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step, relative

TINY = {torch.float32: 2.0**-126, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-126}  # results below may be flushed or denormal


def cpu64(t):
  return None if t is None else t.detach().cpu().double()


def processed(logits, num_options=None, mask=None, bias=None, history=None, repetition=1.0, frequency=0.0, presence=0.0, temperature=1.0):
  """-> (y [B, A] with -inf where illegal, legal, slope d y / d logit, 1 / temperature [B, 1], magnitude of what y was made of)."""
  x = cpu64(logits).clone()
  n, a = x.shape
  col = lambda v: cpu64(v)[:, None] if isinstance(v, torch.Tensor) else torch.full((n, 1), float(v), dtype=torch.float64)  # noqa: E731
  rep, freq, pres, temp = col(repetition), col(frequency), col(presence), col(temperature)
  legal = torch.ones(n, a, dtype=torch.bool)
  if num_options is not None:
    legal &= torch.arange(a)[None] < num_options.cpu()[:, None]
  if mask is not None:
    m = mask.cpu()
    if m.dim() == 1:
      m = m[None]
    if m.dtype == torch.int32:
      j = torch.arange(a)
      m = (m[:, j // 32].long() >> (j % 32)) & 1
    legal &= m != 0
  slope = torch.ones(n, a, dtype=torch.float64)
  size = x.abs()
  if history is not None:
    h = history.cpu().long()
    h = h[None].expand(n, -1) if h.dim() == 1 else h
    count = torch.zeros(n, a + 1, dtype=torch.float64)
    h = torch.where((h < 0) | (h >= a), a, h)
    count.scatter_add_(1, h, torch.ones_like(h, dtype=torch.float64))
    count = count[:, :a]
    seen = count > 0
    slope = torch.where(seen, torch.where(x > 0, 1 / rep, rep), slope)
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    cut = freq * count
    size = torch.maximum(size, x.abs()) + torch.where(seen, cut.abs() + pres.abs(), 0.0)
    x = torch.where(seen, x - cut - pres, x)
  if bias is not None:
    b = cpu64(bias)
    x = x + b
    size = size + b.abs()
  y = torch.where(legal, x / temp, -math.inf)
  return y, legal, slope / temp, 1 / temp, torch.where(legal, size, 0.0) / temp


def distribution(y):
  """-> (m, w, S, empty, bad) of y [B, A]."""
  bad = torch.isnan(y).any(1) | (y == math.inf).any(1)
  m = torch.where(torch.isnan(y), -math.inf, y).max(1, keepdim=True).values
  empty = (m[:, 0] == -math.inf) & ~bad
  ref = torch.where(m.isinf(), 0.0, m)
  w = torch.exp(y - ref)
  return ref, w, w.sum(1), empty, bad


def choose(logits, u=None, **kw):
  y, legal, *_ = processed(logits, **kw)
  m, w, total, empty, bad = distribution(y)
  n, a = y.shape
  action = torch.full((n,), -1, dtype=torch.int64)
  for b in range(n):
    if empty[b] or bad[b]:
      continue
    if u is None:
      action[b] = int(torch.nonzero(y[b] == y[b].max())[0])
    else:
      cum = torch.cumsum(w[b], 0)
      hit = torch.nonzero((cum > float(u[b].double()) * float(cum[-1])) & (w[b] > 0))
      action[b] = int(hit[0]) if len(hit) else int(torch.nonzero(w[b] > 0)[-1])
  z = y - m
  log_s = torch.log(total)
  pick = z.gather(1, action.clamp_min(0)[:, None])[:, 0] - log_s
  ent = log_s - torch.where(w > 0, w * z, 0.0).sum(1) / total
  fix = lambda v: torch.where(bad, math.nan, torch.where(empty, 0.0, v))  # noqa: E731
  return action, fix(pick), fix(ent)


def evaluate(logits, action, g_lp, g_h, **kw):
  """-> dict of log_prob, entropy, grad_logits, grad_bias (per row), and the bounds of a 32-bit evaluation's errors."""
  y, legal, slope, inv_t, size = processed(logits, **kw)
  m, w, total, empty, bad = distribution(y)
  n, a = y.shape
  z = torch.where(w > 0, y - m, 0.0)
  log_s = torch.log(torch.where(total > 0, total, 1.0))  # (rows without a weight: 0 / 0 would reach the bounds)
  p = torch.where(w > 0, w / total[:, None], 0.0)
  logp = torch.where(w > 0, z - log_s[:, None], 0.0)
  act = action.cpu().long()
  inside = (act >= 0) & (act < a)
  at = act.clamp(0, a - 1)[:, None]
  lp = (y - m).gather(1, at)[:, 0] - log_s
  lp = torch.where(empty, -math.inf, lp)
  lp = torch.where(inside, lp, torch.where(act == -1, 0.0, math.nan))
  ent = torch.where(empty, 0.0, log_s - (w * z).sum(1) / total)
  lp, ent = torch.where(bad, math.nan, lp), torch.where(bad, math.nan, ent)
  one = torch.zeros(n, a, dtype=torch.float64)
  one.scatter_(1, at, (inside & ~empty).double()[:, None])
  g1, g2 = torch.where(act == -1, 0.0, cpu64(g_lp))[:, None], cpu64(g_h)[:, None]
  dy = torch.where(legal, g1 * (one - p) - g2 * p * (logp + ent[:, None]), 0.0)
  dy = torch.where(empty[:, None], 0.0, dy)
  dy = torch.where(bad[:, None] & legal, math.nan, dy)
  # 32-bit evaluation, h = 2^-24. z: at most five roundings of values up to `size`; a difference of two z, times
  # 1/T (rounded twice), in the exponent as a product with log2 e (rounded once more, the hardware exponential
  # good to 2 h): relative error of a weight r <= h (10 size + 4 |d| + 4). The sums: A/2048 * 8 additions of a
  # thread, 10 levels across threads. log S takes S's relative error over; one more rounding of each result.
  h = HALF[torch.float32]
  big = size.max(1).values.nan_to_num(0.0, 0.0, 0.0).clamp(max=1e30)
  far = torch.where(w > 0, (y - m).abs(), 0.0).max(1).values
  mean_far = (p * z.abs()).sum(1)
  r_sum = h * (10 * big + 4 * mean_far + 4 + a / 256 + 16)
  z_act = torch.where(inside, z.gather(1, at)[:, 0].abs(), 0.0)
  tol_lp = r_sum + h * (10 * big + 3 * z_act + log_s.abs() + 4)
  tol_h = h * (log_s.abs() + 4) + r_sum * (2 + 2 * mean_far) + h * (10 * big + 4 * (p * z * z).sum(1) + 8 * mean_far)
  r_p = (r_sum + h * (10 * big + 8))[:, None] + h * (4 * z.abs() + 2 * logp.abs())
  tol_y = g1.abs() * (p * r_p + 4 * h) + g2.abs() * p * ((logp + ent[:, None]).abs() * (r_p + 4 * h) + tol_h[:, None] + r_p) + 4 * h * dy.abs()
  return {"log_prob": lp, "entropy": ent, "grad_logits": dy * slope, "grad_bias": dy * inv_t, "tol_log_prob": tol_lp, "tol_entropy": tol_h,
          "tol_logits": tol_y * slope.abs() * (1 + 4 * h), "tol_bias": tol_y * inv_t * (1 + 4 * h)}


def scan(q, k, v, log_decay, fresh=None, state=None, scale=1.0, reverse_from=None, absolute=False, grad_out=None):
  """The recurrence in 64 bits. q [T, B, H, Dk], k, v with their own number of heads. With grad_out (and
  reverse_from, the gradient of the final state) also the gradients. absolute: every operand's magnitude, for bounds."""
  f = (lambda t: cpu64(t).abs()) if absolute else cpu64
  q, k, v = f(q), f(k), f(v)
  t_all, n, h, dk = q.shape
  dv, group = v.shape[3], h // k.shape[2]
  k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
  lam = torch.exp(cpu64(log_decay))[None, :, None, None]
  s = torch.zeros(n, h, dk, dv, dtype=torch.float64) if state is None else f(state).clone()
  keep = lambda t: (0.0 if fresh is None else (fresh[t].cpu() != 0)).double()[:, None, None, None] if fresh is not None else torch.zeros(n, 1, 1, 1).double()  # noqa: E731
  out, gq = [], []
  go = None if grad_out is None else f(grad_out)
  for t in range(t_all):
    s = torch.where(keep(t) > 0, 0.0, s * lam) + k[t][..., :, None] * v[t][..., None, :]
    out.append(scale * torch.einsum("bhd,bhde->bhe", q[t], s))
    if go is not None:
      gq.append(scale * torch.einsum("bhe,bhde->bhd", go[t], s))
  res = {"out": torch.stack(out) if out else torch.zeros(0, n, h, dv).double(), "final": s}
  if go is not None:
    g = torch.zeros(n, h, dk, dv, dtype=torch.float64) if reverse_from is None else f(reverse_from).clone()
    gk, gv = [None] * t_all, [None] * t_all
    for t in reversed(range(t_all)):
      g = g + scale * q[t][..., :, None] * go[t][..., None, :]
      gk[t] = torch.einsum("bhde,bhe->bhd", g, v[t])
      gv[t] = torch.einsum("bhde,bhd->bhe", g, k[t])
      g = torch.where(keep(t) > 0, 0.0, g * lam)
    join = lambda x: torch.stack(x).unflatten(2, (-1, group)).sum(3)  # noqa: E731
    res.update(grad_q=torch.stack(gq), grad_k=join(gk), grad_v=join(gv), grad_state=g)
  return res
