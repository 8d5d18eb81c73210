"""What the policy-side operators are measured on: the choice of an action under the pool's mask,
the log-probability and entropy of stored actions with their gradients, one step of the envs'
memory, and the memory over a rollout segment with its gradients.

`own` False: the plain form, elementary torch operations. `own` True: envpool_amd.policy."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the cases -----------------------------------------------------------------------------------
def _choose(name, rows, options, dtype, mask="count", bias="", history=0, greedy=False, per_row=False):
  return {"name": name, "op": "choose", "rows": rows, "options": options, "dtype": dtype, "mask": mask, "bias": bias,
          "history": history, "greedy": greedy, "per_row": per_row}


def _evaluate(name, rows, options, dtype, mask="count", bias="", history=0):
  return {"name": name, "op": "evaluate", "rows": rows, "options": options, "dtype": dtype, "mask": mask, "bias": bias,
          "history": history, "greedy": False, "per_row": False}


def _step(name, envs, rows, heads, key_dim, value_dim, dtype):
  return {"name": name, "op": "step", "envs": envs, "rows": rows, "heads": heads, "key_dim": key_dim, "value_dim": value_dim,
          "dtype": dtype}


def _scan(name, steps, rows, heads, kv_heads, key_dim, value_dim, dtype, train, fresh):
  return {"name": name, "op": "scan", "steps": steps, "rows": rows, "heads": heads, "kv_heads": kv_heads, "key_dim": key_dim,
          "value_dim": value_dim, "dtype": dtype, "train": train, "fresh": fresh}


def listed():
  return [
    # one batch of the default YGOPro pool: 1024 duels, 16 options, as many legal as num_options says; latency
    _choose("choose-duels", 1024, 16, "f32"),
    # all envs of a node's pool in one go, byte mask as the encoder writes it, one bias for all rows
    _choose("choose-node", 524288, 16, "bf16", mask="bytes", bias="shared"),
    # a policy that answers in tokens: a grammar's bit mask, penalties on what the episode has said so far
    _choose("choose-tokens", 64, 131072, "bf16", mask="bits", bias="shared", history=2048, per_row=True),
    # one minibatch of stored duels
    _evaluate("evaluate-duels", 4096, 16, "f32"),
    # a whole rollout of a large pool at once
    _evaluate("evaluate-rollout", 524288, 24, "bf16", mask="bytes", bias="shared"),
    # stored token answers
    _evaluate("evaluate-tokens", 2048, 32768, "bf16", mask="bits", bias="shared"),
    # the smallest pool, stepped once: latency
    _step("step-8", 8, 8, 4, 64, 64, "f32"),
    # an async pool's batch: half the envs, in arrival order
    _step("step-async", 8192, 4096, 8, 64, 64, "bf16"),
    # every env of the 65 536-env pool
    _step("step-pool", 65536, 65536, 4, 32, 32, "f16"),
    # a training segment of a rollout: 128 steps of 1024 envs, episodes end inside
    _scan("scan-rollout", 128, 1024, 4, 4, 64, 64, "bf16", True, 0.02),
    # one long episode read back at once: few rows, long axis
    _scan("scan-episode", 32768, 1, 16, 16, 128, 128, "bf16", False, 0.0),
    # odd sizes in 32 bits, keys and values shared by three heads each, with gradients
    _scan("scan-odd", 777, 5, 6, 2, 80, 112, "f32", True, 0.01),
  ]


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(["choose", "evaluate", "step", "scan"])
  dtype = rng.choice(["f32", "bf16", "f16"])
  if op in ("choose", "evaluate"):
    options = rng.choice([16, 24, _log_int(rng, 2, 64), _log_int(rng, 64, 131072), _log_int(rng, 1000, 131072)])
    budget = 8388608 if op == "choose" else 33554432
    rows = _log_int(rng, 1, max(1, min(524288, budget // options)))
    mask = rng.choice(["count", "bytes", "bits", "none"])
    bias = rng.choice(["", "shared", "rows"])
    history = rng.choice([0, 0, _log_int(rng, 1, min(2048, max(1, budget // (4 * rows))))])
    if op == "choose":
      return _choose("", rows, options, dtype, mask, bias, history, rng.random() < 0.25, rng.random() < 0.5)
    return _evaluate("", rows, options, dtype, mask, bias, history)
  heads = rng.choice([1, 2, 3, 4, 8, 12, 16])
  key_dim = rng.choice([16, 32, 64, 64, 128, rng.randint(1, 128)])
  value_dim = rng.choice([key_dim, 32, 64, 128, rng.randint(1, 128)])
  if op == "step":
    envs = _log_int(rng, 1, max(1, min(65536, 268435456 // (heads * key_dim * value_dim))))
    rows = rng.choice([envs, max(1, envs // 2), rng.randint(1, envs)])
    return _step("", envs, rows, heads, key_dim, value_dim, dtype)
  steps = _log_int(rng, 1, 16384)
  rows = _log_int(rng, 1, max(1, min(4096, 33554432 // (steps * heads * max(key_dim, value_dim)))))
  kv_heads = rng.choice([h for h in (heads, heads, 1, 2, 4) if heads % h == 0])
  return _scan("", steps, rows, heads, kv_heads, key_dim, value_dim, dtype, rng.random() < 0.6, rng.choice([0.0, 0.01, 0.1]))


def work(case):
  b = _BYTES[case["dtype"]]
  if case["op"] in ("choose", "evaluate"):
    n, a = case["rows"], case["options"]
    row = a * b + {"count": 4, "bytes": a, "bits": 4 * ((a + 31) // 32), "none": 0}[case["mask"]] + 4 * case["history"]
    row += {"": 0, "shared": 0, "rows": 4 * a}[case["bias"]]
    shared = 4 * a if case["bias"] == "shared" else 0
    if case["op"] == "choose":
      row += (0 if case["greedy"] else 4) + 12 + (16 if case["per_row"] else 0)
      return {"bytes": n * row + shared, "flops": 12 * n * a}
    row += 4 + 8 + 8 + a * b + (4 * a if case["bias"] == "rows" else 0)  # action, two results, two gradients in; the logits' gradient out
    return {"bytes": n * row + 2 * shared, "flops": 24 * n * a}
  h, dk, dv = case["heads"], case["key_dim"], case["value_dim"]
  if case["op"] == "step":
    n = case["rows"] * h
    return {"bytes": n * (8 * dk * dv + b * (2 * dk + 2 * dv)) + 8 * case["rows"], "flops": 5 * n * dk * dv}
  t, n, hk = case["steps"], case["rows"], case["kv_heads"]
  qo, kv, st = t * n * h * b, t * n * hk * b * (dk + dv), n * h * dk * dv * 4
  total = qo * (dk + dv) + kv + 2 * st + t * n
  flops = 4 * t * n * h * dk * dv
  if case["train"]:
    total += qo * (dk + dv) + kv + 2 * st
    flops += 8 * t * n * h * dk * dv
  return {"bytes": total, "flops": flops}


# ---- inputs --------------------------------------------------------------------------------------
def _bits_of(mask):
  rows, options = mask.shape
  words = (options + 31) // 32
  out = torch.zeros(rows, words, dtype=torch.int32, device=mask.device)
  for i in range(32):
    col = mask[:, i::32]
    out[:, :col.shape[1]] |= col.to(torch.int32) << i if i < 31 else col.to(torch.int32) * (-2147483648)
  return out


def _inputs(case, seed):
  """The tensors of a case, from the seed alone."""
  dev = torch.device("cuda")
  gen = torch.Generator(device=dev).manual_seed(seed)
  dt = _TYPES[case["dtype"]]

  def randn(*shape):
    return torch.randn(shape, generator=gen, device=dev)

  def rand(*shape):
    return torch.rand(shape, generator=gen, device=dev)

  if case["op"] in ("choose", "evaluate"):
    n, a = case["rows"], case["options"]
    s = {"logits": (3.0 * randn(n, a)).to(dt), "num_options": None, "mask": None, "bias": None, "history": None,
         "repetition": 1.0, "frequency": 0.0, "presence": 0.0, "temperature": 0.7 if case["op"] == "choose" else 1.0}
    empty = rand(n) < 0.01  # rows whose env has ended: nothing is legal
    if case["mask"] == "count":
      count = (1 + (rand(n) * a).to(torch.int32)).clamp(max=a)
      s["num_options"] = torch.where(empty, 0, count).to(torch.int32)
      action = (rand(n) * count).to(torch.int32)
      action = torch.minimum(action, count - 1)
    else:
      action = (rand(n) * a).to(torch.int32).clamp(max=a - 1)
      if case["mask"] != "none":
        legal = rand(n, a) < 0.4
        legal[torch.arange(n, device=dev), action.long()] = True
        legal &= ~empty[:, None]
        s["mask"] = legal if case["mask"] == "bytes" else _bits_of(legal)
      else:
        empty = torch.zeros_like(empty)
    if case["bias"]:
      s["bias"] = 0.5 * (randn(a) if case["bias"] == "shared" else randn(n, a))
    if case["history"]:
      # what was chosen before repeats itself; the unused end of a short history holds -1
      hist = (rand(n, case["history"]) ** 3 * a).to(torch.int32).clamp(max=a - 1)
      used = rand(n, 1) * (case["history"] + 1)
      s["history"] = torch.where(torch.arange(case["history"], device=dev)[None, :] < used, hist, -1).to(torch.int32)
      s["repetition"], s["frequency"], s["presence"] = 1.2, 0.1, 0.3
    if case["op"] == "choose":
      s["u"] = None if case["greedy"] else rand(n)
      if case["per_row"]:
        s["temperature"] = 0.5 + rand(n)
        if case["history"]:
          s["repetition"], s["frequency"], s["presence"] = 1.0 + 0.5 * rand(n), 0.2 * rand(n), 0.5 * rand(n)
    else:
      s["action"] = torch.where(empty, -1, action).to(torch.int32)
      s["grad_log_prob"], s["grad_entropy"] = randn(n), 0.01 * randn(n)
    return s
  h, dk, dv = case["heads"], case["key_dim"], case["value_dim"]
  decay = torch.log1p(-torch.exp2(-5.0 - 4.0 * torch.arange(h, device=dev, dtype=torch.float64) / h)).float()
  if case["op"] == "step":
    n = case["rows"]
    ids = torch.randperm(case["envs"], generator=gen, device=dev)[:n].to(torch.int32)
    elapsed = (rand(n) * 20).to(torch.int32)  # 0: the first step of an episode
    return {"q": randn(n, h, dk).to(dt), "k": (randn(n, h, dk) / math.sqrt(dk)).to(dt), "v": randn(n, h, dv).to(dt),
            "log_decay": decay, "env_id": ids, "elapsed_step": elapsed, "state": randn(case["envs"], h, dk, dv)}
  t, n, hk = case["steps"], case["rows"], case["kv_heads"]
  s = {"q": randn(t, n, h, dk).to(dt), "k": (randn(t, n, hk, dk) / math.sqrt(dk)).to(dt), "v": randn(t, n, hk, dv).to(dt),
       "log_decay": decay, "fresh": rand(t, n) < case["fresh"], "state": randn(n, h, dk, dv)}
  if case["train"]:
    s["grad_out"], s["grad_state"] = randn(t, n, h, dv).to(dt), 0.1 * randn(n, h, dk, dv)
  return s


def prepare(case, seed):
  s = _inputs(case, seed)
  s["case"] = case
  if own and case["op"] == "step":
    from envpool_amd.policy import EnvMemory
    s["memory"] = EnvMemory(case["envs"], case["heads"], case["key_dim"], case["value_dim"], s["log_decay"], state=s["state"])
  return s


# ---- the plain forms -----------------------------------------------------------------------------
def _col(x):
  return x[:, None] if isinstance(x, torch.Tensor) else x


def _legal(s, n, a, dev):
  legal = torch.ones(n, a, dtype=torch.bool, device=dev)
  if s["num_options"] is not None:
    legal &= torch.arange(a, device=dev)[None, :] < s["num_options"][:, None]
  m = s["mask"]
  if m is not None:
    if m.dtype == torch.int32:
      j = torch.arange(a, device=dev)
      m = (m[:, j // 32] >> (j % 32).to(torch.int32)) & 1 == 1
    legal &= m
  return legal


def _scaled(s, x, bias):
  """Penalties, bias and temperature, in x's type."""
  if s["history"] is not None:
    hist, a = s["history"], x.shape[1]
    ok = (hist >= 0) & (hist < a)
    count = torch.zeros_like(x).scatter_add_(1, hist.clamp(0, a - 1).long(), ok.to(x.dtype))
    r, f, p = (_col(s[k]) for k in ("repetition", "frequency", "presence"))
    x = torch.where(count > 0, torch.where(x > 0, x / r, x * r), x) - f * count - p * (count > 0).to(x.dtype)
  if bias is not None:
    x = x + bias
  return x / _col(s["temperature"])


def _plain_choose(s):
  x = s["logits"].double()
  n, a = x.shape
  legal = _legal(s, n, a, x.device)
  for k in ("repetition", "frequency", "presence", "temperature"):
    if isinstance(s[k], torch.Tensor):
      s = {**s, k: s[k].double()}
  y = torch.where(legal, _scaled(s, x, None if s["bias"] is None else s["bias"].double()), -math.inf)
  m = y.max(1, keepdim=True).values
  empty = m[:, 0] == -math.inf
  m = torch.where(m == -math.inf, 0.0, m)
  w = torch.exp(y - m)
  cum = torch.cumsum(w, 1)
  total = cum[:, -1:]
  cols = torch.arange(a, device=x.device)[None, :]
  if s["u"] is None:
    action = torch.where(legal & (y == m), cols, a).min(1).values
  else:
    action = torch.where(legal & (cum > s["u"].double()[:, None] * total), cols, a).min(1).values
    last = torch.where(w > 0, cols, -1).max(1).values
    action = torch.minimum(action, last)
  action = torch.where(empty, -1, action)
  z = torch.where(w > 0, y - m, 0.0)
  log_s = torch.log(total[:, 0])
  log_prob = torch.where(empty, 0.0, z.gather(1, action.clamp(0, a - 1)[:, None])[:, 0] - log_s)
  entropy = torch.where(empty, 0.0, log_s - (w * z).sum(1) / total[:, 0])
  return {"action": action.int(), "log_prob": log_prob.float(), "entropy": entropy.float()}


def _evaluated(log_prob, entropy, grads):
  return {"log_prob": log_prob.detach(), "entropy": entropy.detach(), **dict(zip(("grad_logits", "grad_bias"), grads))}


def _plain_evaluate(s):
  logits = s["logits"].detach().requires_grad_()
  leaves = [logits]
  bias = None
  if s["bias"] is not None:
    bias = s["bias"].detach().requires_grad_()
    leaves.append(bias)
  n, a = logits.shape
  legal = _legal(s, n, a, logits.device)
  empty = ~legal.any(1)
  y = torch.where(legal, _scaled(s, logits.float(), bias), -1e30)
  z = y - y.detach().max(1, keepdim=True).values
  w = torch.where(legal, torch.exp(z), 0.0)
  total = w.sum(1).clamp_min(1e-30)
  log_s = torch.log(total)
  picked = z.gather(1, s["action"].clamp_min(0).long()[:, None])[:, 0] - log_s
  log_prob = torch.where(empty, 0.0, picked)
  entropy = torch.where(empty, 0.0, log_s - (w * torch.where(legal, z, 0.0)).sum(1) / total)
  grads = torch.autograd.grad([log_prob, entropy], leaves, [s["grad_log_prob"], s["grad_entropy"]])
  return _evaluated(log_prob, entropy, grads)


def _plain_step(s):
  ids = s["env_id"].long()
  q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
  keep = (s["elapsed_step"] != 0).float()[:, None] * torch.exp(s["log_decay"])[None, :]
  state = s["state"].index_select(0, ids) * keep[:, :, None, None]
  state = state + k[:, :, :, None] * v[:, :, None, :]
  s["state"].index_copy_(0, ids, state)
  out = torch.matmul(q[:, :, None, :], state)[:, :, 0] * q.shape[-1] ** -0.5
  return {"out": out.to(s["q"].dtype), "state": s["state"]}


def _chunked(q, k, v, log_decay, fresh, state):
  """q, k, v [B, H, T, D] in 32 bits, chunk by chunk; -> out, final state."""
  outs = []
  t_all = q.shape[2]
  a = log_decay[None, :, None]
  for t0 in range(0, t_all, 64):
    n = min(64, t_all - t0)
    qc, kc, vc = q[:, :, t0:t0 + n], k[:, :, t0:t0 + n], v[:, :, t0:t0 + n]
    seg = torch.cumsum(fresh[t0:t0 + n].t().to(torch.int32), 1)[:, None, :]  # [B, 1, n]
    i = torch.arange(n, device=q.device)
    gap = (i[:, None] - i[None, :]).clamp_min(0).float()
    same = (seg[..., :, None] == seg[..., None, :]) & (i[:, None] >= i[None, :])
    inner = torch.matmul(qc, kc.transpose(2, 3)) * torch.where(same, torch.exp(a[..., None] * gap), 0.0)
    carry = torch.exp(a * (i + 1).float()) * (seg == 0).float()
    outs.append(torch.matmul(inner, vc) + torch.matmul(qc * carry[..., None], state))
    left = torch.exp(a * (n - 1 - i).float()) * (seg == seg[..., -1:]).float()
    state = state * (torch.exp(a * n) * (seg[..., -1:] == 0).float())[..., None] + torch.matmul((kc * left[..., None]).transpose(2, 3), vc)
  return torch.cat(outs, 2), state


def _plain_scan(s):
  case = s["case"]
  group = case["heads"] // case["kv_heads"]
  train = case["train"]
  names = ("q", "k", "v", "state")
  leaves = [s[x].detach().requires_grad_(train) for x in names]
  q, k, v = (x.float().permute(1, 2, 0, 3) for x in leaves[:3])
  if group > 1:
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
  out, final = _chunked(q * case["key_dim"] ** -0.5, k, v, s["log_decay"], s["fresh"], leaves[3])
  out = out.permute(2, 0, 1, 3).to(s["q"].dtype)
  res = {"out": out.detach(), "final_state": final.detach()}
  if train:
    grads = torch.autograd.grad([out, final], leaves, [s["grad_out"], s["grad_state"]])
    res.update({"grad_" + x: g for x, g in zip(("q", "k", "v", "initial"), grads)})
  return res


# ---- one pass ------------------------------------------------------------------------------------
def _options(s):
  return {k: s[k] for k in ("num_options", "mask", "bias", "history", "repetition", "frequency", "presence", "temperature")}


def _own_choose(s):
  from envpool_amd import policy
  c = policy.choose(s["logits"], s["u"], **_options(s))
  return {"action": c.action, "log_prob": c.log_prob, "entropy": c.entropy}


def _own_evaluate(s):
  from envpool_amd import policy
  leaves = [s["logits"].detach().requires_grad_()]
  opts = _options(s)
  if s["bias"] is not None:
    opts["bias"] = s["bias"].detach().requires_grad_()
    leaves.append(opts["bias"])
  log_prob, entropy = policy.evaluate(leaves[0], s["action"], **opts)
  grads = torch.autograd.grad([log_prob, entropy], leaves, [s["grad_log_prob"], s["grad_entropy"]])
  return _evaluated(log_prob, entropy, grads)


def _own_step(s):
  out = s["memory"].step(s["q"], s["k"], s["v"], env_id=s["env_id"], elapsed_step=s["elapsed_step"])
  return {"out": out, "state": s["memory"].state}


def _own_scan(s):
  from envpool_amd import policy
  if not s["case"]["train"]:
    out, final = policy.memory_scan(s["q"], s["k"], s["v"], s["log_decay"], fresh=s["fresh"], state=s["state"])
    return {"out": out, "final_state": final}
  leaves = [s[x].detach().requires_grad_() for x in ("q", "k", "v", "state")]
  out, final = policy.memory_scan(*leaves[:3], s["log_decay"], fresh=s["fresh"], state=leaves[3])
  grads = torch.autograd.grad([out, final], leaves, [s["grad_out"], s["grad_state"]])
  res = {"out": out.detach(), "final_state": final.detach()}
  res.update({"grad_" + x: g for x, g in zip(("q", "k", "v", "initial"), grads)})
  return res


def run(state):
  op = state["case"]["op"]
  if own:
    return {"choose": _own_choose, "evaluate": _own_evaluate, "step": _own_step, "scan": _own_scan}[op](state)
  return {"choose": _plain_choose, "evaluate": _plain_evaluate, "step": _plain_step, "scan": _plain_scan}[op](state)


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_log_probs(s):
  """Row-wise log p (-inf where illegal), p, its gradient's factor d y / d x, and the empty rows."""
  x = s["logits"].double()
  n, a = x.shape
  dev = x.device
  slope = torch.ones_like(x)
  wide = {k: (s[k].double()[:, None].expand(n, a) if isinstance(s[k], torch.Tensor) else torch.full((n, a), s[k], dtype=x.dtype, device=dev))
          for k in ("repetition", "frequency", "presence", "temperature")}
  if s["history"] is not None:
    hist = s["history"].long()
    keep = (hist >= 0) & (hist < a)
    flat = (torch.arange(n, device=dev)[:, None] * a + hist)[keep]
    times = torch.bincount(flat, minlength=n * a).view(n, a).double()
    seen = times >= 1
    slope = torch.where(seen, torch.where(x > 0, 1.0 / wide["repetition"], wide["repetition"]), slope)
    x = x * slope
    x = x - wide["frequency"] * times
    x[seen] -= wide["presence"][seen]
  if s["bias"] is not None:
    x = x + s["bias"].double()
  y = x / wide["temperature"]
  slope = slope / wide["temperature"]
  off = torch.zeros(n, a, dtype=torch.bool, device=dev)
  if s["num_options"] is not None:
    off |= s["num_options"].long()[:, None] <= torch.arange(a, device=dev)
  if s["mask"] is not None:
    if s["mask"].dtype == torch.bool:
      off |= s["mask"].logical_not()
    else:
      planes = torch.stack([(s["mask"].long() >> i) % 2 for i in range(32)], 2).view(n, -1)[:, :a]
      off |= planes == 0
  y = y.masked_fill(off, -math.inf)
  log_p = y - torch.logsumexp(y, 1, keepdim=True)
  empty = off.all(1)
  log_p[empty] = -math.inf
  return y, log_p, log_p.exp(), slope, 1.0 / wide["temperature"], empty


def _exact_choose(s):
  y, log_p, p, _, _, empty = _exact_log_probs(s)
  a = y.shape[1]
  if s["u"] is None:
    best = y.max(1, keepdim=True).values
    action = (y == best).int().argmax(1)
  else:
    cum = p.cumsum(1)
    action = torch.searchsorted(cum, (s["u"].double() * cum[:, -1])[:, None], right=True)[:, 0].clamp(max=a - 1)
  lp = torch.where(empty, 0.0, log_p.gather(1, action[:, None])[:, 0])
  ent = -torch.where(p > 0, p * log_p, 0.0).sum(1)
  return {"action": torch.where(empty, -1, action).int(), "log_prob": lp, "entropy": ent}


def _exact_evaluate(s):
  _, log_p, p, slope, inv_t, empty = _exact_log_probs(s)
  act = s["action"].long()
  lp = torch.where(empty, 0.0, log_p.gather(1, act.clamp_min(0)[:, None])[:, 0])
  safe = torch.where(p > 0, log_p, 0.0)
  ent = -(p * safe).sum(1)
  one = torch.zeros_like(p)
  one[torch.arange(len(act), device=p.device), act.clamp_min(0)] = (act >= 0).double()
  g1, g2 = s["grad_log_prob"].double()[:, None], s["grad_entropy"].double()[:, None]
  dy = g1 * (one - p) - g2 * p * (safe + ent[:, None])
  dy[empty] = 0.0
  res = {"log_prob": lp, "entropy": ent, "grad_logits": dy * slope}
  if s["bias"] is not None:
    res["grad_bias"] = dy * inv_t if s["bias"].dim() == 2 else (dy * inv_t).sum(0)
  return res


def _exact_step(s):
  table = s["state"].double()
  out = torch.empty(s["q"].shape[:2] + (s["v"].shape[2],), dtype=torch.float64, device=table.device)
  lam = s["log_decay"].double().exp()
  ids = s["env_id"].long()
  for h in range(out.shape[1]):
    now = table[ids, h] * (lam[h] * (s["elapsed_step"] > 0).double())[:, None, None]
    now += torch.bmm(s["k"][:, h, :, None].double(), s["v"][:, h, None, :].double())
    table[ids, h] = now
    out[:, h] = torch.bmm(s["q"][:, h, None, :].double(), now)[:, 0] / math.sqrt(s["q"].shape[2])
  return {"out": out, "state": table}


def _exact_scan(s):
  case = s["case"]
  group = case["heads"] // case["kv_heads"]
  t_all, scale = case["steps"], 1.0 / math.sqrt(case["key_dim"])
  lam = s["log_decay"].double().exp()[None, :, None, None]
  stay = 1.0 - s["fresh"].double()[:, :, None, None, None]
  wide = lambda x, t: x[t].double().repeat_interleave(group, 1)  # noqa: E731
  state = s["state"].double()
  out = torch.empty(s["q"].shape[:3] + (case["value_dim"],), dtype=torch.float64, device=state.device)
  grad_q = torch.empty(s["q"].shape, dtype=torch.float64, device=state.device) if case["train"] else None
  for t in range(t_all):
    state = state * (lam * stay[t]) + wide(s["k"], t)[..., :, None] * wide(s["v"], t)[..., None, :]
    out[t] = scale * (s["q"][t].double()[..., :, None] * state).sum(2)
    if case["train"]:
      grad_q[t] = scale * (s["grad_out"][t].double()[..., None, :] * state).sum(3)
  res = {"out": out, "final_state": state}
  if not case["train"]:
    return res
  back = s["grad_state"].double()
  grad_k = torch.empty(s["k"].shape, dtype=torch.float64, device=state.device)
  grad_v = torch.empty(s["v"].shape, dtype=torch.float64, device=state.device)
  for t in reversed(range(t_all)):
    back = back + scale * s["q"][t].double()[..., :, None] * s["grad_out"][t].double()[..., None, :]
    per_k = (back * wide(s["v"], t)[..., None, :]).sum(3)
    per_v = (back * wide(s["k"], t)[..., :, None]).sum(2)
    grad_k[t] = per_k.unflatten(1, (-1, group)).sum(2)
    grad_v[t] = per_v.unflatten(1, (-1, group)).sum(2)
    back = back * (lam * stay[t])
  res.update({"grad_q": grad_q, "grad_k": grad_k, "grad_v": grad_v, "grad_initial": back})
  return res


def exact(case, seed):
  if case["op"] == "scan" and case["steps"] > 4096 and case["train"]:
    return None
  s = _inputs(case, seed)
  s["case"] = case
  return {"choose": _exact_choose, "evaluate": _exact_evaluate, "step": _exact_step, "scan": _exact_scan}[case["op"]](s)
