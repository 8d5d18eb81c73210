"""envpool_amd.policy together with the pools, as they are used: memory moved by a pool's own batches, actions
chosen under its mask and sent back; streams, captured graphs, two calls at once."""
import numpy as np
import pytest
import torch

from tests import policy_ref as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def test_a_rollout_with_a_memory_and_its_training_pass():
  """A Dummy pool stepped on the GPU with a memory beside it, then the stored segment read back at once: the same
  outputs, episode starts included, and gradients against the formula's."""
  import envpool_amd
  from envpool_amd import policy
  n, t, h, dk, dv = 6, 40, 2, 16, 24
  env = envpool_amd.make("Dummy-v0", "gymnasium", num_envs=n, seed=3)
  g = _gen(1)
  decay = torch.tensor([-0.05, -0.3])
  mem = env.memory_torch(h, dk, dv, decay.to(DEV))
  obs, info = env.reset_torch()
  act = {"list_action": torch.full((n, 6), 1.5, dtype=torch.float64, device=DEV)}
  q, k, v = (torch.randn(t, n, h, d, generator=g).to(DEV) for d in (dk, dk, dv))
  outs, fresh = [], []
  for i in range(t):
    fresh.append(info["elapsed_step"] == 0)
    outs.append(mem.step(q[i], k[i], v[i], env_id=info["env_id"], elapsed_step=info["elapsed_step"]))
    obs, rew, term, trunc, info = env.step_torch(act)
  outs, fresh = torch.stack(outs), torch.stack(fresh)
  assert fresh[1:].any() and fresh[0].all()  # episodes end inside
  leaves = [x.detach().requires_grad_() for x in (q, k, v)]
  out, final = policy.memory_scan(*leaves, decay.to(DEV), fresh=fresh)
  size = float(out.abs().max())
  assert (out - outs).abs().max() <= 1e-5 * size and (final - mem.state).abs().max() <= 1e-5 * float(final.abs().max())
  logits = out.flatten(2)[..., :16]
  stored = policy.choose(logits.detach().reshape(t * n, 16), torch.rand(t * n, generator=g).to(DEV))
  lp, ent = policy.evaluate(logits.reshape(t * n, 16), stored.action)
  assert (lp - stored.log_prob).abs().max() < 1e-5 and (ent - stored.entropy).abs().max() < 1e-5
  gain = torch.randn(t * n, generator=g)
  ((lp * gain.to(DEV)).sum() + 0.01 * ent.sum()).backward()
  # the same from the definitions
  r = ref.evaluate(logits.detach().reshape(t * n, 16), stored.action, gain, torch.full((t * n,), 0.01))
  do = torch.zeros(t, n, h * dv, dtype=torch.float64)
  do[..., :16] = r["grad_logits"].view(t, n, 16)
  want = ref.scan(q, k, v, decay, fresh=fresh, scale=dk**-0.5, grad_out=do.view(t, n, h, dv))
  for name, leaf in zip("qkv", leaves):
    w = want["grad_" + name]
    assert (leaf.grad.cpu().double() - w).abs().max() <= 2e-5 * float(w.abs().max()), name
  env.close()


def test_choices_under_the_pools_mask():
  """YGOPro: logits -> choose_torch -> send_choice -> the envs got what was chosen, sync and async."""
  import envpool_amd
  from envpool_amd import capi_ygo, ygopro
  from tools import ygo_synth
  n = 48
  table = ygo_synth.make_table(1000, seed=0)
  for batch in (n, n // 2):
    cfg = capi_ygo.default_config(max_batch=batch, ring_depth=0)
    eng = ygo_synth.SynthEngine(cfg, table, n, seed=2)
    ygopro.init_module(eng.factory, table)
    try:
      env = envpool_amd.make("YGOPro-v0", "gymnasium", num_envs=n, batch_size=batch, num_threads=3)
      with pytest.raises(RuntimeError, match="choose_torch"):
        env.choose_torch(torch.zeros(batch, 16, device=DEV))
      env.async_reset()
      obs, rew, term, trunc, info = env.recv_torch()
      sent = {}
      g = _gen(5)
      for step in range(6):
        logits = torch.randn(batch, 16, generator=g)
        u = torch.rand(batch, generator=g)
        mask, count, ids = info["action_mask"].cpu(), info["num_options"].cpu(), env.last_env_ids.copy()
        c = env.choose_torch(logits.to(DEV), u.to(DEV))
        want = ref.choose(logits, u, mask=mask)
        assert torch.equal(c.action.cpu().long(), want[0])
        by_count = ref.choose(logits, u, num_options=count)
        assert torch.equal(by_count[0], want[0])  # the mask is arange(16) < num_options
        assert ((c.action.cpu() < count) | (count == 0)).all()
        with pytest.raises(ValueError, match="mask"):
          env.choose_torch(logits.to(DEV), mask=mask.to(DEV))
        env.send_choice(c)
        sent.update({int(e): max(0, int(a)) for e, a in zip(ids, c.action.cpu())})
        obs, rew, term, trunc, info = env.recv_torch()
        won, start = info["win_reason"].cpu(), info["elapsed_step"].cpu()
        for i, e in enumerate(env.last_env_ids):  # (the stand-in engine echoes the action in win_reason)
          if int(e) in sent and int(start[i]) > 0:
            assert int(won[i]) == sent[int(e)]
      env.close()
    finally:
      ygopro.init_module(None, None)
      eng.close()


def test_other_streams_and_two_calls_at_once():
  """Calls follow torch's current stream, and two that run side by side do not share scratch memory."""
  from envpool_amd import policy
  g = _gen(2)
  s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
  a = 60000  # long rows: these calls have scratch memory
  x = [torch.randn(6, a, generator=g).to(DEV) for _ in range(2)]
  u = [torch.rand(6, generator=g).to(DEV) for _ in range(2)]
  want = [policy.choose(x[i], u[i]) for i in range(2)]
  q, k, v = (torch.randn(700, 2, 2, 64, generator=g).to(DEV) for _ in range(3))
  decay = torch.tensor([-0.01, -0.1], device=DEV)
  want_scan = policy.memory_scan(q, k, v, decay)
  torch.cuda.synchronize()
  got, scans = [], []
  for _ in range(10):
    for i, s in enumerate((s1, s2)):
      with torch.cuda.stream(s):
        got.append((i, policy.choose(x[i], u[i])))
        scans.append(policy.memory_scan(q, k, v, decay))
  torch.cuda.synchronize()
  for i, c in got:
    assert all(torch.equal(p, w) for p, w in zip(c, want[i]))
  for o in scans:
    assert all(torch.equal(p, w) for p, w in zip(o, want_scan))


def test_captured_and_replayed():
  """choose, a memory step and a scan with its backward pass, captured; every replay against the eager result, with
  eager work and synchronisation between the replays. While an eager graph over the same leaves lives, the capture
  is refused: torch would end the process."""
  from envpool_amd import policy
  g = _gen(9)
  n, h, dk, dv, t, a = 1500, 2, 16, 16, 130, 40
  q, k, v = (torch.randn(t, 3, h, d, generator=g).to(DEV).requires_grad_() for d in (dk, dk, dv))
  decay = torch.tensor([-0.02, -0.2], device=DEV)
  logits = torch.randn(n, a, generator=g).to(DEV).requires_grad_()
  bias = torch.zeros(a, device=DEV).requires_grad_()
  u = torch.rand(n, generator=g).to(DEV)
  ids = torch.randperm(n, generator=g).int().to(DEV)
  ids[7] = ids[5]
  rows = [torch.randn(n, h, d, generator=g).to(DEV) for d in (dk, dk, dv)]
  state = torch.randn(n, h, dk, dv, generator=g).to(DEV)
  def work(memory):
    c = policy.choose(logits.detach(), u, bias=bias.detach())
    lp, ent = policy.evaluate(logits, c.action, bias=bias)
    out, final = policy.memory_scan(q, k, v, decay)
    grads = torch.autograd.grad([lp, ent, out, final], [logits, bias, q, k, v],
                                [torch.ones_like(lp), torch.ones_like(ent), torch.ones_like(out), torch.ones_like(final)])
    o = memory.step(*rows, env_id=ids)
    return [*c, lp.detach(), ent.detach(), out.detach(), *grads, o, memory.state]

  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    work(policy.EnvMemory(n, h, dk, dv, decay, state=state.clone()))
  torch.cuda.current_stream().wait_stream(side)
  memory = policy.EnvMemory(n, h, dk, dv, decay, state=state.clone())
  reference = policy.EnvMemory(n, h, dk, dv, decay, state=state.clone())
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = work(memory)
  memory.state.copy_(state)
  del side
  for i in range(4):
    with torch.no_grad():
      logits.copy_(torch.randn(n, a, generator=g).to(DEV))
      u.copy_(torch.rand(n, generator=g).to(DEV))
    graph.replay()
    got = [x.clone() for x in captured]
    torch.cuda.synchronize()
    want = work(reference)
    torch.cuda.synchronize()
    for j, (x, w) in enumerate(zip(got, want)):
      assert torch.equal(x, w), (i, j)


@pytest.mark.parametrize("which", ["scan", "evaluate"])
def test_a_capture_over_leaves_of_a_living_eager_graph_is_refused(which):
  from envpool_amd import policy
  decay = torch.zeros(1, device=DEV)
  act = torch.zeros(3, dtype=torch.int32, device=DEV)
  leaf = torch.randn(3, 2, 1, 8, device=DEV).requires_grad_() if which == "scan" else torch.randn(3, 8, device=DEV).requires_grad_()
  call = (lambda: policy.memory_scan(leaf, leaf, leaf, decay)[0]) if which == "scan" else (lambda: policy.evaluate(leaf, act)[0])
  living = call()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with pytest.raises(RuntimeError, match="recorded outside this capture"):
    with torch.cuda.graph(graph):
      call()
  torch.cuda.synchronize()
  want, = torch.autograd.grad(living.sum(), leaf)  # (the eager graph is as it was)
  del living
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    first, second = call(), call()  # two calls over one leaf
    got, = torch.autograd.grad(first, leaf, torch.ones_like(first))
    again, = torch.autograd.grad(second, leaf, torch.ones_like(second))
  del first, second
  graph.replay()
  torch.cuda.synchronize()
  assert torch.equal(got, want) and torch.equal(again, want)


def test_a_tensor_changed_before_the_backward_pass_is_noticed():
  from envpool_amd import policy
  x = torch.randn(4, 10, device=DEV)
  mask = torch.ones(4, 10, dtype=torch.bool, device=DEV)
  leaf = x.clone().requires_grad_()
  lp, _ = policy.evaluate(leaf, torch.zeros(4, dtype=torch.int32, device=DEV), mask=mask)
  mask[0, 3] = False
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    lp.sum().backward()
  q = torch.randn(5, 2, 1, 8, device=DEV).requires_grad_()
  fresh = torch.zeros(5, 2, dtype=torch.bool, device=DEV)
  out, _ = policy.memory_scan(q, q, q, torch.zeros(1, device=DEV), fresh=fresh)
  fresh[1, 0] = True
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    out.sum().backward()
  # differentiable once
  lp, _ = policy.evaluate(leaf, torch.zeros(4, dtype=torch.int32, device=DEV))
  g1, = torch.autograd.grad(lp.sum(), leaf, create_graph=True)
  with pytest.raises(RuntimeError):
    g1.sum().backward()


def test_gradients_reach_shared_and_expanded_inputs():
  """A bias expanded over the rows by the caller, keys expanded over heads by the caller: autograd sums."""
  from envpool_amd import policy
  g = _gen(4)
  x = torch.randn(33, 12, generator=g).to(DEV)
  act = torch.randint(0, 12, (33,), generator=g, dtype=torch.int32).to(DEV)
  b = torch.randn(12, generator=g).to(DEV).requires_grad_()
  lp1, _ = policy.evaluate(x, act, bias=b)
  lp2, _ = policy.evaluate(x, act, bias=b.expand(33, 12))
  assert torch.allclose(lp1, lp2, atol=1e-6)
  g1, = torch.autograd.grad(lp1.sum(), b)
  g2, = torch.autograd.grad(lp2.sum(), b)
  assert torch.allclose(g1, g2, atol=1e-5)
  q = torch.randn(70, 2, 6, 32, generator=g).to(DEV)
  k = torch.randn(70, 2, 2, 32, generator=g).to(DEV).requires_grad_()
  v = torch.randn(70, 2, 2, 16, generator=g).to(DEV).requires_grad_()
  decay = -torch.rand(6, generator=g).to(DEV)
  w = torch.randn(70, 2, 6, 16, generator=g).to(DEV)
  o1, _ = policy.memory_scan(q, k, v, decay)
  o2, _ = policy.memory_scan(q, k.repeat_interleave(3, 2), v.repeat_interleave(3, 2), decay)
  assert torch.equal(o1, o2)
  for p, r in zip(torch.autograd.grad((o1 * w).sum(), [k, v]), torch.autograd.grad((o2 * w).sum(), [k, v])):
    assert torch.allclose(p, r, atol=2e-5 * float(r.abs().max()))


def test_a_batch_of_ring_views_feeds_the_calls():
  """Views of the pool's device memory (not torch's) are operands like any other."""
  import envpool_amd
  env = envpool_amd.make("Dummy-v0", "gymnasium", num_envs=300, seed=1)
  obs, info = env.reset_torch()
  assert info["elapsed_step"].dtype == torch.int32 and info["env_id"].dtype == torch.int32
  mem = env.memory_torch(1, 4, 4, torch.zeros(1, device=DEV))
  ones = torch.ones(300, 1, 4, device=DEV)
  for i in range(3):
    out = mem.step(ones, ones, ones, env_id=info["env_id"], elapsed_step=info["elapsed_step"], scale=1.0)
    act = {"list_action": torch.full((300, 6), 1.5, dtype=torch.float64, device=DEV)}
    obs, rew, term, trunc, info = env.step_torch(act)
  assert np.all(out.cpu().numpy() >= 4.0)
  env.close()
