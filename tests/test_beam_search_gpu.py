"""Beam search with whole models of the framework: steps of the runner, ``ops.beam_select`` and ``KVCacheManager.fork`` and ``reorder``, against the plain
implementations, which know only the tokens.  Windows whose pages go back, latents, recurrent states and convolutions among the layers."""
import pytest
import torch

import plain_besolix
import plain_qwen3
from gpu_helpers import DEV

pytestmark = pytest.mark.gpu


def ints(x):
  return torch.tensor(x, dtype=torch.int32, device=DEV)


def search(trace_runner, log_probs, prompts, beams, steps, tol):
  """Every selection has to be one that the plain implementation's scores of the same beams allow, within what the float32 path may err; the scores that
  are handed on have to be the plain ones of the whole sequence."""
  from miniinfer_b200.engine.runner import StepItem
  from miniinfer_b200.kernels import ops
  cache, runner = trace_runner.cache, trace_runner.runner
  order, history = [], {}
  for r, prompt in enumerate(prompts):      # the prompt but for its last token, then the beams
    group = [(r, b) for b in range(beams)]
    cache.admit(group[0])
    runner.step([StepItem(group[0], prompt[:-1])])
    cache.fork(group[0], group[1:])
    order += group
    history.update({q: list(prompt) for q in group})
  R = len(prompts)
  cum = torch.tensor([0.0] + [float("-inf")] * (beams - 1), device=DEV).repeat(R)      # at first a request's beams are alike: one counts
  starts = ints([beams * r for r in range(R + 1)])
  out = [torch.empty((R, beams), dtype=t, device=DEV) for t in (torch.int32, torch.int32, torch.float32)]
  for step in range(steps):
    logits = runner.step([StepItem(q, [history[q][-1]], [0]) for q in order])
    ops.beam_select(*out, logits, cum, starts, runner.ws)
    live = [q for q, c in zip(order, cum.tolist()) if c > float("-inf")]
    plain = {q: log_probs(history[q]) for q in live}
    tokens, parents = out[0].flatten().tolist(), [order[p] for p in out[1].flatten().tolist()]
    near = (step + 1) * 2 * tol
    before = dict(zip(order, cum.double().tolist()))
    for r in range(R):
      mine = [(parents[i], tokens[i]) for i in range(beams * r, beams * r + beams)]
      assert len(set(mine)) == beams
      every = torch.cat([before[q] + plain[q] for q in live if q[0] == r])
      least = float(every.topk(beams).values[-1])
      for (q, t), score in zip(mine, out[2][r].tolist()):
        want = before[q] + float(plain[q][t])
        assert abs(score - want) < 2 * tol + 1e-5 and want > least - 4 * tol
    cum = out[2].flatten().clone()
    cache.reorder(dict(zip(order, parents)))
    cache.check_invariants()
    history = {q: history[p] + [t] for q, p, t in zip(order, parents, tokens)}
  for q, c in zip(order, cum.tolist()):      # what was handed on from step to step is the plain score of the whole continuation
    prompt = prompts[q[0]]
    want = sum(float(log_probs(history[q][:n])[history[q][n]]) for n in range(len(prompt), len(prompt) + steps))
    assert abs(c - want) < near + steps * 1e-5
  runner.check_status()
  for q in order:
    cache.release_request(q)
  assert cache.free_pages() == [g.num_pages for g in cache.paged_groups]
  return history


@pytest.mark.parametrize("tag,page", [("A", 16), ("C", 8)])
def test_beams_of_layers_with_and_without_a_window(model_dirs, tag, page):
  from miniinfer_b200.engine.replay import TraceRunner
  d = model_dirs(tag)
  w, cfg = plain_qwen3.read_weights(d), plain_qwen3.read_config(d)
  log_probs = lambda ids: torch.log_softmax(plain_qwen3.forward(w, cfg, ids, rows=[len(ids) - 1]).double(), dim=1)[0]      # noqa: E731
  runner = TraceRunner(d, "float32", 0, device=DEV, page_size=page, num_pages=48, max_requests=8)
  history = search(runner, log_probs, [[5, 17, 3, 200, 9], list(range(40, 75))], 4, 24, 1e-4)
  assert len({tuple(h) for h in history.values()}) == 8


@pytest.mark.parametrize("tag", ["A", "B"])
def test_beams_of_layers_with_states_and_latents(tag, tmp_path):
  from miniinfer_b200.engine.replay import TraceRunner
  d = plain_besolix.make_model_dir(plain_besolix.CONFIGS[tag], str(tmp_path), seed=71)
  w, cfg = plain_besolix.read_weights(d), plain_besolix.read_config(d)
  size = []

  def log_probs(ids):
    with torch.no_grad():
      z = plain_besolix.forward(cfg, w, list(ids))[-1].double()
    size.append(float(z.pow(2).mean().sqrt()))
    return torch.log_softmax(z, dim=0)

  log_probs([5, 6, 7])
  runner = TraceRunner(d, "float32", 0, device=DEV, page_size=8, num_pages=80, max_requests=6)
  assert runner.cache.state_groups
  search(runner, log_probs, [[5, 17, 3, 20, 9], list(range(40, 61))], 3, 16, 3e-4 * max(1.0, 2 * size[0]))
