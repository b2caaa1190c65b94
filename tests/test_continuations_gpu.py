"""The operators for several continuations of a request as they are used together: a beam search whose beams share pages, and trees of drafted tokens of which an
accepted path stays.  The model is one layer of attention over tied projections, small enough to be worked out in 64 bits from the tokens alone."""
import random

import pytest
import torch

from gpu_helpers import DEV
from miniinfer_b200.cache import FixedStateSpec, KVCacheManager, PagedKVSpec
from tree_cases import words_of

pytestmark = pytest.mark.gpu

NH, NKV, HD, P, VOCAB = 4, 2, 64, 16, 600


class Model:
  """Rows of a fused projection and a head that are tables, and what a position adds to queries and keys."""

  def __init__(self, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    self.dtype = dtype
    self.table = torch.randn((VOCAB, (NH + 2 * NKV) * HD), generator=g).to(dtype).to(DEV)
    self.head = (torch.randn((NH * HD, VOCAB), generator=g) * 0.3).to(dtype).to(DEV)
    self.shift = torch.randn((64, 1), generator=g).to(DEV)

  def rows(self, tokens, positions):
    """The fused rows of tokens at positions, as they go into the cache."""
    r = self.table[torch.as_tensor(tokens, device=DEV).long()].float()
    return (r * (1 + 0.1 * self.shift[torch.as_tensor(positions, device=DEV).long()])).to(self.dtype)

  def attention(self, tokens, positions=None):
    """In 64 bits: the last token's attention over all of them."""
    r = self.rows(tokens, positions if positions is not None else range(len(tokens))).double()
    q = r[-1, :NH * HD].view(NH, HD)
    k, v = (r[:, (NH + w * NKV) * HD:(NH + (w + 1) * NKV) * HD].view(-1, NKV, HD).repeat_interleave(NH // NKV, dim=1) for w in (0, 1))
    w = torch.softmax(torch.einsum("hd,nhd->hn", q, k) * HD ** -0.5, dim=1)
    return torch.einsum("hn,nhd->hd", w, v).reshape(-1)

  def log_probs(self, tokens):
    return torch.log_softmax(self.attention(tokens) @ self.head.double(), dim=0)


def ints(x):
  return torch.tensor(x, dtype=torch.int32, device=DEV)


def store(m, req, rows, first):
  """A step's keys and values into the request's pages, as the QKV preparation does."""
  places = torch.as_tensor(m.slot_mapping(req, 0, first, rows.shape[0]), device=DEV).long()
  kv = m.paged_groups[0].kv
  for w in (0, 1):
    kv[0, places // P, w, :, places % P] = rows[:, (NH + w * NKV) * HD:(NH + (w + 1) * NKV) * HD].view(-1, NKV, HD)


def attend(m, reqs, rows, masks, positions):
  """``tree_attention`` of the last appended tokens of each request: rows[i], with masks[i][t] the new tokens that t sees."""
  from miniinfer_b200.kernels import ops
  n = [r.shape[0] for r in rows]
  ctx = [m.length_of(q) + k for q, k in zip(reqs, n)]
  m.sync()
  words = -(-max(n) // 32)
  qkv = torch.cat(rows)
  batch = ops.AttentionBatch(q_start=ints([sum(n[:i]) for i in range(len(n))]), q_len=ints(n), ctx_len=ints(ctx), seq_slot=ints([m.slot_of(q) for q in reqs]),
                             positions=ints([p for ps in positions for p in ps]), num_tokens=sum(n), num_items=len(n), max_ctx_len=max(ctx), max_q_len=max(n),
                             tree_mask=ints([words_of(x, words) for ms in masks for x in ms]), scratch=None)
  out = torch.empty((sum(n), NH * HD), dtype=qkv.dtype, device=DEV)
  g = m.paged_groups[0]
  ops.tree_attention(out, qkv, g.kv[0], g.block_table, batch, NH, NKV, HD, HD ** -0.5)
  return out


def test_beam_search():
  """Two requests with prompts that end inside a page, three beams each, against a search in 64 bits that knows only the tokens."""
  from miniinfer_b200.kernels import ops
  model, beams, steps = Model(torch.float32, 1), 3, 20
  m = KVCacheManager([PagedKVSpec(NKV, HD), FixedStateSpec((5,))], P, 40, 2 * beams, 64, torch.float32, DEV)
  prompts = [[5, 17, 3, 200, 9], list(range(40, 72))]
  groups = [[(r, b) for b in range(beams)] for r in range(2)]
  tokens = {}
  for prompt, group in zip(prompts, groups):      # the prompt but for its last token, then the beams
    q = group[0]
    m.admit(q)
    m.append(q, len(prompt) - 1)
    store(m, q, model.rows(prompt[:-1], range(len(prompt) - 1)), 0)
    m.commit(q, len(prompt) - 1)
    m.state_groups[0].state[:, m.slot_of(q)] = float(len(prompt))
    m.fork(q, group[1:])
    tokens.update({b: prompt[-1] for b in group})
  cum = torch.tensor([0.0] + [float("-inf")] * (beams - 1), device=DEV).repeat(2)      # at first a request's beams are alike: one counts
  want = [[(0.0, list(p))] for p in prompts]
  history = {b: list(p) for p, group in zip(prompts, groups) for b in group}
  order = [b for group in groups for b in group]
  for step in range(steps):
    rows = [model.rows([tokens[b]], [m.length_of(b)]) for b in order]
    positions = [[m.length_of(b)] for b in order]
    for b, r in zip(order, rows):
      m.append(b, 1)
      store(m, b, r, m.length_of(b))
      m.state_groups[0].state[:, m.slot_of(b)] += tokens[b] / 1000
    out = attend(m, order, rows, [[1]] * len(order), positions)
    for b in order:
      m.commit(b, 1)
    logits = out.float() @ model.head.float()
    got = [torch.empty((2, beams), dtype=t, device=DEV) for t in (torch.int32, torch.int32, torch.float32)]
    ops.beam_select(*got, logits.contiguous(), cum, ints([0, beams, 2 * beams]))
    new_tokens, parents = got[0].flatten().tolist(), [order[p] for p in got[1].flatten().tolist()]
    cum = got[2].flatten()
    m.reorder(dict(zip(order, parents)))
    m.check_invariants()
    history = {b: history[p] + [t] for b, p, t in zip(order, parents, new_tokens)}
    tokens = dict(zip(order, new_tokens))
    for i, known in enumerate(want):      # the search in 64 bits
      scored = [(s + float(lp), seq + [v]) for s, seq in known for v, lp in enumerate(model.log_probs(seq).tolist())]
      want[i] = sorted(scored, key=lambda x: -x[0])[:beams]
  for i, group in enumerate(groups):
    for (score, seq), b in zip(want[i], group):
      assert history[b] == seq
      # 20 normalisers of 3.5e-6 each, and scores whose logits err by float32 sums of 256 products of size one
      assert abs(float(cum[order.index(b)]) - score) < 20 * (3.5e-6 + 2 * 256 * 2.0 ** -24) + 2.0 ** -24 * abs(score) * 20
      state = float(len(prompts[i])) + sum(seq[len(prompts[i]) - 1:-1]) / 1000
      assert torch.allclose(m.state_groups[0].state[:, m.slot_of(b)].cpu(), torch.tensor(state), rtol=1e-5)
  shared = sum(m.paged_groups[0].allocator.holders(p) > 1 for p in m.paged_groups[0].allocator.held())
  assert shared >= 3      # the full pages of the second prompt, at least


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_tree_of_which_a_path_is_accepted(dtype):
  """Trees over two requests; a path of each stays, and what comes next sees the context, the path and nothing else."""
  model, rng = Model(dtype, 2), random.Random(4)
  m = KVCacheManager([PagedKVSpec(NKV, HD)], P, 40, 4, 64, dtype, DEV)
  seqs = {"a": [5, 17, 3, 200, 9, 11, 12], "b": list(range(40, 71))}
  for q, seq in seqs.items():
    m.admit(q)
    m.append(q, len(seq))
    store(m, q, model.rows(seq, range(len(seq))), 0)
    m.commit(q, len(seq))
  tol = 2e-5 if dtype == torch.float32 else 3e-2      # values of unit size; bfloat16: weights and results rounded, 2^-7 and 2^-8
  for turn in range(3):
    rows, masks, positions, nodes, paths = [], [], [], {}, {}
    for q, seq in seqs.items():
      n = rng.randint(2, 8)
      tokens, parent = [rng.randrange(VOCAB) for _ in range(n)], [-1] + [rng.randrange(-1, j) for j in range(1, n)]
      path = [[] for _ in range(n)]
      for j in range(n):
        path[j] = (path[parent[j]] if parent[j] >= 0 else []) + [j]
      nodes[q], paths[q] = tokens, path
      positions.append([len(seq) + len(p) - 1 for p in path])
      masks.append([sum(1 << j for j in p) for p in path])
      rows.append(model.rows(tokens, positions[-1]))
      m.append(q, n)
      store(m, q, rows[-1], len(seq))
    out = attend(m, list(seqs), rows, masks, positions)
    at = 0
    kept = {}
    for q, seq in seqs.items():
      for p in paths[q]:
        want = model.attention(seq + [nodes[q][j] for j in p])
        assert (out[at].double() - want).abs().max() < tol
        at += 1
      kept[q] = paths[q][-1] if turn < 2 else []      # at last nothing is accepted
    m.keep(kept)
    m.check_invariants()
    seqs = {q: seq + [nodes[q][j] for j in kept[q]] for q, seq in seqs.items()}
    assert all(m.length_of(q) == len(seq) for q, seq in seqs.items())
  # one more token behind what stayed
  rows = [model.rows([7], [len(seq)]) for seq in seqs.values()]
  for (q, seq), r in zip(seqs.items(), rows):
    m.append(q, 1)
    store(m, q, r, len(seq))
  out = attend(m, list(seqs), rows, [[1], [1]], [[len(seq)] for seq in seqs.values()])
  for o, seq in zip(out, seqs.values()):
    assert (o.double() - model.attention(seq + [7])).abs().max() < tol


def test_more_tokens_are_kept_than_go_through_shared_memory_at_a_time():
  m = KVCacheManager([PagedKVSpec(1, 16)], 64, 420, 2, 26000, torch.float32, DEV)
  m.admit("a")
  m.append("a", 26000)
  places = torch.tensor(m.slot_mapping("a", 0, 0, 26000), device=DEV).long()
  kv = m.paged_groups[0].kv
  kv[0, places // 64, :, :, places % 64] = torch.arange(26000.0, device=DEV)[:, None, None, None]
  m.keep({"a": list(range(1, 26000, 2))})
  places = places[:13000]
  assert m.length_of("a") == 13000
  assert (kv[0, places // 64, :, :, places % 64] == torch.arange(1.0, 26000, 2, device=DEV)[:, None, None, None]).all()
  m.check_invariants()
