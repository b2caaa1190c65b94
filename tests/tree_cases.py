"""Random trees of drafted tokens over a paged cache, for the tests of ``tree_attention``."""
import random

import torch

from gpu_helpers import DEV
from miniinfer_b200.kernels.ops import AttentionBatch


def make_tree(rng: random.Random, nodes: int, reach: int = 5, empty: float = 0.0):
  """For each node the bits of what it sees (its ancestors and itself; nothing for the share ``empty`` of padded places) and its depth."""
  sees, depth = [], []
  for j in range(nodes):
    parent = rng.randint(max(0, j - reach), j - 1) if j else -1
    sees.append((sees[parent] if j else 0) | 1 << j)
    depth.append(depth[parent] + 1 if j else 0)
  return [0 if rng.random() < empty else m for m in sees], depth


def words_of(mask: int, words: int):
  """A bit mask as ``words`` int32 words, the lowest bits first."""
  got = []
  for w in range(words):
    x = mask >> 32 * w & 0xffffffff
    got.append(x - (1 << 32) if x >> 31 else x)
  return got


def tree_case(items, nh, nkv, hd, page_size, dtype, seed=0, empty=0.0, scale_q=1.0, gap=0, extra_words=0, scratch=None, most=None, longest=None):
  """``items``: (context keys, new tokens) of each request.  Returns (qkv, cache layer, block table, batch).  ``gap``: rows of no item between
  the requests' rows.  The pages lie in any order; what no request has written holds NaN."""
  rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
  lengths = [c + n for c, n in items]
  span = max(-(-c // page_size) for c in lengths) + 1
  pages = sum(-(-c // page_size) for c in lengths)
  ids = list(range(1, pages + 3))
  rng.shuffle(ids)
  table = torch.zeros((len(items) + 3, span), dtype=torch.int32)
  slots = rng.sample(range(len(items) + 3), len(items))
  kv = torch.full((pages + 3, 2, nkv, page_size, hd), float("nan"))
  words = -(-max(n for _, n in items) // 32) + extra_words
  mask, positions, q_start, row = [], [], [], 0
  for b, (context, n) in enumerate(items):
    for i in range(-(-lengths[b] // page_size)):
      p = table[slots[b], i] = ids.pop()
      rows = min(page_size, lengths[b] - i * page_size)
      kv[p, :, :, :rows] = torch.randn((2, nkv, rows, hd), generator=g)
    sees, depth = make_tree(rng, n, empty=empty)
    q_start.append(row)
    for m, d in zip(sees, depth):
      mask.append(words_of(m, words))
      positions.append(context + d)
    mask += [[-1] * words] * gap
    positions += [0] * gap
    row += n + gap
  qkv = torch.randn((row, (nh + 2 * nkv) * hd), generator=g) * scale_q
  dev = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)      # noqa: E731
  batch = AttentionBatch(q_start=dev(q_start), q_len=dev([n for _, n in items]), ctx_len=dev(lengths), seq_slot=dev(slots), positions=dev(positions),
                         num_tokens=row, num_items=len(items), max_ctx_len=longest or max(lengths), max_q_len=most or max(n for _, n in items),
                         tree_mask=dev(mask), scratch=scratch)
  return qkv.to(dtype).to(DEV), kv.to(dtype).to(DEV), table.to(DEV), batch


def close_enough(got, terms, dtype, hd, keys, softcap=0.0):
  """Whether rows of ``got`` [T, nh * hd] lie where rounding may put them, given ``torch_ops.tree_terms``.

  A score is a sum of hd products in float32 and errs by at most (hd + 3) 2^-24 B, B being its largest sum of |q| |k| (a cap's tanh by 2^-20 of
  the cap), a weight so by twice that, relative to itself, beside 2^-21 of the exponential; sums over the keys by 2^-24 of each addition.
  bfloat16: a weight is rounded before it multiplies a value and once more in the sum that divides, 2^-8 each, and the result, 2^-8."""
  worst = 0.0
  for t, (want, size, score) in terms.items():
    nh = want.shape[0]
    d = (got[t].double().view(nh, hd) - want).abs()
    delta = 2 * ((hd + 3) * 2.0 ** -24 * score + 2.0 ** -20 * softcap)[:, None] + 2.0 ** -21 + (keys + 8) * 2.0 ** -23
    bound = size * delta + 2.0 ** -24 * want.abs() + 1e-9
    if dtype == torch.bfloat16:
      bound = bound + 2.0 ** -7 * size + 2.0 ** -8 * want.abs()
    if not torch.isfinite(d).all():
      return float("inf")
    worst = max(worst, float((d / bound).max()))
  return worst
