"""Attention of trees whose largest scores come late: what a row has summed up so far is then scaled by powers of two and more, tile after
tile.  Against the definition in 64 bits, within the bound of ``tree_cases.close_enough``."""
import pytest
import torch

import torch_ops
from gpu_helpers import DEV
from miniinfer_b200.kernels.ops import AttentionBatch
from tree_cases import close_enough, tree_case

pytestmark = pytest.mark.gpu

PAGE = 64


def places_of(table, batch, b, first, n, device):
  """Pages and offsets of n keys of item b from `first` on."""
  key = torch.arange(first, first + n)
  pages = table[int(batch.seq_slot[b])].cpu().long()[key // PAGE]
  return pages.to(device), (key % PAGE).to(device)


def make(shape, heads, hd, n, kind, dtype):
  """Requests of ``shape`` - context lengths - with trees of n tokens, four query heads a key/value head.

  ``planted``: in one tile of each request, another one from request to request, a key of each head that lies along the query of one of the tree's
  rows; it scores about 20 in base 2 above the mean of the others, whose largest is about 9.  ``rising``: keys grow with their place, so the largest score of a tile beats
  that of the tile before by more the further it goes."""
  nkv, G = heads
  qkv, kv, table, batch = tree_case([(c, n) for c in shape], nkv * G, nkv, hd, PAGE, torch.float32, seed=len(shape) + hd + n, scale_q=2.0)
  q = qkv[:, :nkv * G * hd].view(-1, nkv, G, hd)
  tile = 64 if hd > 128 else 128
  for b, c in enumerate(shape):
    if kind == "rising":
      pages, at = places_of(table, batch, b, 0, c + n, kv.device)
      grown = kv[pages, 0, :, at] * (0.2 + 4.0 * torch.arange(c + n, device=kv.device) / (c + n))[:, None, None]
      kv[pages, 0, :, at] = grown
    else:
      tiles = -(-c // tile)
      t = min((0, 1, 2, 3, tiles - 1)[b % 5], tiles - 1)
      key = min(t * tile + (37 * b) % tile, c - 1)
      row = int(batch.q_start[b]) + (5 * b + 1) % n
      pages, at = places_of(table, batch, b, key, 1, kv.device)
      along = q[row, :, b % G]
      kv[pages[0], 0, :, at[0]] = along * (14 * hd ** 0.5 / along.pow(2).sum(-1, keepdim=True))      # scores of 14, 20 in base 2
  return qkv.to(dtype), kv.to(dtype), table, batch


def some(batch, items):
  """The batch with a few of its items, for the definition's sake."""
  at = torch.tensor(items, device=batch.q_start.device)
  return AttentionBatch(q_start=batch.q_start[at], q_len=batch.q_len[at], ctx_len=batch.ctx_len[at], seq_slot=batch.seq_slot[at], positions=batch.positions,
                        num_items=len(items), max_ctx_len=batch.max_ctx_len, max_q_len=batch.max_q_len, tree_mask=batch.tree_mask)


def check(shape, heads, hd, n, kind, dtype, window=None, sink=None, cap=0.0, items=None):
  from miniinfer_b200.kernels import ops
  qkv, kv, table, batch = make(shape, heads, hd, n, kind, dtype)
  nh, nkv = heads[0] * heads[1], heads[0]
  out, again = (torch.full((qkv.shape[0], nh * hd), 777.0, dtype=dtype, device=DEV) for _ in range(2))
  for o in (out, again):
    ops.tree_attention(o, qkv, kv, table, batch, nh, nkv, hd, hd ** -0.5, window, sink, cap)
  assert torch.equal(out, again)
  terms = torch_ops.tree_terms(qkv, kv, table, some(batch, items or list(range(len(shape)))), nh, nkv, hd, hd ** -0.5, window, sink, cap)
  assert close_enough(out, terms, dtype, hd, max(shape) + n, cap) <= 1.0


# many requests, whose heads lie in one block each; a few long ones, whose heads are shared by blocks
WHOLE = [600 + 13 * (b % 7) for b in range(74)]
SPLIT = [1300, 2500, 900, 1700, 1100]


@pytest.mark.parametrize("kind", ["planted", "rising"])
@pytest.mark.parametrize("n", [24, 64])
@pytest.mark.parametrize("hd", [64, 80, 128, 192, 256])
def test_requests_that_lie_in_one_block(hd, n, kind):
  check(WHOLE, (2, 4), hd, n, kind, torch.bfloat16, items=[0, 1, 2, 3, 4, 73])


@pytest.mark.parametrize("kind", ["planted", "rising"])
@pytest.mark.parametrize("n", [24, 64])
@pytest.mark.parametrize("hd", [64, 80, 128, 192, 256])
def test_requests_that_blocks_share(hd, n, kind):
  check(SPLIT, (8, 4), hd, n, kind, torch.bfloat16)


@pytest.mark.parametrize("kind", ["planted", "rising"])
@pytest.mark.parametrize("n,hd", [(24, 128), (64, 128), (64, 64), (24, 256)])
@pytest.mark.parametrize("with_sink,cap", [(True, 0.0), (False, 30.0), (True, 50.0)])
def test_with_sinks_and_caps(with_sink, cap, n, hd, kind):
  sink = torch.linspace(-4, 12, 8).to(DEV) if with_sink else None
  check(WHOLE, (2, 4), hd, n, kind, torch.bfloat16, sink=sink, cap=cap, items=[0, 1, 4])


@pytest.mark.parametrize("kind", ["planted", "rising"])
@pytest.mark.parametrize("n", [24, 64, 100])
@pytest.mark.parametrize("past", [125, 126, 127])
def test_a_window_that_leaves_some_rows_a_key_or_two_of_the_first_tile(past, n, kind):
  """The window of the tree's root begins `past` keys into a tile: its children see a key less, deeper rows none of the tile's."""
  window = 300
  check([128 * k + past + window - 1 for k in (1, 3, 2, 9)] * 19, (2, 4), 128, n, kind, torch.bfloat16, window=window, items=[0, 1, 2, 3])


@pytest.mark.parametrize("kind", ["planted", "rising"])
@pytest.mark.parametrize("n", [1, 3, 13])
@pytest.mark.parametrize("hd", [64, 256])
def test_in_32_bits(hd, n, kind):
  check([700, 1300], (2, 4), hd, n, kind, torch.float32)


@pytest.mark.parametrize("kind", ["planted", "rising"])
@pytest.mark.parametrize("n", [1, 3, 8])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
def test_few_rows_whose_pieces_the_last_block_joins(hd, n, kind):
  """Up to 32 rows of heads up to 128, beside heads of 256, whose pieces another kernel joins."""
  check(SPLIT[:2], (8, 4), hd, n, kind, torch.bfloat16)
