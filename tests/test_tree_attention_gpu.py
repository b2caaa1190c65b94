"""Attention of trees of new tokens over a paged cache, against its definition in 64 bits."""
import random

import pytest
import torch

import torch_ops
from gpu_helpers import DEV
from tree_cases import close_enough, tree_case, words_of

pytestmark = pytest.mark.gpu

# (items (context keys, new tokens), heads, kv heads, head size, page size, window, sink, softcap, share of empty rows)
CASES = [
  ([(0, 1)], 4, 2, 128, 64, None, False, 0.0, 0.0),                                 # nothing before a single token
  ([(1, 1), (63, 1), (64, 1), (65, 2)], 4, 4, 64, 64, None, False, 0.0, 0.0),       # a page just full, and one key over
  ([(127, 1), (128, 1), (129, 3), (0, 7)], 16, 8, 128, 64, None, False, 0.0, 0.0),
  ([(1000, 8)], 16, 8, 128, 64, None, False, 0.0, 0.0),
  ([(700, 32), (513, 17), (2100, 31)], 32, 8, 128, 64, None, False, 0.0, 0.0),      # 128 rows a key/value head
  ([(300, 64), (90, 33)], 32, 8, 128, 64, None, True, 0.0, 0.1),                    # 256 rows, rows that see nothing beside a sink
  ([(250, 100), (5, 65)], 12, 2, 64, 128, None, False, 30.0, 0.0),                  # masks of several words, six heads a group
  ([(333, 21)], 20, 4, 80, 16, None, False, 0.0, 0.2),                              # five heads a group, small pages
  ([(500, 40), (31, 9)], 8, 8, 96, 32, 100, False, 0.0, 0.0),                       # a window that begins inside the context
  ([(40, 60), (3, 50)], 8, 2, 128, 64, 4, True, 0.0, 0.0),                          # a window shorter than the tree is deep
  ([(400, 30), (129, 12)], 8, 2, 256, 64, None, False, 50.0, 0.0),
  ([(200, 9)], 6, 1, 192, 64, 64, False, 0.0, 0.3),
  ([(60, 5), (200, 11)], 2, 2, 16, 16, None, False, 0.0, 0.0),
  ([(60, 5), (77, 3)], 4, 2, 20, 7, None, True, 0.0, 0.0),                          # sizes that no tile likes
  ([(90, 6)], 3, 1, 33, 5, 30, False, 10.0, 0.2),
  ([(50, 9)], 2, 1, 640, 16, None, False, 0.0, 0.0),
  ([(5, 3)] * 70, 4, 2, 64, 64, None, False, 0.0, 0.0),                             # more requests than a warp has lanes, twice
  ([(0, 40), (0, 3)], 64, 8, 128, 64, None, False, 0.0, 0.4),                       # trees without a context
]


def run(case, dtype, scratch=None, **more):
  from miniinfer_b200.kernels import ops
  items, nh, nkv, hd, P, window, with_sink, cap, empty = CASES[case] if isinstance(case, int) else case
  qkv, kv, table, batch = tree_case(items, nh, nkv, hd, P, dtype, seed=len(items) + nh + hd, empty=empty, scale_q=2.0, scratch=scratch, **more)
  sink = torch.randn(nh, generator=torch.Generator().manual_seed(nh)).to(DEV) if with_sink else None
  out = torch.full((qkv.shape[0], nh * hd), 777.0, dtype=dtype, device=DEV)
  args = (qkv, kv, table, batch, nh, nkv, hd, hd ** -0.5, window, sink, cap)
  ops.tree_attention(out, *args)
  return out, args


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_tree_attention(case, dtype):
  out, args = run(case, dtype)
  terms = torch_ops.tree_terms(*args)
  assert close_enough(out, terms, dtype, args[6], int(args[3].max_ctx_len), args[10]) <= 1.0


@pytest.mark.parametrize("hd,page", [(128, 64), (256, 64), (100, 7)])
@pytest.mark.parametrize("rows", [1, 3, 4, 5, 8, 9, 16, 17])
def test_few_rows_in_32_bits(rows, hd, page):
  """Up to 16 rows several warps share a row's keys: contexts that end in each warp's share of a tile, and rows that see few of them."""
  group = 1 if rows % 2 else 2
  items = [(c, rows // group) for c in (0, 5, 30, 61, 64, 700, 1333)]
  out, args = run((items, 2 * group, 2, hd, page, 90, rows % 3 == 0, 0.0, 0.2), torch.float32)
  assert close_enough(out, torch_ops.tree_terms(*args), torch.float32, hd, 1400) <= 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_between_requests_are_left_and_slack_in_the_sizes_does_not_matter(dtype):
  from miniinfer_b200.engine.context import Workspace
  case = ([(150, 9), (70, 20), (3, 1)], 8, 4, 128, 64, None, False, 0.0, 0.0)
  out, args = run(case, dtype)
  for scratch in (None, Workspace(DEV)):
    more, padded = run(case, dtype, scratch=scratch, gap=2, extra_words=1, most=64, longest=4000)
    start, length = padded[3].q_start.tolist(), padded[3].q_len.tolist()
    mine = [t for s, n in zip(start, length) for t in range(s, s + n)]
    rest = [t for t in range(more.shape[0]) if t not in mine]
    assert (more[rest] == 777.0).all()
    assert close_enough(more, torch_ops.tree_terms(*padded), dtype, 128, 4000) <= 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_numbers_that_are_not_finite_reach_only_rows_that_see_them(dtype, bad):
  """Keys and values of a drafted token that one branch sees, and of a context key that the window hides from some rows."""
  from miniinfer_b200.kernels import ops
  case = ([(200, 40)], 8, 2, 128, 64, 60, False, 0.0, 0.0)
  clean, args = run(case, dtype)
  qkv, kv, table, batch = args[:4]
  page = lambda key: int(table[int(batch.seq_slot[0]), key // 64])      # noqa: E731
  mask = [sum((w & 0xffffffff) << 32 * i for i, w in enumerate(row)) for row in batch.tree_mask.tolist()]
  pos = batch.positions.tolist()
  node, key = 7, 145      # a drafted token; a context key at the edge of the window
  for which in (0, 1):
    for place, column in ((200 + node, 3), (key, 90)):
      spoiled = kv.clone()
      spoiled[page(place), which, :, place % 64, column] = bad
      out = torch.full_like(clean, 777.0)
      ops.tree_attention(out, qkv, spoiled, *args[2:])
      sees = [bool(m >> node & 1) if place > 200 else key > p - 60 for m, p in zip(mask, pos)]
      assert any(sees) and not all(sees)
      heads = out.view(40, 8, 128)
      for t, s in enumerate(sees):
        if not s:
          assert torch.equal(out[t], clean[t])
        elif which == 1:
          assert not torch.isfinite(heads[t, :, column]).any()
          other = torch.arange(128, device=DEV) != column
          assert torch.isfinite(heads[t][:, other]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_cap_hides_infinite_scores_and_no_scores_that_are_no_numbers(hd, dtype):
  """Scores far beyond the cap, and infinite ones, are the cap; a key that holds a NaN makes the rows NaN that see it."""
  from miniinfer_b200.kernels import ops
  case = ([(130, 12)], 8, 2, hd, 64, None, False, 5.0, 0.0)
  clean, args = run(case, dtype)
  qkv, kv, table, batch = args[:4]
  node, place = 4, 130 + 4
  sees = [bool(m >> node & 1) for m in batch.tree_mask[:, 0].tolist()]
  assert any(sees) and not all(sees)
  page = int(table[int(batch.seq_slot[0]), place // 64])
  for bad in (float("nan"), 3e38, -3e38, float("inf")):
    spoiled = kv.clone()
    spoiled[page, 0, :, place % 64, 3] = bad
    out = torch.full_like(clean, 777.0)
    ops.tree_attention(out, qkv, spoiled, *args[2:])
    for t, s in enumerate(sees):
      if not s:
        assert torch.equal(out[t], clean[t])
      elif bad != bad:
        assert torch.isnan(out[t]).all()
      else:
        assert torch.isfinite(out[t]).all()


def test_a_chain_is_causal_attention():
  """A tree without branches is a prompt portion: the same as ``attention`` gives."""
  from miniinfer_b200.kernels import ops
  from gpu_helpers import make_attention_case
  items = [(500, 17), (64, 64), (129, 2)]
  for dtype in (torch.float32, torch.bfloat16):
    qkv, kv, bt, batch = make_attention_case(items, 8, 4, 128, 64, dtype, seed=3)
    want, got = (torch.empty((qkv.shape[0], 8 * 128), dtype=dtype, device=DEV) for _ in range(2))
    ops.attention(want, qkv, kv, bt, batch, 8, 4, 128, 128 ** -0.5, None, force_generic=True)
    mask = [words_of((1 << i + 1) - 1, 2) for _, n in items for i in range(n)]
    batch.tree_mask, batch.max_q_len = torch.tensor(mask, dtype=torch.int32, device=DEV), 64
    ops.tree_attention(got, qkv, kv, bt, batch, 8, 4, 128, 128 ** -0.5)
    # both within the bound of test_tree_attention of the definition; values of unit size
    assert (want.double() - got.double()).abs().max() < (2e-5 if dtype == torch.float32 else 3e-2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dtype):
  """The launches of a captured call follow what its lists hold when it is replayed, and two graphs share a workspace."""
  from miniinfer_b200.engine.context import Workspace
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("graphs")
  ws = Workspace(DEV)
  graphs = []
  for case in (([(900, 24), (100, 30)], 16, 4, 128, 64, None, False, 0.0, 0.0), ([(2000, 5)], 8, 8, 64, 64, None, True, 0.0, 0.0)):
    out, args = run(case, dtype, scratch=ws)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    graphs.append((graph, out, args, out.clone()))
  for graph, out, args, _ in graphs:
    with torch.cuda.graph(graph):
      ops.tree_attention(out, *args)
  rng = random.Random(5)
  for turn in range(4):
    for graph, out, args, before in graphs:
      out.fill_(777.0)
      graph.replay()
    for graph, out, args, before in graphs:
      if turn == 0:
        assert torch.equal(out, before)
      else:
        assert close_enough(out, torch_ops.tree_terms(*args), dtype, args[6], 2100) <= 1.0
      batch = args[3]      # other lengths and masks, no longer than those it was captured with
      batch.q_len.sub_(1)
      batch.ctx_len.sub_(rng.randint(1, 40))
      batch.tree_mask.bitwise_and_(rng.randint(0, 1 << 24))


def test_on_a_stream_of_its_own():
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("streams")
  case = ([(1500, 24)], 16, 4, 128, 64, None, False, 0.0, 0.0)
  want, args = run(case, torch.bfloat16)
  torch.cuda.synchronize()
  got = torch.zeros_like(want)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    ops.tree_attention(got, *args)
  side.synchronize()
  assert torch.equal(want, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_beyond_32_bits_of_a_cache(dtype):
  """The last pages of a layer's cache of more than 2^31 values."""
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("memory")
  qkv, kv, table, batch = tree_case([(300, 20), (70, 3)], 16, 8, 128, 64, dtype, seed=9)
  want = torch.empty((qkv.shape[0], 16 * 128), dtype=dtype, device=DEV)
  ops.tree_attention(want, qkv, kv, table, batch, 16, 8, 128, 128 ** -0.5)
  pages = (1 << 31) // kv[0].numel() + kv.shape[0] + 1
  large = torch.zeros((pages,) + kv.shape[1:], dtype=dtype, device=DEV)
  large[-kv.shape[0]:] = kv
  got = torch.empty_like(want)
  ops.tree_attention(got, qkv, large, table + (pages - kv.shape[0]), batch, 16, 8, 128, 128 ** -0.5)
  assert torch.equal(got, want)


@pytest.mark.parametrize("case", [3, 4, 6])
def test_a_workspace_in_which_a_wait_has_run_out_gives_no_numbers(case):
  """Its counters may be off then: rows become NaN instead of sums of some of their pieces, rows of no item stay, and the status says it again."""
  from miniinfer_b200.engine.context import Workspace
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("a status word")
  ws = Workspace(DEV)
  out, args = run(case, torch.bfloat16, scratch=ws, gap=2)
  want = out.clone()
  batch = args[3]
  mine = torch.zeros(out.shape[0], dtype=torch.bool)
  for s, n in zip(batch.q_start.tolist(), batch.q_len.tolist()):
    mine[s:s + n] = True
  assert torch.isfinite(want[mine.to(DEV)]).all() and ops.device_status(ws) == 0
  word = ws.zeros("attention_tree_status", 1, torch.int32)
  word[0] = 64      # as a call leaves it whose wait has run out
  out.fill_(777.0)
  ops.tree_attention(out, *args)
  assert torch.isnan(out[mine.to(DEV)]).all() and (out[~mine.to(DEV)] == 777.0).all()
  assert ops.device_status(ws) == 64
  word[0] = 0
  ops.tree_attention(out, *args)
  assert torch.equal(out, want)


def test_a_call_without_a_workspace_is_not_captured():
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("graphs")
  want, args = run(3, torch.bfloat16)
  out = torch.zeros_like(want)
  with pytest.raises(ops.KernelError, match="captured"):
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
      ops.tree_attention(out, *args)
  ops.tree_attention(out, *args)
  assert torch.equal(out, want)


@pytest.mark.parametrize("case,dtype,kernels", [(3, torch.bfloat16, 1), (5, torch.bfloat16, 2), (10, torch.bfloat16, 2), (3, torch.float32, 2), (0, torch.float32, 1)])
def test_the_launches_of_a_call_are_counted(case, dtype, kernels):
  """One kernel, or two where another one joins the pieces: in bfloat16 where a unit's rows are many, in float32 wherever there are pieces."""
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("launches")
  out, args = run(case, dtype)
  before = ops.launch_count()
  ops.tree_attention(out, *args)
  assert ops.launch_count() - before == kernels
