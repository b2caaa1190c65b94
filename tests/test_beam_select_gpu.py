"""Beam search's selection against its definition in 64 bits."""
import pytest
import torch

import torch_ops
from gpu_helpers import DEV

pytestmark = pytest.mark.gpu

NINF = float("-inf")


def select(logits, cum, start, n, workspace=None):
  from miniinfer_b200.kernels import ops
  requests = len(start) - 1
  out = [torch.full((requests, n), 99, dtype=t, device=DEV) for t in (torch.int32, torch.int32, torch.float32)]
  ops.beam_select(*out, logits, cum, torch.tensor(start, dtype=torch.int32, device=DEV), workspace)
  return out


def statement(logits, cum, start, n):
  requests = len(start) - 1
  out = [torch.zeros((requests, n), dtype=t) for t in (torch.int32, torch.int32, torch.float32)]
  torch_ops.beam_select(*out, logits, cum, torch.tensor(start, dtype=torch.int32))
  return out


def check(got, logits, cum, start, n):
  """The scores of the definition, in its order.  A normaliser errs by less than 3.5e-6: the exponentials by 2^-22 each, their arguments by two
  roundings of up to 12 (what lies further below the maximum has no weight), 25 additions by 2^-24; a score is rounded to float32 once.  So
  two candidates may change places only if their scores are within twice that."""
  tokens, parents, scores = (t.cpu() for t in got)
  want_tokens, want_parents, want = statement(logits, cum, start, n)
  every = torch.log_softmax(logits.double(), dim=1).cpu() + cum.double().cpu()[:, None]
  for i in range(len(start) - 1):
    live = want[i] > NINF
    assert ((scores[i] > NINF) == live).all()
    assert (tokens[i][~live] == -1).all() and (parents[i][~live] == -1).all()
    places = list(zip(parents[i][live].tolist(), tokens[i][live].tolist()))
    assert len(set(places)) == len(places) and all(start[i] <= r < start[i + 1] for r, _ in places)
    mine = torch.tensor([float(every[r, v]) for r, v in places], dtype=torch.float64)
    assert ((scores[i][live].double() - mine).abs() <= 3.5e-6 + 2.0 ** -24 * mine.abs()).all()
    assert ((mine - want[i][live].double()).abs() <= 7e-6 + 2.0 ** -24 * mine.abs()).all()
    sharp = torch.ones_like(live)
    gap = (want[i][1:] - want[i][:-1]).abs() < 1e-5
    sharp[1:] &= ~gap
    sharp[:-1] &= ~gap
    if n:
      sharp[-1] = False      # (its neighbour outside is not known)
    assert torch.equal(tokens[i][live & sharp], want_tokens[i][live & sharp])
    assert torch.equal(parents[i][live & sharp], want_parents[i][live & sharp])


# (beams of each request, vocabulary, places)
SIZES = [
  ([1], 1, 1), ([1], 5, 8), ([2, 1], 31, 3), ([4], 1000, 8), ([1, 0, 3, 0], 2048, 5), ([3], 2049, 17), ([8, 5, 1], 8192, 16), ([2], 50000, 128),
  ([4, 4], 151936, 8), ([12] * 9, 32003, 26), ([64], 4097, 100), ([1] * 70, 513, 2), ([0], 10, 4), ([8] * 40, 9001, 16),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beams,V,n", SIZES)
def test_beam_select(beams, V, n, dtype):
  g = torch.Generator().manual_seed(V + n)
  start = [0]
  for b in beams:
    start.append(start[-1] + b)
  logits = (torch.randn((start[-1], V), generator=g) * 3).to(dtype).to(DEV)
  cum = (-20 * torch.rand(start[-1], generator=g)).to(DEV)
  check(select(logits, cum, start, n), logits, cum, start, n)


@pytest.mark.parametrize("V", [700, 9000, 70000])
def test_equal_scores_go_to_the_lower_row_and_token(V):
  """Logits that are whole numbers, and beams that are alike: ties everywhere, decided by row and token."""
  g = torch.Generator().manual_seed(V)
  one = torch.randint(0, 4, (1, V), generator=g).float()
  for logits in (one.repeat(3, 1), torch.zeros((3, V)), torch.full((3, V), -7.5), one.repeat(3, 1) * -0.0):
    logits, cum = logits.to(DEV), torch.full((3,), -1.25, device=DEV)
    for n in (1, 7, 40, 128):
      tokens, parents, scores = select(logits, cum, [0, 3], n)
      # the largest logit's tokens, row by row, then the next one's
      order = [(-v, r, t) for r in range(3) for t, v in enumerate(logits[r].tolist())]
      order.sort()
      assert tokens[0].tolist() == [t for _, _, t in order[:n]]
      assert parents[0].tolist() == [r for _, r, _ in order[:n]]
      assert (scores[0][1:] <= scores[0][:-1]).all()


@pytest.mark.parametrize("V", [300, 20000])
def test_masked_tokens_ended_beams_and_numbers_that_are_not_finite(V):
  g = torch.Generator().manual_seed(V)
  logits = torch.randn((9, V), generator=g) * 2
  logits[0, torch.rand(V, generator=g) < 0.9] = NINF
  logits[1, 4:] = NINF                      # four tokens are left
  logits[2, :] = NINF                       # none
  logits[3, 17] = float("nan")              # a row that is no distribution
  logits[4, 250] = float("inf")
  logits[5, :V // 2] = NINF                 # whole tiles without a token
  logits[6, :] = torch.finfo(torch.float32).min
  cum = -torch.rand(9, generator=g)
  cum[7] = NINF                             # a beam that has ended
  cum[8] = float("nan")
  logits, cum = logits.to(DEV), cum.to(DEV)
  for start, n in (([0, 9], 12), ([0, 1, 2, 3, 4, 5, 6, 7, 8, 9], 6), ([1, 3, 5], 10)):
    check(select(logits, cum, start, n), logits, cum, start, n)


def test_the_best_of_a_row_may_lie_anywhere():
  """Rising and falling rows, and all of the best tokens in one thread's or one warp's share of a tile."""
  V, n = 40000, 64
  rows = [torch.linspace(-30, 5, V), torch.linspace(5, -30, V)]
  for lo, step in ((0, 1), (8192, 1), (3, 256), (100, 1024), (39000, 1), (4, 4)):
    row = torch.full((V,), -3.0) + torch.arange(V) * 1e-5
    row[lo:lo + step * n:step] = 4 + torch.arange(len(row[lo:lo + step * n:step])) * 0.01
    rows.append(row)
  row = torch.full((V,), NINF)
  row[64:128] = torch.arange(64.0)          # one warp has numbers, the others none
  rows.append(row)
  logits, cum = torch.stack(rows).to(DEV), torch.zeros(len(rows), device=DEV)
  start = list(range(len(rows) + 1))
  check(select(logits, cum, start, n), logits, cum, start, n)
  check(select(logits, cum, [0, len(rows)], 128), logits, cum, [0, len(rows)], 128)


def test_addresses_that_are_not_aligned():
  g = torch.Generator().manual_seed(1)
  for dtype in (torch.float32, torch.bfloat16):
    flat = torch.randn(1 + 4 * 1024, generator=g).to(dtype).to(DEV)
    logits, cum = flat[1:].view(4, 1024), torch.zeros(4, device=DEV)
    check(select(logits, cum, [0, 2, 4], 6), logits, cum, [0, 2, 4], 6)


def test_captured_and_replayed_with_a_shared_workspace():
  from miniinfer_b200.engine.context import Workspace
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("graphs")
  ws, calls = Workspace(DEV), []
  for beams, V, n in (([4, 2], 30000, 8), ([1, 1, 1], 5000, 3)):
    start = [0]
    for b in beams:
      start.append(start[-1] + b)
    logits, cum = torch.randn((start[-1], V), device=DEV), torch.zeros(start[-1], device=DEV)
    out, starts = select(logits, cum, start, n, ws), torch.tensor(start, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    calls.append((graph, out, logits, cum, starts, start, n))
  for graph, out, logits, cum, starts, start, n in calls:
    with torch.cuda.graph(graph):
      ops.beam_select(*out, logits, cum, starts, ws)
  for turn in range(3):
    for graph, out, logits, cum, *_ in calls:
      logits.normal_()
      cum.uniform_()
      graph.replay()
    for _, out, logits, cum, starts, start, n in calls:
      check(out, logits, cum, start, n)


def test_on_a_stream_of_its_own():
  if DEV == "cpu":
    pytest.skip("streams")
  logits, cum = torch.randn((6, 20000), device=DEV), torch.zeros(6, device=DEV)
  want = select(logits, cum, [0, 2, 6], 12)
  torch.cuda.synchronize()
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    got = select(logits, cum, [0, 2, 6], 12)
  side.synchronize()
  assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("start", [[0, 2, 5], [1, 3, 3, 4], [3, 8], [0, 0, 0]])
def test_rows_of_no_request_and_lists_that_end_behind_the_rows(start):
  """Rows in front of the first request and behind the last belong to nobody; a list that goes on past the rows is cut."""
  g = torch.Generator().manual_seed(sum(start))
  logits, cum = torch.randn((5, 6000), generator=g).to(DEV), torch.zeros(5, device=DEV)
  cut = [min(s, 5) for s in start]
  for _ in range(2):      # (the second call finds the counters as the first left them)
    check(select(logits, cum, start, 7), logits, cum, cut, 7)


@pytest.mark.parametrize("V", [50000, 50001])
@pytest.mark.parametrize("n", [3, 128])
def test_many_rows_whose_best_come_early_or_late(n, V):
  """A block walks a whole row: rising rows have more candidates than there is room for, others none in their first tiles, or no more than n."""
  at = torch.arange(V).float()
  rows = [at * 1e-4, -at * 1e-4, (at - 30000).abs() * 1e-4, torch.where(at < 20000, NINF, at * 1e-4), torch.where(at < 4096, NINF, -at * 1e-4),
          torch.where(at % 997 == 5, at * 1e-3, NINF), torch.zeros(V), torch.floor(at / 8192), torch.floor(at / 700), torch.where(at == V - 1, 1.0, NINF),
          torch.full((V,), NINF), torch.randn(V, generator=torch.Generator().manual_seed(V))]
  logits = torch.stack(rows * 13).to(DEV)
  cum = torch.randn(len(logits), generator=torch.Generator().manual_seed(n)).to(DEV)
  cum = cum + torch.arange(len(logits), device=DEV) * 10      # (so that rows do not tie)
  for start in (list(range(len(logits) + 1)), [0, 12, 24, 36, len(logits)]):
    check(select(logits, cum, start, n), logits, cum, start, n)


def test_a_list_that_does_not_rise_harms_no_later_call():
  """What such a call answers is open; the counters of the workspace that it shares with later ones are left as every call finds them."""
  from miniinfer_b200.engine.context import Workspace
  if DEV == "cpu":
    pytest.skip("counters")
  g = torch.Generator().manual_seed(3)
  logits, cum = torch.randn((8, 40000), generator=g).to(DEV), torch.zeros(8, device=DEV)
  for bad in ([0, 5, 2, 8], [4, 0, 8], [0, 3, 1, 6, 8], [8, 6, 4, 2, 0]):
    ws = Workspace(DEV)
    select(logits, cum, [0, 2, 4, 6, 8], 5, ws)
    select(logits, cum, bad, 5, ws)
    assert not ws._bufs[("beam_arrivals", torch.int32)].any()
    for start in ([0, 4, 8], [0, 2, 3, 8], [0, 2, 4, 6, 8]):
      check(select(logits, cum, start, 5, ws), logits, cum, start, 5)
