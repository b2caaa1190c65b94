"""Copies inside caches and states, bit for bit against plain statements: every source is read before any destination is written."""
import random

import pytest
import torch

import torch_ops
from gpu_helpers import DEV

pytestmark = pytest.mark.gpu


def ints(x):
  return torch.tensor(x, dtype=torch.int32, device=DEV)


def filled_tensor(shape, dtype, seed):
  g = torch.Generator().manual_seed(seed)
  if dtype.is_floating_point:
    return torch.randn(shape, generator=g).to(dtype).to(DEV)
  return torch.randint(0, 100, shape, generator=g).to(dtype).to(DEV)


def compare(name, base, *args):
  from miniinfer_b200.kernels import ops
  want = base.clone()
  getattr(torch_ops, name)(want, *args)
  getattr(ops, name)(base, *args)
  assert torch.equal(base, want)


@pytest.mark.parametrize("layers,slots,shape,pairs,dtype", [
  (1, 3, (5,), 2, torch.float32), (6, 17, (2048, 3), 4, torch.float32), (3, 65, (2, 64, 64), 64, torch.float32), (2, 9, (33,), 8, torch.bfloat16),
  (2, 300, (7, 5), 300, torch.float32), (1, 40, (100000,), 17, torch.bfloat16), (4, 8, (1,), 8, torch.uint8), (1, 4100, (64,), 4096, torch.float32),
  (2, 5, (16, 128, 128), 5, torch.float32), (3, 12, (3,), 12, torch.float64),
])
def test_reorder_states(layers, slots, shape, pairs, dtype):
  rng = random.Random(slots)
  for turn in range(3):
    state = filled_tensor((layers, slots) + shape, dtype, turn)
    dst = rng.sample(range(slots), pairs)
    if turn == 0:      # beams that change places, some of them twice a parent
      src = [rng.choice(dst) for _ in dst]
    elif turn == 1:    # a cycle through all of them
      src = dst[1:] + dst[:1]
    else:
      src = [rng.randrange(slots) for _ in dst]
    compare("reorder_states", state, ints(src), ints(dst))


def test_pairs_out_of_range_are_left_out():
  state = filled_tensor((2, 6, 40), torch.float32, 0)
  compare("reorder_states", state, ints([0, -1, 6, 3, 1 << 30]), ints([1, 2, 3, -1, 4]))
  compare("reorder_states", state, ints([5, 5, -7]), ints([0, 5, 6]))
  kv = filled_tensor((2, 5, 2, 2, 8, 16), torch.bfloat16, 1)
  compare("copy_cache_pages", kv, ints([1, 9, -1, 2]), ints([0, 3, 4, 5]))
  compare("copy_cache_pages", kv, ints([1, 3, 2]), ints([0, 4, 3]), ints([0, -5, 100]))
  compare("move_cache_rows", kv, ints([3, 40, -1, 7]), ints([1, 2, 3, 45]), ints([0, 4]), 4)
  compare("move_cache_rows", kv, ints([3, 4]), ints([1, 2]), ints([0, 1]), 2)      # a pair of no group


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,pages,heads,P,hd,pairs", [
  (1, 4, 1, 16, 64, 1), (28, 12, 8, 64, 128, 4), (3, 70, 2, 32, 80, 60), (2, 30, 3, 7, 33, 15), (1, 1100, 1, 16, 16, 1024), (4, 20, 2, 128, 256, 9),
])
def test_copy_cache_pages(layers, pages, heads, P, hd, pairs, dtype):
  rng = random.Random(pairs)
  for partial in (False, True):
    kv = filled_tensor((layers, pages, 2, heads, P, hd), dtype, pairs)
    dst = rng.sample(range(pages), pairs)
    src = [rng.randrange(pages) for _ in dst]      # some pages several times, some of them destinations too
    filled = ints([rng.randint(0, P) for _ in dst]) if partial else None
    compare("copy_cache_pages", kv, ints(src), ints(dst), filled)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,groups,nodes,kept,heads,P,hd", [
  (1, 1, 2, 1, 1, 16, 64), (28, 1, 16, 4, 8, 64, 128), (3, 20, 64, 8, 8, 64, 128), (2, 5, 100, 60, 2, 16, 80), (2, 3, 9, 9, 3, 5, 33), (1, 2, 300, 256, 2, 64, 256),
  (1, 70, 5, 2, 4, 16, 16),
])
def test_move_cache_rows(layers, groups, nodes, kept, heads, P, hd, dtype):
  rng, span = random.Random(nodes), -(-nodes // P) + 1
  pages = list(range(1, groups * span + 1))
  rng.shuffle(pages)
  for turn in range(3):
    src, dst, start = [], [], [0]
    for q in range(groups):
      mine, first = pages[q * span:(q + 1) * span], rng.randrange(P)
      place = lambda i: mine[(first + i) // P] * P + (first + i) % P      # noqa: E731
      n = rng.randint(0, kept) if turn else kept
      path = rng.sample(range(nodes), n)
      if turn < 2:      # an accepted path: to the front, in order; else any rows in any order
        path.sort()
      src += [place(i) for i in path]
      dst += [place(i) for i in (range(n) if turn < 2 else rng.sample(range(nodes), n))]
      start.append(len(src))
    kv = filled_tensor((layers, len(pages) + 1, 2, heads, P, hd), dtype, turn)
    # paths that move to the front may go a few rows at a time
    for most in ((kept, max(1, kept // 3)) if turn < 2 else (kept,)):
      compare("move_cache_rows", kv, ints(src), ints(dst), ints(start), most)


def test_rows_that_change_places_and_do_not_fit_a_block_whole():
  """A cycle through more bytes of rows than a block's shared memory holds: still read before they are written."""
  for dtype, dim in ((torch.float32, 512), (torch.bfloat16, 36)):
    kv = filled_tensor((1, 20, 2, 1, 64, dim), dtype, dim)
    places = random.Random(1).sample(range(64, 20 * 64), 1100)
    compare("move_cache_rows", kv, ints(places), ints(places[1:] + places[:1]), ints([0, 1100]), 1100)


def test_places_that_pass_32_bits():
  """Offsets in bytes and in values beyond 2^32: 5 GiB of pages, the last of them."""
  if DEV == "cpu":
    pytest.skip("memory")
  from miniinfer_b200.kernels import ops
  kv = torch.zeros((2, 2600, 2, 8, 64, 1024 // 2), dtype=torch.bfloat16, device=DEV)
  assert kv.numel() > 1 << 31
  kv[:, 2599] = 3
  kv[1, 2598, 1, 7, 63] = 5
  ops.copy_cache_pages(kv, ints([2599]), ints([2500]))
  ops.move_cache_rows(kv, ints([2598 * 64 + 63]), ints([2597 * 64 + 1]), ints([0, 1]), 1)
  assert (kv[:, 2500] == 3).all() and (kv[1, 2597, 1, 7, 1] == 5).all() and kv[1, 2597].float().sum() == 5 * 512
  ops.reorder_states(kv.view(2, 2600, -1), ints([2598, 2599]), ints([2599, 2598]))
  assert (kv[:, 2598] == 3).all() and (kv[1, 2599, 1, 7, 63] == 5).all()


def test_captured_and_replayed():
  from miniinfer_b200.kernels import ops
  if DEV == "cpu":
    pytest.skip("graphs")
  state, kv = filled_tensor((2, 8, 300), torch.float32, 0), filled_tensor((2, 9, 2, 2, 16, 64), torch.bfloat16, 1)
  src, dst, start = ints([0, 1, 2, 3]), ints([1, 0, 3, 2]), ints([0, 2, 4])
  ops.reorder_states(state, src, dst)
  ops.move_cache_rows(kv, src, dst, start, 2)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    ops.reorder_states(state, src, dst)
    ops.copy_cache_pages(kv, src, dst)
    ops.move_cache_rows(kv, src, dst, start, 2)
  for a, b in (([4, 5, 6, 7], [0, 1, 2, 3]), ([3, 2, 1, 0], [2, 3, 0, 1]), ([-1, 7, 2, 2], [1, 0, -1, 5])):
    src.copy_(ints(a))
    dst.copy_(ints(b))
    want_state, want_kv = state.clone(), kv.clone()
    torch_ops.reorder_states(want_state, src, dst)
    torch_ops.copy_cache_pages(want_kv, src, dst)
    torch_ops.move_cache_rows(want_kv, src, dst, start, 2)
    graph.replay()
    assert torch.equal(state, want_state) and torch.equal(kv, want_kv)


@pytest.mark.parametrize("heads,P,hd,pairs", [(1, 4, 16, 4096), (3, 7, 5, 1000), (2, 64, 64, 300), (1, 1, 8, 40)])
def test_many_pages_in_part(heads, P, hd, pairs):
  """Lists of up to the most pairs, of pages that are filled to any length, not at all, beyond their end, or padded."""
  rng = random.Random(pairs)
  ids = list(range(2 * pairs + 1))
  rng.shuffle(ids)
  src, dst = ids[:pairs], ids[pairs:2 * pairs]
  dst[1], src[2], src[3], dst[4] = -1, len(ids), dst[5], src[5]      # padding, out of range, a page that is written and read, and one read and written
  filled = [rng.randint(-1, P + 1) for _ in src]
  kv = filled_tensor((2, len(ids), 2, heads, P, hd), torch.bfloat16, P)
  compare("copy_cache_pages", kv, ints(src), ints(dst), ints(filled))
