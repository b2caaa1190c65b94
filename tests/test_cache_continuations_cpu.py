"""Forking, reordering and keeping part of what was appended, on the host: contents, holders of pages, refusals.  The copies are the kernels'
plain statements."""
import random

import pytest
import torch

from miniinfer_b200.cache import FixedStateSpec, KVCacheManager, OutOfPages, OutOfSlots, PageAllocator, PagedKVSpec
from miniinfer_b200.cache.specs import CompositeSpec

pytestmark = pytest.mark.usefixtures("cpu_kernels")


def make(window=None, pages=40, page=4, seqs=8, max_len=64, state=False):
  specs = [PagedKVSpec(1, 2), PagedKVSpec(1, 2)] + ([PagedKVSpec(2, 2, window)] if window else []) + ([FixedStateSpec((3,))] if state else [])
  return KVCacheManager(specs, page, pages, seqs, max_len, torch.float32, "cpu")


def write(m, req, tokens):
  """What a step of these tokens leaves: rows that hold the token, a state that holds a sum over the sequence."""
  first = m.length_of(req)
  m.append(req, len(tokens))
  for g in m.paged_groups:
    for i, (place, t) in enumerate(zip(m.slot_mapping(req, g.index, first, len(tokens)), tokens)):
      g.kv[:, place // g.page_size, :, :, place % g.page_size] = float(t)
  for s in m.state_groups:
    for t in tokens:
      s.state[:, m.slot_of(req)] = s.state[:, m.slot_of(req)] * 0.5 + t


def check(m, sequences):
  m.check_invariants()
  for req, tokens in sequences.items():
    assert m.length_of(req) == len(tokens)
    for g in m.paged_groups:
      first = g.spec.first_needed(len(tokens))
      for pos in range(first, len(tokens)):
        place = m.slot_at(req, g.index, pos)
        assert (g.kv[:, place // g.page_size, :, :, place % g.page_size] == float(tokens[pos])).all()
        assert g.block_table_host[m.slot_of(req), pos // g.page_size] == place // g.page_size
    for s in m.state_groups:
      want = 0.0
      for t in tokens:
        want = want * 0.5 + t
      assert torch.allclose(s.state[:, m.slot_of(req)], torch.tensor(want))


def test_a_shared_page_is_free_when_the_last_holder_has_freed_it():
  a = PageAllocator(3)
  p = a.alloc(2)
  a.share(p)
  a.free(p)
  assert a.num_free == 1 and a.held() == sorted(p) and a.holders(p[0]) == 1
  a.free(p)
  assert a.num_free == 3
  with pytest.raises(AssertionError):
    a.free(p)
  with pytest.raises(AssertionError):
    a.share(p)


@pytest.mark.parametrize("length", [0, 1, 3, 4, 5, 8])
@pytest.mark.parametrize("state", [False, True])
def test_fork(length, state):
  m = make(state=state)
  m.admit("a")
  tokens = list(range(10, 10 + length))
  write(m, "a", tokens)
  m.commit("a", length)
  before = m.free_pages()[0]
  m.fork("a", ["b", "c"])
  assert m.free_pages()[0] == before - (2 if length % 4 else 0)
  seqs = {"a": tokens, "b": tokens, "c": tokens}
  check(m, seqs)
  for k, q in enumerate("abc"):      # each goes its own way
    write(m, q, [100 * (k + 1), 100 * (k + 1) + 1])
    m.commit(q, 2)
    seqs[q] = tokens + [100 * (k + 1), 100 * (k + 1) + 1]
  check(m, seqs)
  for q in "bac":
    m.release_request(q)
    del seqs[q]
    check(m, seqs)
  assert m.free_pages()[0] == 40


def test_refusals_change_nothing():
  m = make(pages=3, seqs=3)
  m.admit("a")
  write(m, "a", [1, 2, 3, 4, 5])
  with pytest.raises(ValueError):
    m.fork("a", ["b"])                      # not settled
  m.commit("a", 5)
  with pytest.raises(OutOfSlots):
    m.fork("a", ["b", "c", "d"])
  with pytest.raises(OutOfPages):
    m.fork("a", ["b", "c"])                 # two pages for what the last one holds, one is free
  with pytest.raises(KeyError):
    m.fork("a", ["a"])
  with pytest.raises(KeyError):
    m.fork("a", ["b", "b"])
  check(m, {"a": [1, 2, 3, 4, 5]})
  m.fork("a", ["b"])
  with pytest.raises(KeyError):
    m.reorder({"a": "x", "b": "a"})
  with pytest.raises(KeyError):
    m.reorder({"a": "b"})                   # a parent that is not itself reordered
  m.append("a", 2)
  for kept in ([2], [-1], [1, 1], [1, 0]):
    with pytest.raises(ValueError):
      m.keep({"a": kept})
  m.cancel("a", 2)
  check(m, {"a": [1, 2, 3, 4, 5], "b": [1, 2, 3, 4, 5]})
  s = make(state=True)
  s.admit("a")
  s.append("a", 3)
  with pytest.raises(ValueError):
    s.keep({"a": [0, 2]})


@pytest.mark.parametrize("window", [None, 6])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_calls(seed, state, window):
  rng = random.Random(seed)
  m, seqs, names = make(window=window, state=state), {}, iter(range(10 ** 6))
  for _ in range(150):
    what = rng.choice(("admit", "step", "step", "step", "fork", "reorder", "reorder", "keep", "release"))
    if what == "admit" and m.num_free_slots:
      q = next(names)
      m.admit(q)
      seqs[q] = []
    elif what == "step" and seqs:
      q = rng.choice(sorted(seqs))
      n = rng.randint(1, 6)
      if m.can_append(q, n):
        tokens = [rng.randint(1, 999) for _ in range(n)]
        write(m, q, tokens)
        m.commit(q, n)
        seqs[q] = seqs[q] + tokens
    elif what == "fork" and seqs:
      q = rng.choice(sorted(seqs))
      children = [next(names) for _ in range(rng.randint(1, 3))]
      try:
        m.fork(q, children)
        seqs.update({c: list(seqs[q]) for c in children})
      except (OutOfPages, OutOfSlots):
        pass
    elif what == "reorder" and seqs:
      group = rng.sample(sorted(seqs), rng.randint(1, len(seqs)))
      parents = {q: rng.choice(group) for q in group}
      try:
        m.reorder(parents)
        seqs.update({q: list(s) for q, s in {q: seqs[p] for q, p in parents.items()}.items()})
      except OutOfPages:
        pass
    elif what == "keep" and seqs:
      kept, new = {}, {}
      for q in rng.sample(sorted(seqs), rng.randint(1, len(seqs))):
        n = rng.randint(1, 9)
        if not m.can_append(q, n):
          continue
        tokens = [rng.randint(1, 999) for _ in range(n)]
        write(m, q, tokens)
        nodes = list(range(n)) if state else sorted(rng.sample(range(n), rng.randint(0, n)))
        kept[q], new[q] = nodes, [tokens[i] for i in nodes]
      m.keep(kept)
      for q in kept:
        seqs[q] = seqs[q] + new[q]
    elif what == "release" and seqs:
      q = rng.choice(sorted(seqs))
      m.release_request(q)
      del seqs[q]
    check(m, seqs)


def test_a_composite_layer_is_forked_whole():
  m = KVCacheManager([CompositeSpec((PagedKVSpec(1, 2), FixedStateSpec((3,)))), None], 4, 10, 3, 32, torch.float32, "cpu")
  m.admit("a")
  write(m, "a", [1, 2, 3])
  m.commit("a", 3)
  m.fork("a", ["b"])
  check(m, {"a": [1, 2, 3], "b": [1, 2, 3]})


def test_more_copies_than_go_in_one_call(monkeypatch):
  """A call of the copies takes MOVE_MAX_PAIRS pairs at most, of pages and of states."""
  from miniinfer_b200.kernels import ops
  most, calls = 3, []
  monkeypatch.setattr(ops, "MOVE_MAX_PAIRS", most)
  for name in ("copy_cache_pages", "reorder_states"):
    def limited(base, src, *rest, plain=getattr(ops, name), name=name):
      if src.shape[0] > most:
        raise ops.KernelError(f"{src.shape[0]} pairs")
      calls.append((name, src.shape[0]))
      plain(base, src, *rest)
    monkeypatch.setattr(ops, name, limited)
  m = make(seqs=9, state=True)
  m.admit(0)
  write(m, 0, [1, 2, 3, 4, 5])
  m.commit(0, 5)
  m.fork(0, range(1, 9))
  seqs = {q: [1, 2, 3, 4, 5] for q in range(9)}
  check(m, seqs)
  assert sorted(calls) == sorted([("copy_cache_pages", n) for n in (3, 3, 2)] + [("reorder_states", n) for n in (3, 3, 2)])
  for q in range(9):
    write(m, q, [10 + q])
    m.commit(q, 1)
    seqs[q] = seqs[q] + [10 + q]
  m.reorder({q: 4 + q % 2 for q in range(9)})
  check(m, {q: seqs[4 + q % 2] for q in range(9)})


@pytest.mark.parametrize("fails", ["copy_cache_pages", "copy_cache_pages, the second group", "reorder_states"])
@pytest.mark.parametrize("pages", [40, 10])
def test_an_error_of_a_launch_leaves_the_requests_as_they_were(pages, fails, monkeypatch):
  from miniinfer_b200.kernels import ops
  m = make(window=6, pages=pages, seqs=5, state=True)
  seqs = {}
  for q, n in (("a", 5), ("b", 9), ("c", 2)):
    m.admit(q)
    seqs[q] = [100 * len(seqs) + i for i in range(n)]
    write(m, q, seqs[q])
    m.commit(q, n)

  def everything():
    return (m.free_pages(), sorted(m._free_slots), [g.block_table_host.copy().tolist() for g in m.paged_groups], [list(g.allocator._held) for g in m.paged_groups],
            {q: (r.slot, r.length, r.reserved, [list(p) for p in r.pages]) for q, r in m._requests.items()})

  name, plain, left = fails.split(",")[0], getattr(ops, fails.split(",")[0]), [1 if "second" in fails else 0]

  def failing(*args):
    if not left[0]:
      raise ops.KernelError("a launch failed")
    left[0] -= 1
    plain(*args)

  before = everything()
  for call in (lambda: m.fork("b", ["d", "e"]), lambda: m.reorder({"a": "b", "b": "b", "c": "a"})):
    with monkeypatch.context() as patch:
      patch.setattr(ops, name, failing)
      left[0] = 1 if "second" in fails else 0
      with pytest.raises(ops.KernelError):
        call()
    assert everything() == before
    m.check_invariants()
  for q in "ab":      # what a request goes on from is as it was
    check(m, {q: seqs[q]})
  m.reorder({"a": "b", "b": "b", "c": "a"})
  seqs = {"a": seqs["b"], "b": seqs["b"], "c": seqs["a"]}
  check(m, seqs)
  for q in "abc":
    m.release_request(q)
  assert m.free_pages() == [g.num_pages for g in m.paged_groups]


def test_copies_go_into_the_pages_that_come_back():
  m = make(pages=4, seqs=3)
  seqs = {"a": [1, 2, 3, 4, 5], "b": [6, 7], "c": [8]}
  for q, tokens in seqs.items():
    m.admit(q)
    write(m, q, tokens)
    m.commit(q, len(tokens))
  assert m.free_pages() == [0]
  m.reorder({"a": "a", "b": "a", "c": "a"})
  check(m, {q: seqs["a"] for q in "abc"})
  assert m.free_pages() == [0]
  m.release_request("c")
  m.fork("a", ["d"])
  check(m, {q: seqs["a"] for q in "abd"})
  with pytest.raises(OutOfPages):
    m.append("a", 4)
