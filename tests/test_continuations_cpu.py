"""What the operators for several continuations of a request refuse; no kernel runs."""
import pytest
import torch

from miniinfer_b200.kernels import ops
from miniinfer_b200.kernels.ops import KernelError

I32 = torch.int32


def beam(**change):
  a = dict(tokens=torch.zeros((2, 4), dtype=I32), parents=torch.zeros((2, 4), dtype=I32), scores=torch.zeros((2, 4)), logits=torch.zeros((3, 10)),
           cum=torch.zeros(3), row_start=torch.zeros(3, dtype=I32))
  a.update(change)
  ops.beam_select(**a)


@pytest.mark.parametrize("change", [
  {}, dict(logits=torch.zeros(10)), dict(cum=torch.zeros(4)), dict(parents=torch.zeros((2, 5), dtype=I32)), dict(scores=torch.zeros((1, 4))),
  dict(row_start=torch.zeros(4, dtype=I32)), dict(logits=torch.zeros((3, 10), dtype=torch.float16)), dict(logits=torch.zeros((3, 0))),
  dict(tokens=torch.zeros((2, 0), dtype=I32), parents=torch.zeros((2, 0), dtype=I32), scores=torch.zeros((2, 0))),
  dict(tokens=torch.zeros((2, 129), dtype=I32), parents=torch.zeros((2, 129), dtype=I32), scores=torch.zeros((2, 129))),
])
def test_beam_select_refuses(change):
  with pytest.raises(KernelError):
    beam(**change)


def test_moves_refuse():
  ints = lambda *x: torch.tensor(x, dtype=I32)      # noqa: E731
  state, kv = torch.zeros((2, 4, 8)), torch.zeros((2, 4, 2, 1, 8, 16))
  for call in (
      lambda: ops.reorder_states(state, ints(0), ints(1)),                                  # not on a device
      lambda: ops.reorder_states(state, ints(0, 1), ints(1)),
      lambda: ops.reorder_states(state.transpose(0, 1), ints(0), ints(1)),
      lambda: ops.reorder_states(state[0, 0], ints(0), ints(1)),
      lambda: ops.reorder_states(state, torch.zeros(4097, dtype=I32), torch.zeros(4097, dtype=I32)),
      lambda: ops.copy_cache_pages(kv, ints(0), ints(1)),
      lambda: ops.copy_cache_pages(kv[0], ints(0), ints(1)),
      lambda: ops.copy_cache_pages(kv, ints(0), ints(1), ints(1, 2)),
      lambda: ops.copy_cache_pages(kv[:, :, :, :, ::2], ints(0), ints(1)),
      lambda: ops.copy_cache_pages(kv, torch.zeros(4097, dtype=I32), torch.zeros(4097, dtype=I32)),
      lambda: ops.move_cache_rows(kv, ints(0), ints(1), ints(0, 1), 1),
      lambda: ops.move_cache_rows(kv, ints(0), ints(1), ints(0, 1), 0),
      lambda: ops.move_cache_rows(kv, ints(0), ints(1, 2), ints(0, 1), 1),
      lambda: ops.move_cache_rows(kv[:, :, :1], ints(0), ints(1), ints(0, 1), 1)):
    with pytest.raises(KernelError):
      call()


def test_tree_attention_refuses():
  def call(change=None, batch_change=None):
    a = dict(out=torch.zeros((3, 32)), qkv=torch.zeros((3, 64)), kv_layer=torch.zeros((4, 2, 1, 16, 16)), block_table=torch.zeros((1, 4), dtype=I32),
             num_heads=2, num_kv_heads=1, head_dim=16, scale=0.25)
    one = torch.ones(1, dtype=I32)
    b = dict(q_start=one * 0, q_len=one * 3, ctx_len=one * 8, seq_slot=one * 0, num_items=1, max_q_len=3, max_ctx_len=8,
             tree_mask=torch.zeros((3, 1), dtype=I32), positions=torch.zeros(3, dtype=I32))
    a.update(change or {})
    b.update(batch_change or {})
    ops.tree_attention(batch=ops.AttentionBatch(**b), **a)

  for change in (None, dict(out=torch.zeros((3, 31))), dict(out=torch.zeros((3, 32), dtype=torch.bfloat16)), dict(qkv=torch.zeros((3, 31))),
                 dict(kv_layer=torch.zeros((4, 2, 2, 16, 16))), dict(kv_layer=torch.zeros((4, 2, 1, 16, 16), dtype=torch.bfloat16)), dict(num_heads=3, num_kv_heads=2),
                 dict(softcap=-1.0), dict(window=-2), dict(sink=torch.zeros(3)), dict(block_table=torch.zeros(4, dtype=I32)), dict(head_dim=641)):
    with pytest.raises(KernelError):
      call(change)
  for change in (dict(tree_mask=None), dict(max_q_len=None), dict(max_ctx_len=None), dict(max_q_len=33), dict(tree_mask=torch.zeros((2, 1), dtype=I32)), dict(num_items=2)):
    with pytest.raises(KernelError):
      call(None, change)
  with pytest.raises(KernelError):
    call(dict(window=4), dict(positions=None))


@pytest.mark.parametrize("code,name", [(64, "attention over trees"), (128, "its place in shared memory")])
def test_a_wait_that_ran_out_over_a_tree_is_told_from_those_of_other_kernels(code, name):
  """A bit of its own for each: 2 is the prefill attention's, 4 the tcgen05 matrix product's."""
  import os
  import re
  from types import SimpleNamespace

  from miniinfer_b200.engine.context import Workspace
  from miniinfer_b200.engine.runner import ModelRunner
  from miniinfer_b200.kernels import build
  source = open(os.path.join(build.CSRC, "attention_tree_tc.cu"), encoding="utf-8").read()
  bits = dict(re.findall(r"(STATUS_\w+) = (\d+)", source))
  assert str(code) in bits.values()
  assert set(re.findall(r"atomic(?:Exch|Or)\(\w*\.?status, (\w+)\)", source)) == set(bits)      # the kernel sets these and no others
  ws = Workspace(torch.device("cpu"))
  word = ws.zeros("attention_tree_status", 1, torch.int32)
  runner = SimpleNamespace(ws=ws, _graphs={}, _step_graphs={})
  ModelRunner.check_status(runner)
  word[0] = code
  with pytest.raises(KernelError, match=f"status bits {code}:.* {code} {name}"):
    ModelRunner.check_status(runner)
