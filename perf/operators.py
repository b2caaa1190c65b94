"""Operators for requests that have several open continuations - beams, trees of drafted tokens - as cases whose time can be measured.

Kinds of cases:

  * ``beam``    the best ``n`` continuations of a request over all of its beams and the vocabulary;
  * ``states``  the per-request states of a model's layers, put in the order of the beams that go on;
  * ``pages``   pages of a cache copied for a fork, whole or as far as they are filled, over all layers of a pool;
  * ``rows``    rows of a cache moved: the accepted path of a drafted tree goes to the front of the tree's rows;
  * ``tree``    attention of the tokens of a drafted tree over a paged cache.

Every kind has a plain form in elementary operations (``own = False``), the framework's call (``own = True``) and its definition in 64 bits
(``exact``).  Sizes: the Qwen3-0.6B and 8B shapes, the sizes of the recurrent mixers' states, and generic ones.
``ragged`` is 0 where all requests are alike; otherwise the sizes of the requests are drawn from it."""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
VOCAB = 151936


# ------------------------------------------------------------------------------------------------ the cases


def listed():
  return [
      # the step after a prompt: one request, four beams, the smallest call of a selection
      {"name": "beam_one_request", "kind": "beam", "ragged": 0, "requests": 1, "beams": 4, "n": 8, "vocab": VOCAB, "masked": False, "dtype": "float32"},
      # a loaded server: 64 requests with up to eight beams each, twice as many continuations wanted as there are beams
      {"name": "beam_64_requests", "kind": "beam", "ragged": 64, "requests": 64, "beams": 8, "n": 16, "vocab": VOCAB, "masked": False, "dtype": "float32"},
      # a short convolution's window of four beams in a small model: latency alone
      {"name": "states_conv_4", "kind": "states", "layers": 6, "slots": 17, "requests": 1, "beams": 4, "row": 3 * 2048, "dtype": "float32"},
      # matrix states, 16 heads of 128 x 128, of eight requests with four beams each
      {"name": "states_matrix_32", "kind": "states", "layers": 12, "slots": 65, "requests": 8, "beams": 4, "row": 16 * 128 * 128, "dtype": "float32"},
      # a fork into four: the last, partly filled page of a request, for three more beams
      {"name": "pages_fork_3", "kind": "pages", "layers": 28, "pages": 64, "pairs": 3, "partial": True, "heads": 8, "page": 64, "dim": 128, "dtype": "bfloat16"},
      # prompts copied whole
      {"name": "pages_whole_96", "kind": "pages", "layers": 28, "pages": 224, "pairs": 96, "partial": False, "heads": 8, "page": 64, "dim": 128, "dtype": "bfloat16"},
      # one user: four of sixteen drafted tokens are accepted
      {"name": "rows_one_request", "kind": "rows", "layers": 28, "requests": 1, "nodes": 16, "kept": 4, "heads": 8, "page": 64, "dim": 128, "dtype": "bfloat16"},
      # 64 users with trees of 64
      {"name": "rows_64_requests", "kind": "rows", "layers": 28, "requests": 64, "nodes": 64, "kept": 8, "heads": 8, "page": 64, "dim": 128, "dtype": "bfloat16"},
      # one user in the middle of an answer, eight drafted tokens
      {"name": "tree_one_request", "kind": "tree", "ragged": 0, "requests": 1, "nodes": 8, "context": 2047, "heads": 16, "kv_heads": 8, "dim": 128,
       "page": 64, "window": 0, "sink": False, "softcap": 0.0, "empty": False, "dtype": "bfloat16"},
      # eight users with trees of 32, contexts of any length
      {"name": "tree_8_ragged", "kind": "tree", "ragged": 8, "requests": 8, "nodes": 32, "context": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
       "page": 64, "window": 0, "sink": False, "softcap": 0.0, "empty": False, "dtype": "bfloat16"},
      # a loaded server: 32 users with trees of 64 over long contexts
      {"name": "tree_32_long", "kind": "tree", "ragged": 32, "requests": 32, "nodes": 64, "context": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
       "page": 64, "window": 0, "sink": False, "softcap": 0.0, "empty": False, "dtype": "bfloat16"},
      # the true float32 path, as a trace is replayed to check results: an odd tree, small pages
      {"name": "tree_float32", "kind": "tree", "ragged": 3, "requests": 3, "nodes": 13, "context": 1000, "heads": 16, "kv_heads": 8, "dim": 128,
       "page": 16, "window": 0, "sink": False, "softcap": 0.0, "empty": False, "dtype": "float32"},
  ]


def _about(rng, low, high):
  """A whole number of low .. high, spread over its logarithm."""
  return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
  kind = rng.choice(("beam", "beam", "states", "pages", "rows", "tree", "tree", "tree"))
  dtype = "float32" if rng.random() < 0.25 else "bfloat16"
  if kind == "beam":
    beams, vocab = rng.randint(1, 12), rng.choice((VOCAB, _about(rng, 50, 200000)))
    requests = _about(rng, 1, max(1, min(64, 512 * VOCAB // (beams * vocab))))
    return {"kind": kind, "requests": requests, "beams": beams, "ragged": rng.choice((0, 0, rng.randint(1, 1 << 20))), "n": rng.randint(1, 2 * beams + 2), "vocab": vocab,
            "masked": rng.random() < 0.3, "dtype": "bfloat16" if rng.random() < 0.3 else "float32"}
  if kind == "states":
    row, layers, beams = _about(rng, 1, 16 * 128 * 128), rng.randint(1, 12), rng.randint(1, 8)
    requests = _about(rng, 1, 64 // beams)
    return {"kind": kind, "layers": layers, "slots": requests * beams + rng.randint(1, 9), "requests": requests, "beams": beams, "row": row,
            "dtype": "bfloat16" if rng.random() < 0.3 else "float32"}
  if kind in ("pages", "rows"):
    shape = {"heads": rng.choice((1, 2, 4, 8)), "page": rng.choice((16, 32, 64, 128)), "dim": rng.choice((64, 80, 128, 256))}
    layers = rng.randint(1, 28)
    page_bytes = layers * 2 * shape["heads"] * shape["page"] * shape["dim"] * (2 if dtype == "bfloat16" else 4)
    if kind == "pages":
      pairs = _about(rng, 1, max(1, min(512, 700_000_000 // page_bytes)))
      return dict(shape, kind=kind, layers=layers, pages=2 * pairs + rng.randint(1, 20), pairs=pairs, partial=rng.random() < 0.5, dtype=dtype)
    nodes = _about(rng, 2, 128)
    most = max(1, 1_400_000_000 // (page_bytes * (-(-nodes // shape["page"]) + 1)))
    return dict(shape, kind=kind, layers=layers, requests=_about(rng, 1, min(64, most)), nodes=nodes, kept=rng.randint(1, min(nodes, 16)), dtype=dtype)
  heads, kv_heads = rng.choice(((16, 8), (32, 8), (64, 8), (8, 8), (12, 2), (20, 4)))
  dim, nodes, context = rng.choice((64, 128, 128, 80, 256)), _about(rng, 1, 64), _about(rng, 1, 8192)
  if dtype == "float32":
    context = min(context, 1024)
  work = nodes * context * heads * dim * (16 if dtype == "float32" else 1)
  requests = _about(rng, 1, max(1, min(64, 64 * 8192 * 32 * 128 * 16 // work)))
  return {"kind": kind, "requests": requests, "nodes": nodes, "context": context, "ragged": rng.choice((0, rng.randint(1, 1 << 20), rng.randint(1, 1 << 20))), "heads": heads, "kv_heads": kv_heads,
          "dim": dim, "page": rng.choice((16, 32, 64, 64, 128)), "window": rng.choice((0, 0, 0, _about(rng, 16, 4096))), "sink": rng.random() < 0.25,
          "softcap": rng.choice((0.0, 0.0, 30.0)), "empty": rng.random() < 0.2, "dtype": dtype}


# ------------------------------------------------------------------------------------------------ the inputs


def _device_rng(seed):
  g = torch.Generator(device=DEVICE)
  g.manual_seed(seed)
  return g


def _ints(values, dtype=torch.int32):
  return torch.tensor(values, dtype=dtype, device=DEVICE)


def _dtype(case):
  return getattr(torch, case["dtype"])


def _beam_rows(case):
  """The number of beams of every request."""
  rng = random.Random(case["ragged"])
  return [rng.randint(1, case["beams"]) if case["ragged"] else case["beams"] for _ in range(case["requests"])]


def _prepare_beam(case, seed):
  g, counts = _device_rng(seed), _beam_rows(case)
  start = [0]
  for c in counts:
    start.append(start[-1] + c)
  rows, n = start[-1], case["n"]
  logits = torch.randn((rows, case["vocab"]), generator=g, device=DEVICE) * 3.0
  cum = -torch.rand(rows, generator=g, device=DEVICE) * 20.0
  if case["masked"]:      # tokens that a grammar forbids, and beams that have ended
    logits[torch.rand(logits.shape, generator=g, device=DEVICE) < 0.4] = -math.inf
    cum[torch.rand(rows, generator=g, device=DEVICE) < 0.2] = -math.inf
  out = [torch.empty((case["requests"], n), dtype=t, device=DEVICE) for t in (torch.int32, torch.int32, torch.float32)]
  return {"logits": logits.to(_dtype(case)), "cum": cum, "start": _ints(start), "most": max(counts), "out": out}


def _prepare_states(case, seed):
  g, rng = _device_rng(seed), random.Random(seed)
  state = torch.randn((case["layers"], case["slots"], case["row"]), generator=g, device=DEVICE).to(_dtype(case))
  slots = rng.sample(range(case["slots"]), case["requests"] * case["beams"])
  src, dst = [], []
  for r in range(case["requests"]):
    mine = slots[r * case["beams"]:(r + 1) * case["beams"]]
    for s in mine:      # a beam goes on from any beam of its request, itself among them
      src.append(rng.choice(mine))
      dst.append(s)
  return {"state": state, "src": _ints(src), "dst": _ints(dst)}


def _prepare_pages(case, seed):
  g, rng = _device_rng(seed), random.Random(seed)
  kv = torch.randn((case["layers"], case["pages"], 2, case["heads"], case["page"], case["dim"]), generator=g, device=DEVICE, dtype=_dtype(case))
  ids = rng.sample(range(case["pages"]), 2 * case["pairs"])
  src, dst = ids[:case["pairs"]], ids[case["pairs"]:]
  if case["partial"]:      # one page forked several times, as far as it is filled
    src = [src[0]] * case["pairs"]
  rows = [rng.randint(1, case["page"])] * case["pairs"] if case["partial"] else None
  return {"kv": kv, "src": _ints(src), "dst": _ints(dst), "rows": _ints(rows) if rows else None}


def _paths(case, seed):
  """For every request the rows of its accepted path, from and to, as places page * page_size + offset; and the number of pages."""
  rng, P = random.Random(seed), case["page"]
  span = -(-case["nodes"] // P) + 1
  pages = list(range(1, case["requests"] * span + 1))
  rng.shuffle(pages)
  src, dst, start = [], [], [0]
  for r in range(case["requests"]):
    mine = pages[r * span:(r + 1) * span]
    first = rng.randint(0, P - 1)      # where the tree begins in its first page
    kept = sorted(rng.sample(range(case["nodes"]), case["kept"]))
    place = lambda i: mine[(first + i) // P] * P + (first + i) % P      # noqa: E731
    src += [place(i) for i in kept]
    dst += [place(i) for i in range(len(kept))]
    start.append(len(src))
  return src, dst, start, len(pages) + 1


def _prepare_rows(case, seed):
  src, dst, start, pages = _paths(case, seed)
  kv = torch.randn((case["layers"], pages, 2, case["heads"], case["page"], case["dim"]), generator=_device_rng(seed), device=DEVICE, dtype=_dtype(case))
  return {"kv": kv, "src": _ints(src), "dst": _ints(dst), "start": _ints(start), "most": case["kept"]}


def _tree_sizes(case):
  """For every request the number of its context keys and of its drafted tokens."""
  rng, sizes = random.Random(case["ragged"]), []
  for r in range(case["requests"]):
    context = rng.randint(max(1, case["context"] // 8), case["context"]) if case["ragged"] else case["context"]
    nodes = rng.randint(max(1, case["nodes"] // 2), case["nodes"]) if case["ragged"] else case["nodes"]
    sizes.append((0 if case["empty"] and r % 2 else context, nodes))      # some requests start with a tree
  return sizes


def _trees(case, seed):
  """For every request: context keys, and for each of its drafted tokens the set of the drafted tokens that it sees, as a bit mask, and its depth."""
  rng, trees = random.Random(seed), []
  for context, nodes in _tree_sizes(case):
    sees, depth = [], []
    for j in range(nodes):
      parent = rng.randint(max(0, j - 6), j - 1) if j else -1
      sees.append((sees[parent] if j else 0) | 1 << j)
      depth.append(depth[parent] + 1 if j else 0)
    if case["empty"]:      # padded places of a tree see nothing
      sees = [0 if rng.random() < 0.2 else m for m in sees]
    trees.append((context, sees, depth))
  return trees


def _prepare_tree(case, seed):
  g, rng, trees = _device_rng(seed), random.Random(seed + 1), _trees(case, seed)
  nh, nkv, hd, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
  words = -(-max(len(sees) for _, sees, _ in trees) // 32)
  lengths = [context + len(sees) for context, sees, _ in trees]
  span = max(-(-c // P) for c in lengths)
  pages = list(range(1, sum(-(-c // P) for c in lengths) + 1))
  rng.shuffle(pages)
  table, mask, positions, q_start = [[0] * span for _ in range(len(trees) + 1)], [], [], [0]
  slots = rng.sample(range(len(trees) + 1), len(trees))
  for b, (context, sees, depth) in enumerate(trees):
    for i in range(-(-lengths[b] // P)):
      table[slots[b]][i] = pages.pop()
    for m, d in zip(sees, depth):
      mask.append([((m >> 32 * w) & 0xffffffff) - ((m >> 32 * w & 0x80000000) << 1) for w in range(words)])
      positions.append(context + d)
    q_start.append(len(positions))
  T, dt = q_start[-1], _dtype(case)
  kv = torch.randn((sum(-(-c // P) for c in lengths) + 1, 2, nkv, P, hd), generator=g, device=DEVICE).to(dt)
  qkv = (torch.randn((T, (nh + 2 * nkv) * hd), generator=g, device=DEVICE) * 1.5).to(dt)
  sink = torch.randn(nh, generator=g, device=DEVICE) if case["sink"] else None
  return {"qkv": qkv, "kv": kv, "table": _ints(table), "slots": _ints(slots), "q_start": _ints(q_start[:-1]), "q_len": _ints([len(t[1]) for t in trees]),
          "ctx_len": _ints(lengths), "mask": _ints(mask), "positions": _ints(positions), "sink": sink, "tokens": T, "items": len(trees),
          "most": max(len(t[1]) for t in trees), "longest": max(lengths), "out": torch.empty((T, nh * hd), dtype=dt, device=DEVICE)}


def prepare(case, seed):
  state = {"beam": _prepare_beam, "states": _prepare_states, "pages": _prepare_pages, "rows": _prepare_rows, "tree": _prepare_tree}[case["kind"]](case, seed)
  state["case"] = case
  return state


# ------------------------------------------------------------------------------------------------ the plain forms


def _rising(x):
  """Whole numbers that rise as float32 values do."""
  bits = (x + 0.0).view(torch.int32)      # (one zero)
  return (bits ^ ((bits >> 31) & 0x7fffffff)).long()


def _plain_beam(s):
  # candidates of two beams may lie closer than 32 bits tell apart: the scores are made in 64
  case, n = s["case"], s["case"]["n"]
  x, V = s["logits"].float(), case["vocab"]
  k, most, requests = min(n, V), s["most"], case["requests"]
  wide = x.double()
  top = wide.amax(1, keepdim=True)
  total = (wide - top).exp().sum(1, keepdim=True).log()
  del wide
  places = _rising(x) << 32 | (V - 1 - torch.arange(V, device=x.device))      # equal values: the lowest index first
  tokens = V - 1 - (places.topk(k, dim=1).values & 0xffffffff)
  scores = s["cum"].double()[:, None] + (x.gather(1, tokens).double() - top - total)
  start = s["start"].long()
  rows = start[:-1, None] + torch.arange(most, device=x.device)
  there = rows < start[1:, None]
  rows = torch.where(there, rows, 0)
  scores = torch.where(there[:, :, None], scores[rows], -math.inf).view(requests, most * k)
  scores = torch.where(scores.isnan(), -math.inf, scores)
  best, order = scores.sort(dim=1, descending=True, stable=True)
  pad = max(0, n - most * k)
  best = torch.nn.functional.pad(best[:, :n], (0, pad), value=-math.inf)
  order = torch.nn.functional.pad(order[:, :n], (0, pad))
  live = best > -math.inf
  got_tokens = torch.where(live, tokens[rows].view(requests, most * k).gather(1, order), -1)
  got_parents = torch.where(live, rows.gather(1, order // k), -1)
  return got_tokens.int(), got_parents.int(), best.float()


def _plain_states(s):
  state, src, dst = s["state"], s["src"].long(), s["dst"].long()
  state[:, dst] = state[:, src]
  return state


def _plain_pages(s):
  kv, src, dst = s["kv"], s["src"].long(), s["dst"].long()
  if s["rows"] is None:
    kv[:, dst] = kv[:, src]
  else:
    filled = torch.arange(kv.shape[4], device=kv.device) < s["rows"][:, None]
    kv[:, dst] = torch.where(filled[:, None, None, :, None], kv[:, src], kv[:, dst])
  return kv


def _plain_rows(s):
  kv, src, dst = s["kv"], s["src"].long(), s["dst"].long()
  P = kv.shape[4]
  kv[:, dst // P, :, :, dst % P] = kv[:, src // P, :, :, src % P]
  return kv


def _plain_tree(s):
  case = s["case"]
  nh, nkv, hd, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
  B, most, longest, G = s["items"], s["most"], s["longest"], nh // nkv
  pages = s["table"].long()[s["slots"].long(), :-(-longest // P)]
  keys, values = (s["kv"][pages, w].transpose(1, 2).reshape(B, nkv, -1, hd)[:, :, :longest].float() for w in (0, 1))
  node = torch.arange(most, device=keys.device)
  q_start, q_len, ctx = s["q_start"].long(), s["q_len"].long(), s["ctx_len"].long()
  first = ctx - q_len
  rows = torch.where(node < q_len[:, None], q_start[:, None] + node, 0)
  q = s["qkv"][:, :nh * hd].float()[rows].view(B, most, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * most, hd)
  scores = (q @ keys.transpose(2, 3)).view(B, nkv, G, most, longest) * hd ** -0.5
  if case["softcap"]:
    scores = case["softcap"] * torch.tanh(scores / case["softcap"])
  key = torch.arange(longest, device=keys.device)
  new = key - first[:, None]      # a key's place among the drafted tokens
  inside = (new >= 0) & (new < q_len[:, None])
  place = new.clamp(0, most - 1)
  words = s["mask"][rows].long()
  bit = words.gather(2, (place // 32)[:, None].expand(B, most, longest)) >> (place % 32)[:, None] & 1
  visible = (new < 0)[:, None] | (inside[:, None] & (bit > 0))
  if case["window"]:
    positions = s["positions"].long()[rows]
    where = torch.where(inside, positions.gather(1, place), key)
    visible = visible & (where[:, None] > positions[:, :, None] - case["window"])
  scores = scores.masked_fill(~visible[:, None, None], -math.inf)
  top = scores.amax(-1, keepdim=True)
  if case["sink"]:
    top = torch.maximum(top, s["sink"].view(1, nkv, G, 1, 1))
  top = torch.where(top.isinf(), 0.0, top)
  weights = (scores - top).exp()
  total = weights.sum(-1, keepdim=True)
  if case["sink"]:
    total = total + (s["sink"].view(1, nkv, G, 1, 1) - top).exp()
  weights = weights / torch.where(total > 0, total, 1.0)
  out = weights.view(B, nkv, G * most, longest) @ values
  out = out.view(B, nh, most, hd).transpose(1, 2).reshape(B, most, nh * hd)
  return out[node < q_len[:, None]].to(_dtype(case))


# ------------------------------------------------------------------------------------------------ the framework's calls


_kept = {}


def _workspace():
  """What a program keeps for all of its calls."""
  if "workspace" not in _kept:
    from miniinfer_b200.engine.context import Workspace
    _kept["workspace"] = Workspace(DEVICE)
  return _kept["workspace"]


def _own(s):
  from miniinfer_b200.kernels import ops
  case = s["case"]
  if case["kind"] == "beam":
    tokens, parents, scores = s["out"]
    ops.beam_select(tokens, parents, scores, s["logits"], s["cum"], s["start"], _workspace())
    return tokens, parents, scores
  if case["kind"] == "states":
    ops.reorder_states(s["state"], s["src"], s["dst"])
    return s["state"]
  if case["kind"] == "pages":
    ops.copy_cache_pages(s["kv"], s["src"], s["dst"], s["rows"])
    return s["kv"]
  if case["kind"] == "rows":
    ops.move_cache_rows(s["kv"], s["src"], s["dst"], s["start"], s["most"])
    return s["kv"]
  batch = s.get("batch")
  if batch is None:      # a program makes it once a step, for all layers
    batch = s["batch"] = ops.AttentionBatch(positions=s["positions"], seq_slot=s["slots"], q_start=s["q_start"], q_len=s["q_len"], ctx_len=s["ctx_len"],
                                            num_tokens=s["tokens"], num_items=s["items"], max_ctx_len=s["longest"], max_q_len=s["most"],
                                            tree_mask=s["mask"], scratch=_workspace())
  ops.tree_attention(s["out"], s["qkv"], s["kv"], s["table"], batch, case["heads"], case["kv_heads"], case["dim"], case["dim"] ** -0.5,
                     case["window"] or None, sink=s["sink"], softcap=case["softcap"])
  return s["out"]


def run(state):
  if own:
    return _own(state)
  return {"beam": _plain_beam, "states": _plain_states, "pages": _plain_pages, "rows": _plain_rows, "tree": _plain_tree}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
  size = 2 if case["dtype"] == "bfloat16" else 4
  kind = case["kind"]
  if kind == "beam":
    rows = sum(_beam_rows(case))
    return {"bytes": rows * (case["vocab"] * size + 4) + case["requests"] * (12 * case["n"] + 4), "flops": 4 * rows * case["vocab"]}
  if kind == "states":
    pairs, beams = case["requests"] * case["beams"], case["beams"]
    read = case["requests"] * beams * (1 - (1 - 1 / beams) ** beams)      # distinct sources, on average
    return {"bytes": case["layers"] * case["row"] * size * (read + pairs), "flops": 0}
  if kind == "pages":
    row = case["layers"] * 2 * case["heads"] * case["dim"] * size
    rows, sources = ((case["page"] + 1) / 2, 1) if case["partial"] else (case["page"], case["pairs"])
    return {"bytes": row * rows * (sources + case["pairs"]), "flops": 0}
  if kind == "rows":
    return {"bytes": 2 * case["requests"] * case["kept"] * case["layers"] * 2 * case["heads"] * case["dim"] * size, "flops": 0}
  keys = tokens = products = 0
  for context, nodes in _tree_sizes(case):
    if case["window"]:
      context = min(context, case["window"])
    keys, tokens, products = keys + context + nodes, tokens + nodes, products + nodes * (context + nodes / 2)
  return {"bytes": size * case["dim"] * (2 * keys * case["kv_heads"] + 2 * tokens * case["heads"]), "flops": 4 * products * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits


def _exact_beam(case, seed):
  s = _prepare_beam(case, seed)
  first = s["start"].tolist()
  tokens, parents, scores = [], [], []
  for lo, hi in zip(first, first[1:]):
    every = s["logits"][lo:hi].double().log_softmax(1) + s["cum"][lo:hi].double()[:, None]
    flat = every.reshape(-1)
    enough = min(flat.numel(), 4 * case["n"] + 64)
    at = flat.topk(enough).indices.tolist()
    value = flat[torch.tensor(at, device=DEVICE)].tolist()
    best = sorted(zip([-v for v in value], at))[:case["n"]]
    best = [(-v, i) for v, i in best if v < math.inf]
    best += [(-math.inf, None)] * (case["n"] - len(best))
    scores.append([v for v, _ in best])
    parents.append([-1 if i is None else lo + i // case["vocab"] for _, i in best])
    tokens.append([-1 if i is None else i % case["vocab"] for _, i in best])
  return _ints(tokens), _ints(parents), torch.tensor(scores, dtype=torch.float64)


def _exact_moves(case, seed):
  """What is moved keeps its values: the same places, one pair at a time, out of a copy."""
  if case["kind"] == "states":
    s = _prepare_states(case, seed)
    old = s["state"].clone()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
      s["state"][:, b].copy_(old[:, a])
    return s["state"]
  s = _prepare_pages(case, seed) if case["kind"] == "pages" else _prepare_rows(case, seed)
  kv, old, P = s["kv"], s["kv"].clone(), case["page"]
  rows = s.get("rows")
  for k, (a, b) in enumerate(zip(s["src"].tolist(), s["dst"].tolist())):
    if case["kind"] == "rows":
      kv[:, b // P, :, :, b % P].copy_(old[:, a // P, :, :, a % P])
    else:
      filled = P if rows is None else int(rows[k])
      kv[:, b, :, :, :filled].copy_(old[:, a, :, :, :filled])
  return kv


def _exact_tree(case, seed):
  s, trees = _prepare_tree(case, seed), _trees(case, seed)
  nh, nkv, hd, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
  table, slots, q_start = s["table"].tolist(), s["slots"].tolist(), s["q_start"].tolist()
  outs = []
  for b, (context, sees, depth) in enumerate(trees):
    n, total = len(sees), context + len(sees)
    pages = _ints(table[slots[b]][:-(-total // P)], torch.int64)
    k, v = (s["kv"][pages, w].double().permute(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :total].repeat_interleave(nh // nkv, 0) for w in (0, 1))
    q = s["qkv"][q_start[b]:q_start[b] + n, :nh * hd].double().view(n, nh, hd).transpose(0, 1)
    z = torch.bmm(q, k.transpose(1, 2)) / math.sqrt(hd)
    if case["softcap"]:
      z = torch.tanh(z / case["softcap"]) * case["softcap"]
    where = list(range(context)) + [context + d for d in depth]
    allowed = torch.tensor([[1] * context + [m >> j & 1 for j in range(n)] for m in sees], dtype=torch.bool, device=DEVICE)
    if case["window"]:
      p = _ints(where, torch.int64)
      allowed &= p[context:, None] - p[None, :] < case["window"]
    z = z.masked_fill(~allowed, -math.inf)
    rest = s["sink"].double() if case["sink"] else torch.full((nh,), -math.inf, dtype=torch.float64, device=DEVICE)
    norm = torch.logaddexp(z.logsumexp(-1), rest[:, None])
    w = torch.where(norm[..., None].isinf(), 0.0, (z - norm[..., None]).exp())
    w = torch.where(allowed, w, 0.0)
    outs.append(torch.bmm(w, v).transpose(0, 1).reshape(n, nh * hd))
  return torch.cat(outs)


def exact(case, seed):
  if case["kind"] == "beam":
    return _exact_beam(case, seed)
  return _exact_tree(case, seed) if case["kind"] == "tree" else _exact_moves(case, seed)
