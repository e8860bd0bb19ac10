"""The operators on tables of learned vectors, as cases that can be timed: rows looked up by id and the gradient of
that (`rows.lookup`), products of queries with rows held in 4 bits (`rows.PackedRows.scores`), and the selection of the
best candidates over beams and vocabulary with the reordering of the beams' states (`rows.select_beams`,
`rows.reorder_states`).

With `own` set the calls are the framework's; without, the same operators in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZE = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "int64": 8}
_END = 2  # the token that ends a sequence


def listed():
  return [
      # the words of one query, fetched from the headline configuration's table: latency
      dict(name="lookup_words", kind="lookup", n=1_183_514, d=50, t=8, dtype="float32", ids="int64", scale=1.0, law="uniform"),
      # a large request of long descriptors from a table in half precision, an odd number of them
      dict(name="lookup_gist", kind="lookup", n=400_000, d=960, t=50_003, dtype="float16", ids="int32", scale=0.5, law="uniform"),
      # a training step on the small angular table: a thousand words of a skewed vocabulary
      dict(name="train_words", kind="train", n=100_000, d=50, t=1000, dtype="float32", ids="int64", scale=1.0, law="skewed"),
      # a training step of a token table in bfloat16, with padded places (id -1) and tokens that come thousands of times
      dict(name="train_tokens", kind="train", n=131_072, d=1024, t=65_536, dtype="bfloat16", ids="int64", scale=32.0, law="padded"),
      # one query against the small angular table: latency
      dict(name="scores_one", kind="scores", n=100_000, d=50, nq=1, dtype="float32", group=32, offsets=False, bias=False),
      # one token's state against a wide matrix, as a decoder does it for every token
      dict(name="scores_token", kind="scores", n=16_384, d=4096, nq=1, dtype="bfloat16", group=128, offsets=False, bias=False),
      # an odd handful of queries against long non-negative rows, ordered by squared distance
      dict(name="scores_gist", kind="scores", n=200_003, d=960, nq=33, dtype="float32", group=32, offsets=True, bias=True),
      # a batch of queries against integer descriptors
      dict(name="scores_sift", kind="scores", n=500_000, d=128, nq=256, dtype="float16", group=64, offsets=True, bias=True),
      # a whole batch of states against a vocabulary: bound by arithmetic
      dict(name="scores_batch", kind="scores", n=131_072, d=1024, nq=1024, dtype="bfloat16", group=64, offsets=False, bias=False),
      # one sequence with four beams: latency
      dict(name="beams_one", kind="select", b=1, k=4, v=32_000, num=8, dtype="float32", normalise=True, layers=2, state=2048),
      # a batch of sequences, eight beams each, over a large vocabulary, with their states
      dict(name="beams_batch", kind="select", b=32, k=8, v=131_072, num=16, dtype="bfloat16", normalise=True, layers=4, state=65_536),
      # the hundred nearest of the headline table for a hundred queries, their scores being there
      dict(name="nearest_100", kind="select", b=100, k=1, v=1_183_514, num=100, dtype="float32", normalise=False, layers=0, state=0),
  ]


def _log_int(rng, low, high):
  return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
  kind = rng.choice(["lookup", "train", "scores", "scores", "select", "select"])
  c = dict(kind=kind, dtype=rng.choice(["float32", "bfloat16", "float16"]))
  if kind in ("lookup", "train"):
    c["d"] = _log_int(rng, 24, 1024)
    c["n"] = _log_int(rng, 1000, min(1_183_514, 131_072 * 1024 // c["d"]))
    c["t"] = _log_int(rng, 1, min(100_000, (50_000 if kind == "lookup" else 65_536) * 960 // c["d"]))
    c["ids"] = rng.choice(["int32", "int64"])
    c["scale"] = rng.choice([1.0, 0.5, math.sqrt(c["d"])])
    c["law"] = rng.choice(["uniform", "skewed", "padded"])
  elif kind == "scores":
    c["d"] = _log_int(rng, 24, 4096)
    c["n"] = _log_int(rng, 1000, min(1_183_514, 190_000_000 // c["d"]))
    c["nq"] = _log_int(rng, 1, max(1, min(1024, 131_072 * 1024 // c["n"], 131_072 * 1024 * 1024 // (c["n"] * c["d"]))))
    c["group"] = rng.choice([32, 64, 128])
    c["offsets"] = rng.random() < 0.5
    c["bias"] = c["offsets"] and rng.random() < 0.7
  else:
    c["normalise"] = rng.random() < 0.7
    c["k"] = rng.randint(1, 8) if c["normalise"] else 1
    c["v"] = _log_int(rng, 1000, 1_183_514)
    c["b"] = _log_int(rng, 1, max(1, min(100, 33_000_000 // (c["k"] * c["v"]))))
    c["num"] = rng.randint(1, 2 * c["k"]) if c["normalise"] else _log_int(rng, 1, 100)
    c["layers"] = rng.randint(0, 4) if c["normalise"] else 0
    c["state"] = _log_int(rng, 16, min(262_144, 32 * 8 * 65_536 // (c["b"] * c["k"]))) if c["layers"] else 0
  return c


def _ids(c, g):
  n, t = c["n"], c["t"]
  if c["law"] == "uniform":
    ids = torch.randint(0, n, (t,), generator=g, device="cuda")
  else:  # the r-th most frequent row about 1 / r as often as the first, the frequent ones anywhere in the table
    rank = torch.exp(torch.rand(t, generator=g, device="cuda", dtype=torch.float64) * math.log(n)).long().clamp_(1, n) - 1
    ids = torch.randperm(n, generator=g, device="cuda")[rank]
  if c["law"] == "padded":  # sequences of different lengths in one batch
    ids[torch.rand(t, generator=g, device="cuda") < 0.1] = -1
  return ids.to(torch.int32 if c["ids"] == "int32" else torch.int64)


def _vectors(c, g):
  """Rows and queries of the kinds that are searched: centred where there are no offsets, else not negative."""
  n, d, nq = c["n"], c["d"], c["nq"]
  if not c["offsets"]:
    return torch.randn(n, d, generator=g, device="cuda"), torch.randn(nq, d, generator=g, device="cuda")
  x = torch.rand(d, generator=g, device="cuda") + 0.2 * torch.randn(n + nq, d, generator=g, device="cuda")
  x.clamp_(0.0, 1.7)
  return x[:n], x[n:]


def _quantised(rows, group, offsets):
  """codes [n, 16 * ceil(d / 32)] (element 2 i in the low half of byte i), scales and offsets [n, ceil(d / group)]."""
  n, d = rows.shape
  groups, width = -(-d // group), 32 * -(-d // 32)
  padded = torch.nn.functional.pad(rows, (0, groups * group - d)).view(n, groups, group)
  if offsets:  # (a short last group's padding counts among its values: the rows are not negative)
    low, high = padded.amin(2, keepdim=True), padded.amax(2, keepdim=True)
    scale, offset = ((high - low) / 15).clamp_min(1e-4).half(), low.half()
    codes = ((padded - offset.float()) / scale.float()).round_().clamp_(0, 15)
  else:
    scale, offset = (padded.abs().amax(2, keepdim=True) / 7).clamp_min(1e-4).half(), None
    codes = (padded / scale.float()).round_().clamp_(-8, 7) + 8
  codes = torch.nn.functional.pad(codes.view(n, -1)[:, :d].to(torch.uint8), (0, width - d))
  packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
  return packed.contiguous(), scale.squeeze(2).contiguous(), None if offset is None else offset.squeeze(2).contiguous()


def prepare(case, seed):
  c = dict(case)
  g = torch.Generator(device="cuda")
  g.manual_seed(1_000_003 * int(seed) + 29)
  kind, dtype = c["kind"], _TYPES[c["dtype"]]
  s = dict(case=c)
  if kind in ("lookup", "train"):
    s["table"] = torch.empty(c["n"], c["d"], dtype=dtype, device="cuda").normal_(generator=g)
    s["ids"] = _ids(c, g)
    if kind == "train":
      s["table"].requires_grad_(True)
      s["grad"] = torch.empty(c["t"], c["d"], dtype=dtype, device="cuda").normal_(0.0, 0.01, generator=g)
  elif kind == "scores":
    rows, queries = _vectors(c, g)
    s["codes"], s["scales"], s["offsets"] = _quantised(rows, c["group"], c["offsets"])
    s["queries"] = queries.to(dtype)
    s["alpha"] = 2.0 if c["bias"] else 1.0  # 2 <q, w> - |w|^2: the nearest by squared distance is the largest
    s["bias"] = -(rows * rows).sum(1) if c["bias"] else None
    if own:
      from cuhnsw_amd import rows as own_rows
      s["packed"] = own_rows.PackedRows(s["codes"], s["scales"], s["offsets"], num_dims=c["d"], group=c["group"])
  else:
    b, k, v = c["b"], c["k"], c["v"]
    x = torch.randn(b, k, v, generator=g, device="cuda") * (2.5 if c["normalise"] else 0.2)
    if c["normalise"]:  # banned tokens, sequences that ended, what the beams have gathered so far
      x[:, :, torch.rand(v, generator=g, device="cuda") < 0.01] = -math.inf
      s["finished"] = torch.rand(b, k, generator=g, device="cuda") < 0.1
      s["beams"] = -30.0 * torch.rand(b, k, generator=g, device="cuda")
    s["logits"] = x.to(dtype)
    s["states"] = [torch.empty(b, k, c["state"], dtype=dtype, device="cuda").normal_(generator=g) for _ in range(c["layers"])]
  return s


def _lookup(table, ids, scale):
  there = ((ids >= 0) & (ids < table.shape[0]))[:, None]
  rows = table.detach()[ids.clamp(0, table.shape[0] - 1).long()].float()
  return torch.where(there, rows * scale, 0.0).to(table.dtype)


def _lookup_grad(grad, ids, n, scale):
  there = (ids >= 0) & (ids < n)
  g = torch.where(there[:, None], grad.float() * scale, 0.0)
  out = torch.zeros(n, grad.shape[1], device=grad.device)
  return out.index_add_(0, ids.clamp(0, n - 1).long(), g).to(grad.dtype)


def _scores(queries, codes, scales, offsets, d, group, alpha, bias):
  n = codes.shape[0]
  values = torch.stack((codes & 15, codes >> 4), dim=2).view(n, -1)[:, :d].float()
  column = torch.arange(d, device=codes.device) // group
  if offsets is None:
    w = (values - 8.0) * scales.float()[:, column]
  else:
    w = values * scales.float()[:, column] + offsets.float()[:, column]
  y = alpha * (queries.float() @ w.t())
  return (y if bias is None else y + bias).to(queries.dtype)


def _select(logits, beams, num, normalise, finished):
  b, k, v = logits.shape
  x = logits.float() + 0.0
  x = torch.where(torch.isnan(x), -math.inf, x)
  bits = x.view(torch.int32)
  order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()  # ordered as the values are
  m = min(num, v)
  key = (order << 32) | (v - 1 - torch.arange(v, device=x.device))
  token = v - 1 - (key.topk(m, dim=2).values & 0xFFFFFFFF)
  total = x.gather(2, token).double()
  if normalise:  # (in 64 bits: candidates of different beams stand next to each other)
    top = x.amax(2, keepdim=True).double()
    total = total - (top + torch.exp(x.double() - top).sum(2, keepdim=True).log())
  total = torch.where(torch.isnan(total), -math.inf, total)
  if beams is not None:
    total = total + beams.double()[:, :, None]
  if finished is not None:
    first = torch.arange(m, device=x.device) == 0
    ended = torch.where(first, beams.double()[:, :, None], -math.inf)
    total = torch.where(finished[:, :, None], ended, total)
    token = torch.where(finished[:, :, None], _END, token)
  total, at = total.view(b, k * m).sort(dim=1, descending=True, stable=True)
  total, at = total[:, :num], at[:, :num]
  some = total > -math.inf
  parent = torch.where(some, at // m, -1).int()
  token = torch.where(some, token.view(b, k * m).gather(1, at), -1).int()
  return total.float(), parent, token


def _reorder(state, parents):
  there = (parents >= 0)[:, :, None]
  picked = state[torch.arange(state.shape[0], device=state.device)[:, None], parents.clamp_min(0).long()]
  return torch.where(there, picked, torch.zeros_like(picked))


def run(s):
  c = s["case"]
  if own:
    from cuhnsw_amd import rows
  if c["kind"] == "lookup":
    return rows.lookup(s["table"], s["ids"], scale=c["scale"]) if own else _lookup(s["table"], s["ids"], c["scale"])
  if c["kind"] == "train":
    if own:
      out = rows.lookup(s["table"], s["ids"], scale=c["scale"])
      return out, torch.autograd.grad(out, s["table"], s["grad"])[0]
    return _lookup(s["table"], s["ids"], c["scale"]), _lookup_grad(s["grad"], s["ids"], c["n"], c["scale"])
  if c["kind"] == "scores":
    if own:
      return s["packed"].scores(s["queries"], alpha=s["alpha"], bias=s["bias"])
    return _scores(s["queries"], s["codes"], s["scales"], s["offsets"], c["d"], c["group"], s["alpha"], s["bias"])
  beams, finished = s.get("beams"), s.get("finished")
  if own:
    total, parents, tokens = rows.select_beams(s["logits"], beams, c["num"], normalise=c["normalise"], finished=finished, end=_END)
    states = rows.reorder_states(s["states"], parents[:, :c["k"]]) if s["states"] else []
  else:
    total, parents, tokens = _select(s["logits"], beams, c["num"], c["normalise"], finished)
    states = [_reorder(x, parents[:, :c["k"]]) for x in s["states"]]
  return [total, parents, tokens] + list(states)


def _distinct(c):
  """Rows that t lookups meet, about."""
  n, t = c["n"], c["t"]
  if c["law"] == "uniform":
    return n * -math.expm1(t * math.log1p(-1.0 / n))
  r = np.arange(1, n, dtype=np.float64)
  return float(-np.expm1(t * (0.9 if c["law"] == "padded" else 1.0) * np.log1p(-np.minimum(np.log1p(1.0 / r) / math.log(n), 0.999))).sum())


def work(case):
  c = case
  size = _SIZE[c["dtype"]]
  if c["kind"] in ("lookup", "train"):
    row = c["d"] * size
    moved = c["t"] * (_SIZE[c["ids"]] + row) + _distinct(c) * row
    flops = c["t"] * c["d"]
    if c["kind"] == "train":
      moved += c["t"] * row + c["n"] * row
      flops *= 3
    return {"bytes": moved, "flops": flops}
  if c["kind"] == "scores":
    n, d, nq = c["n"], c["d"], c["nq"]
    held = n * (-(-d // 2) + 2 * -(-d // c["group"]) * (2 if c["offsets"] else 1) + (4 if c["bias"] else 0))
    return {"bytes": held + nq * d * size + nq * n * size, "flops": 2 * n * d * nq}
  values = c["b"] * c["k"] * c["v"]
  kept = min(c["k"], c["num"])
  return {"bytes": values * size + c["b"] * c["num"] * 12 + c["layers"] * c["state"] * size * c["b"] * (c["k"] + kept),
          "flops": values * (4 if c["normalise"] else 1)}


def exact(case, seed):
  s = prepare(case, seed)
  c = s["case"]
  if c["kind"] in ("lookup", "train"):
    n, d = c["n"], c["d"]
    t = torch.nn.functional.pad(s["table"].detach().double(), (0, 0, 0, 1))  # row n: what an id outside the table gives
    at = s["ids"].long()
    at = torch.where((at < 0) | (at >= n), n, at)
    out = t.index_select(0, at) * c["scale"]
    if c["kind"] == "lookup":
      return out
    del t
    order = torch.argsort(at, stable=True)
    ends = torch.searchsorted(at[order], torch.arange(n, device="cuda"), right=True)
    sums = torch.nn.functional.pad(s["grad"].double()[order].cumsum(0), (0, 0, 1, 0))
    starts = torch.nn.functional.pad(ends, (1, 0))[:-1]
    return out, (sums[ends] - sums[starts]) * c["scale"]
  if c["kind"] == "scores":
    n, d, q = c["n"], c["d"], s["queries"].double()
    y = torch.empty(c["nq"], n, dtype=torch.float64, device="cuda")
    k = torch.arange(d, device="cuda")
    for low in range(0, n, 65_536):
      high = min(n, low + 65_536)
      w = (s["codes"][low:high].long()[:, k // 2] >> (4 * (k % 2))) & 15
      w = w.double() - (8.0 if s["offsets"] is None else 0.0)
      w *= s["scales"][low:high].double().repeat_interleave(c["group"], 1)[:, :d]
      if s["offsets"] is not None:
        w += s["offsets"][low:high].double().repeat_interleave(c["group"], 1)[:, :d]
      y[:, low:high] = s["alpha"] * (q @ w.t())
    return y if s["bias"] is None else y + s["bias"].double()
  x = s["logits"].double()
  if c["normalise"]:
    x = torch.log(torch.softmax(x, 2)) + s["beams"].double()[:, :, None]
    x = torch.where(s["finished"][:, :, None], -math.inf, x)
    x[:, :, _END] = torch.where(s["finished"], s["beams"].double(), x[:, :, _END])
  total = x.flatten(1).topk(c["num"], dim=1).values
  return [total, None, None] + [None] * c["layers"]
