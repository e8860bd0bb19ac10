"""Plain statements in 64 bits, on the CPU, of the operators on rows, and how far a kernel may be from them.

A rounding to a type is off by at most half a step: eps(type) / 2 relative to the value, or half the smallest subnormal."""
import torch

HALF32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def stored(value, dtype):
  """Bound of the rounding to dtype when `value` is stored."""
  return value.abs() * HALF[dtype] + SMALLEST[dtype]


def lookup(table, ids, scale):
  table, ids = table.detach().cpu(), ids.cpu().long()
  there = (ids >= 0) & (ids < table.shape[0])
  if table.shape[0] == 0:
    return torch.zeros(*ids.shape, table.shape[1], dtype=torch.float64)
  return torch.where(there[..., None], table.double()[ids.clamp(0, table.shape[0] - 1)] * scale, 0.0)


def lookup_grad(grad, ids, num_rows, scale):
  """(gradient, bound): a sum of n terms in 32 bits is off by at most n 2^-24 times the sum of their magnitudes (n - 1 additions,
  and one product with the scale), whatever the order."""
  g, ids = grad.detach().cpu().double().reshape(-1, grad.shape[-1]), ids.cpu().long().reshape(-1)
  there = (ids >= 0) & (ids < num_rows)
  out, size, count = (torch.zeros(num_rows, g.shape[1], dtype=torch.float64) for _ in range(3))
  out.index_add_(0, ids[there], g[there])
  size.index_add_(0, ids[there], g[there].abs())
  count.index_add_(0, ids[there], torch.ones_like(g[there]))
  return out * scale, abs(scale) * count * HALF32 * size * 1.001


def unpack(codes, scales, offsets, d, group):
  """(code term, offset term) of the rows, whose sum they are."""
  codes, scales = codes.cpu(), scales.cpu().double()
  k = torch.arange(d)
  c = ((codes.long()[:, k // 2] >> (4 * (k % 2))) & 15).double()
  s = scales.repeat_interleave(group, 1)[:, :d]
  if offsets is None:
    return (c - 8.0) * s, torch.zeros_like(s)
  return c * s, offsets.cpu().double().repeat_interleave(group, 1)[:, :d]


def scores(queries, codes, scales, offsets, d, group, alpha, bias):
  """(scores, bound).  The bound: every product and every addition of a sum in 32 bits over d elements, their groups and what
  surrounds them, 2^-24 each of the sum of magnitudes; the queries' own representation, 2^-22 relative and 2^-38 of the
  query's largest element."""
  a, b = unpack(codes, scales, offsets, d, group)
  q = queries.cpu().double()
  y = alpha * (q @ (a + b).t())
  size = abs(alpha) * (q.abs() @ (a.abs() + b.abs()).t())
  most = abs(alpha) * q.abs().amax(1, keepdim=True) * (a.abs() + b.abs()).sum(1)[None]
  if bias is not None:
    y = y + bias.cpu().double()
    size = size + bias.cpu().double().abs()
  steps = d + -(-d // group) + 16
  return y, steps * HALF32 * size * 1.001 + most * 2.0 ** -38


def select(x, beams, num, normalise, finished, end):
  """(totals, parents, tokens) by sorting every candidate."""
  x = x.detach().cpu().float()
  b, k, v = x.shape
  x = torch.where(torch.isnan(x), float("-inf"), x) + 0.0
  beams = torch.zeros(b, k) if beams is None else beams.cpu()
  totals, parents, tokens = torch.full((b, num), float("-inf"), dtype=torch.float64), torch.full((b, num), -1), torch.full((b, num), -1)
  for i in range(b):
    found = []
    for j in range(k):
      if finished is not None and bool(finished[i, j]):
        t, order = beams[i, j].double()[None], torch.tensor([end])
      else:
        row = x[i, j].double()
        order = torch.sort(row, descending=True, stable=True).indices[:num]
        t = row[order]
        if normalise:
          top = row.max()
          if top == float("inf"):
            t = torch.where(t == top, -torch.log((row == top).double().sum()), float("-inf"))
          elif top > float("-inf"):
            t = (t - top) - torch.log(torch.exp(row - top).sum())   # (in this order: beside 3e38 a logarithm is lost)
        t = t + beams[i, j].double()
      found += [(float(a), j, int(c)) for a, c in zip(t, order) if a > float("-inf")]
    found.sort(key=lambda f: -f[0])  # (stable: the lower beam, then its own order)
    for n, (a, j, c) in enumerate(found[:num]):
      totals[i, n], parents[i, n], tokens[i, n] = a, j, c
  return totals, parents, tokens


def select_bound(totals):
  """The logarithm of a sum of exponentials whose terms are off by 2^-20 at most (two roundings of the argument, weighed with
  their size, the exponential's own and the additions'), and the rounding of the total."""
  return 2.0 ** -20 + totals.abs().nan_to_num(0.0, 0.0, 0.0) * HALF32
