"""The operators on rows as a decoder uses them: the tokens' vectors looked up, a state moved on, scores of the whole
vocabulary (the same table, in 4 bits), the best beams selected, their states reordered -- a whole search against a plain one."""
import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu


def _plain_search(table, weights, steps, k, end):
  """Beam search in 64 bits on the CPU over a model with one state: h = tanh(0.5 h + 0.5 table[token])."""
  table, weights = table.double().cpu(), weights.double().cpu()
  beams = [(0.0, [0], torch.zeros(table.shape[1], dtype=torch.float64), False)]
  for _ in range(steps):
    found = []
    for j, (total, tokens, h, done) in enumerate(beams):
      if done:
        found.append((total, j, end, h))
        continue
      h = torch.tanh(0.5 * h + 0.5 * table[tokens[-1]])
      lp = torch.log_softmax(weights @ h * 4.0, 0)
      for c in torch.sort(lp, descending=True, stable=True).indices[:k].tolist():
        found.append((total + float(lp[c]), j, c, h))
    found.sort(key=lambda f: -f[0])
    gap = min((found[i][0] - found[i + 1][0]) for i in range(min(k, len(found) - 1)))
    assert gap > 1e-3         # (no two candidates are so near that 16-bit states could order them)
    beams = [(t, beams[j][1] + [c], h, c == end) for t, j, c, h in found[:k]]
  return beams


def test_a_beam_search_with_one_table():
  from cuhnsw_amd import rows
  v, d, k, steps, end = 500, 64, 3, 6, 1
  g = torch.Generator().manual_seed(11)
  table = torch.randn(v, d, generator=g).cuda()
  packed = rows.pack(table)
  want = _plain_search(table, packed.unpack(), steps, k, end)

  beams = torch.tensor([[0.0] + [-float("inf")] * (k - 1)], device="cuda")
  tokens = torch.zeros(1, k, dtype=torch.int32, device="cuda")
  finished = torch.zeros(1, k, dtype=torch.bool, device="cuda")
  h, taken = torch.zeros(1, k, d, device="cuda"), torch.zeros(1, k, 1, dtype=torch.int32, device="cuda")
  for _ in range(steps):
    h = torch.where(finished[..., None], h, torch.tanh(0.5 * h + rows.lookup(table, tokens, scale=0.5)))
    scores = packed.scores(h.view(k, d), alpha=4.0).view(1, k, v)
    beams, parents, tokens = rows.select_beams(scores, beams, k, finished=finished, end=end)
    h, taken = rows.reorder_states([h, taken], parents)
    taken = torch.cat([taken, tokens[..., None]], 2)
    finished = tokens == end
  assert taken[0].tolist() == [w[1] for w in want]
  assert max(abs(float(a) - w[0]) for a, w in zip(beams[0], want)) < 1e-4


def test_training_a_table_and_searching_it():
  """Words that stand together are pulled together: the gradient of a step against the formula's, then the table is indexed."""
  from cuhnsw_amd import CuHNSW, rows
  n, d, t = 400, 32, 3000
  g = torch.Generator().manual_seed(4)
  table = torch.randn(n, d, generator=g).cuda().requires_grad_(True)
  a, b = (torch.randint(0, n, (t,), generator=g).cuda() for _ in range(2))
  loss = (rows.lookup(table, a) - rows.lookup(table, b)).square().sum()
  loss.backward()
  diff = 2 * (table.detach()[a] - table.detach()[b])
  one, bound_one = ref.lookup_grad(diff, a, n, 1.0)
  two, bound_two = ref.lookup_grad(diff, b, n, 1.0)
  # the two gradients are rounded once each and added once; `diff` was formed in 32 bits, as in the backward pass
  bound = bound_one + bound_two + (one.abs() + two.abs()) * 2.0 ** -22
  assert ((table.grad.cpu().double() - (one - two)).abs() <= bound + 1e-12).all()
  h = CuHNSW({"py_log_level": 1, "heuristic_coef": 0.0, "dist_type": "l2", "max_m": 8, "max_m0": 16})
  h.set_data((table.detach() - 0.01 * table.grad).cpu().numpy())
  h.build()
  nns, _, found = h.search_items([5, 17], 4, 50)
  assert (nns[:, 0] == [5, 17]).all() and (found == 4).all()
