"""Selection over beams and vocabulary and the reordering of states, on the GPU, against a sort of every candidate in 64 bits."""
import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def _check(x, beams, num, normalise=True, finished=None, end=None, near=False):
  """near: candidates of different beams may be nearer to each other than a log_softmax is exact."""
  from cuhnsw_amd import rows
  totals, parents, tokens = rows.select_beams(x, beams, num, normalise=normalise, finished=finished, end=end)
  want = ref.select(x, beams, num, normalise, finished, end)
  assert totals.shape == parents.shape == tokens.shape == (x.shape[0], num)
  if near and normalise:
    # Two totals that are each off by the bound can change places where they differ by less than twice that: what stands at a place
    # is a candidate, no other place's, whose total is that near to the place's; and one beam's own stand in their order.
    all_of = ref.select(x, beams, x.shape[1] * num, True, finished, end)   # (every beam with its best num, and more)
    for b in range(x.shape[0]):
      total_of = {(int(p), int(t)): float(v) for v, p, t in zip(*(o[b] for o in all_of)) if p >= 0}
      got = list(zip(parents[b].tolist(), tokens[b].tolist()))
      for i, pair in enumerate(got):
        if pair != (int(want[1][b, i]), int(want[2][b, i])):
          assert abs(total_of[pair] - float(want[0][b, i])) <= 2 * float(ref.select_bound(want[0][b, i]))
      assert len(set(g for g in got if g[0] >= 0)) == sum(g[0] >= 0 for g in got)
      for k in range(x.shape[1]):
        own = [t for p, t in got if p == k]
        assert own == [int(t) for p, t in zip(all_of[1][b], all_of[2][b]) if p == k][:len(own)]
  else:
    assert (parents.cpu() == want[1]).all()
    assert (tokens.cpu() == want[2]).all()
  some = torch.isfinite(want[0])
  got = totals.cpu().double()
  assert (got[~some] == want[0][~some]).all()
  assert ((got[some] - want[0][some]).abs() <= ref.select_bound(want[0][some])).all()
  if not normalise:   # sums of two float32 in 64 bits, rounded once
    assert (got == want[0].float().double()).all()
  return totals, parents, tokens


def _scores(b, k, v, dtype, seed=0, spread=2.5):
  return (torch.randn(b, k, v, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype).cuda()


def _beams(b, k, seed=3):
  return (torch.rand(b, k, generator=torch.Generator().manual_seed(seed)) * -20).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b, k, v, num", [
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 6), (1, 4, 1000, 8), (3, 4, 1001, 8), (2, 8, 32_000, 16), (5, 1, 4097, 100), (1, 2, 65_537, 4), (2, 2, 131_073, 256),
    (1, 16, 300, 256), (7, 5, 63, 10), (1, 1, 300_001, 3), (40, 8, 2000, 16), (1, 300, 40, 13)])
def test_select(b, k, v, num, dtype):
  print("select", b, k, v, num, dtype, flush=True)
  x = _scores(b, k, v, dtype)
  _check(x, _beams(b, k), num)
  _check(x, None, num, normalise=False)
  _check(x, _beams(b, k), num, normalise=False)


@pytest.mark.parametrize("v, num", [(1_183_514, 100), (1_000_003, 256), (262_144, 1)])
def test_nearest_of_a_large_table(v, num):
  x = _scores(2, 1, v, torch.float32, seed=v)
  _check(x, None, num, normalise=False)
  _check(x.half(), None, num, normalise=False)   # equal values everywhere


@pytest.mark.parametrize("v", [50, 5000, 100_000])
@pytest.mark.parametrize("law", ["equal", "two values", "rising", "falling", "steps", "spike", "zeros"])
def test_equal_scores_and_orders_that_are_hard(v, law):
  at = torch.arange(v, dtype=torch.float32)
  row = {"equal": torch.full((v,), 0.5), "two values": (at * 7 % 3 == 0).float(), "rising": at / 16, "falling": -at / 16, "steps": (at / 700).floor(),
         "spike": torch.where(at % 997 == 996, 9.0, 0.0), "zeros": torch.where(at % 2 == 0, 0.0, -0.0)}[law]
  x = torch.stack([row, row.flip(0), row]).view(1, 3, v).cuda()
  for num in (1, 40, 200):
    print("hard", law, v, num, flush=True)
    _check(x, None, num, normalise=False)
    # (the second beam holds the first one's scores in another order: its sum of exponentials is the same but for roundings, and
    # -0.5 is a whole number of the steps between scores)
    _check(x, torch.tensor([[0.0, -0.5, 0.0]]).cuda(), num, near=True)
    _check(x[:, [0, 0, 0]], torch.tensor([[0.0, -0.5, 0.0]]).cuda(), num)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [333, 32_001, 150_003])
def test_equal_beams_take_turns(v, dtype):
  """Beams that are the same, wherever their rows lie in memory: of equal candidates the lower beam's stands first."""
  x = _scores(2, 1, v, dtype, seed=v).expand(2, 5, v).contiguous()
  for num in (1, 7, 30):
    _, parents, _ = _check(x, None, num)
    assert (parents.cpu() == torch.arange(num) % 5).all() or dtype != torch.float32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [9, 3000, 70_000])
def test_masked_places(v, dtype):
  x = _scores(4, 3, v, dtype, seed=9)
  x[0, 0] = -INF                        # a beam that masks everything
  x[1] = -INF                           # a batch entry that does
  x[2, 1, :-1] = -INF                   # one token is left, the last
  x[2, 0] = float("nan")                # NaN counts as masked
  x[2, 2, 1:] = float("nan")
  x[3, :, ::2] = -INF
  beams = _beams(4, 3)
  beams[3, 1] = -INF                    # a beam that is not alive
  for num in (1, 5, 20):
    _, parents, tokens = _check(x, beams, num)
    _check(x, beams, num, normalise=False)
    assert (parents[1] == -1).all() and (tokens[1] == -1).all()
    assert not (parents[3] == 1).any()


def test_infinite_scores():
  x = _scores(2, 2, 500, torch.float32)
  x[0, 0, 17] = INF
  x[1, 1, [3, 400]] = INF
  _check(x, _beams(2, 2), 4)
  _check(x, _beams(2, 2), 4, normalise=False)
  many = _scores(1, 1, 70_000, torch.float32)
  many[0, 0, ::5000] = INF             # (in several stretches of the row)
  _check(many, _beams(1, 1), 20)
  lowest = torch.full((1, 2, 500), torch.finfo(torch.float32).min, device="cuda")    # a mask of the type's lowest value
  lowest[0, 1, 44] = 0.0
  _check(lowest, _beams(1, 2), 6)
  _check(torch.full((1, 1, 300), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device="cuda"), None, 6)


@pytest.mark.parametrize("v", [100, 40_000])
def test_finished_beams(v):
  x = _scores(6, 4, v, torch.float32)
  beams = _beams(6, 4)
  finished = torch.tensor([[0, 0, 0, 0], [1, 0, 0, 0], [0, 1, 0, 1], [1, 1, 1, 1], [0, 0, 0, 1], [1, 0, 1, 0]], dtype=torch.bool).cuda()
  beams[5, 0] = 3.0
  beams[1, 0] = -INF
  for num in (1, 4, 8):
    _, parents, tokens = _check(x, beams, num, finished=finished, end=2)
    assert (tokens[3, 4:] == -1).all() if num > 4 else True
    _check(x, beams, num, normalise=False, finished=finished, end=99)


def test_strided_scores_and_a_vocabulary_in_a_wider_row():
  base = _scores(3, 8, 1003, torch.bfloat16)
  _check(base[:, :4, 1:1001], _beams(3, 4), 6)
  _check(base[::2, 1::3, 5:600], _beams(2, 3), 6)
  _check(base[:, 3:4, 3:].expand(3, 5, 1000), _beams(3, 5), 6)
  _check(base[1:2].transpose(0, 1)[:, :, 7:], _beams(8, 1), 6)


def test_a_row_that_begins_behind_the_2_31st_element():
  x = torch.zeros(5, 1, 500_000_000, dtype=torch.float16, device="cuda")
  at = torch.tensor([499_999_999, 3, 250_000_001, 0, 77], device="cuda")
  x[torch.arange(5, device="cuda"), 0, at] = 1.0
  from cuhnsw_amd import rows
  totals, parents, tokens = rows.select_beams(x, None, 3, normalise=False)
  assert (tokens[:, 0] == at).all() and (parents == 0).all() and (totals[:, 0] == 1).all()
  for i in range(5):
    left = [t for t in range(3) if t != at[i]][:2]
    assert tokens[i, 1:].tolist() == left


def test_the_same_scores_give_the_same_answer():
  from cuhnsw_amd import rows
  x, beams = _scores(16, 4, 50_000, torch.bfloat16), _beams(16, 4)
  first = rows.select_beams(x, beams, 8)
  for _ in range(5):
    for a, b in zip(first, rows.select_beams(x, beams, 8)):
      assert torch.equal(a, b)
  # Alone a row is split over more workgroups, and its sum is rounded in other places: each answer is off by the bound at most, two
  # of them by twice that.  (The best eight are of one beam, in the order of its scores, and no other's is
  # as near as 0.6.)
  part = rows.select_beams(x[5:6], beams[5:6], 8)
  assert ((first[0][5:6] - part[0]).abs().cpu().double() <= 2 * ref.select_bound(first[0][5:6].cpu().double())).all()
  assert torch.equal(first[1][5:6], part[1]) and torch.equal(first[2][5:6], part[2])


@pytest.mark.parametrize("dtype", TYPES + [torch.int64, torch.uint8, torch.bool, torch.float64])
def test_reorder(dtype):
  from cuhnsw_amd import rows
  b, k = 3, 5
  parents = torch.tensor([[0, 0, 4, 2], [-1, 1, 5, 3], [4, 3, 2, 1]], dtype=torch.int32).cuda()
  shapes = [(), (1,), (7,), (3, 11), (64,), (2, 129, 8), (4096,), (0,)]
  states = [(torch.randn(b, k, *s) * 50).to(dtype).cuda() for s in shapes]
  wide = (torch.randn(b, k + 2, 48) * 50).to(dtype).cuda()
  states.append(wide[:, 1:-1, 3:40])                      # strided, at an odd address
  states.append((torch.randn(k, b, 33) * 50).to(dtype).cuda().transpose(0, 1))
  for p in (parents, parents[:, ::2], parents.t().contiguous().t()):
    outs = rows.reorder_states(states, p)
    for x, out in zip(states, outs):
      assert out.shape == (b, p.shape[1], *x.shape[2:]) and out.dtype == dtype
      for i in range(b):
        for j in range(p.shape[1]):
          parent = int(p[i, j])
          assert torch.equal(out[i, j], x[i, parent] if 0 <= parent < k else torch.zeros_like(out[i, j]))
  assert rows.reorder_states([], parents) == []


def test_reorder_of_many_and_of_large_states():
  from cuhnsw_amd import rows
  parents = torch.tensor([[1, 1], [0, 1]], dtype=torch.int32).cuda()
  states = [torch.randn(2, 2, 3 + i, device="cuda") for i in range(70)] + [torch.randn(2, 2, 1_000_003, device="cuda").half()]
  for x, out in zip(states, rows.reorder_states(states, parents)):
    assert torch.equal(out[0, 0], x[0, 1]) and torch.equal(out[0, 1], x[0, 1]) and torch.equal(out[1], x[1])


def test_selection_and_reordering_in_a_graph():
  from cuhnsw_amd import rows
  x, beams, state = _scores(4, 4, 20_000, torch.bfloat16), _beams(4, 4), torch.randn(4, 4, 300, device="cuda")

  def step():
    out = rows.select_beams(x, beams, 8)
    return list(out) + rows.reorder_states([state], out[1][:, :4])

  step()
  torch.cuda.synchronize()
  graphs = []
  for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      out = step()
    graphs.append((graph, out))
  for _ in range(4):
    x.normal_()
    beams.uniform_(-5, 0)
    state.normal_()
    for graph, _ in graphs:
      graph.replay()
    want = step()
    torch.cuda.synchronize()
    for _, out in graphs:
      for a, b in zip(out, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("b, k, v, num", [(1, 16, 5000, 256), (2, 4, 70_000, 256), (1, 1, 400_000, 256), (3, 64, 3000, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_lists_full_of_good_candidates(b, k, v, num, dtype):
  """All lists are as good as each other, so that most of what is in them reaches a first guess of the bar."""
  _check(_scores(b, k, v, dtype), None, num, normalise=False)


def test_more_equal_totals_than_are_held():
  x = torch.zeros(2, 64, 1000).cuda()      # 4096 candidates of each batch entry, all with the same total
  _check(x, None, 64, normalise=False)
  x[1, 40, 7] = 1.0
  x[1, 50:, ::3] = -1.0
  _check(x, torch.zeros(2, 64).cuda(), 64, normalise=False)


def test_more_batch_entries_than_a_launch_holds():
  from cuhnsw_amd import rows
  b = (1 << 22) + 4321
  x = torch.randint(-4, 4, (b, 1, 3), generator=torch.Generator().manual_seed(8)).float().cuda()
  totals, parents, tokens = rows.select_beams(x, None, 2, normalise=False)
  want = torch.sort(x[:, 0], dim=1, descending=True, stable=True)
  assert torch.equal(totals, want.values[:, :2]) and torch.equal(tokens.long(), want.indices[:, :2]) and not parents.any()
