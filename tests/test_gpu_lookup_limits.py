"""The gradient of a lookup at its limits, where one launch has not threads enough: 2^31 - 2 rows, 2^30 ids."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1000, 5000])   # (picked out of all ids, and sorted)
def test_gradient_of_as_many_rows_as_there_may_be(t):
  from cuhnsw_amd import rows
  n = (1 << 31) - 2      # 2^24 workgroups of 128 rows: one more than a launch takes
  print("rows", n, "ids", t, flush=True)
  g = torch.Generator(device="cuda").manual_seed(t)
  ids = torch.randint(0, n, (t,), generator=g, device="cuda")
  ids[:6] = torch.tensor([0, n - 1, n, -1, n - 127, n - 1], device="cuda")
  grad = torch.randint(1, 9, (t, 1), generator=g, device="cuda").half()    # (sums of a few small whole numbers are exact)
  got = rows.lookup_grad(grad, ids, n).view(-1)
  there = (ids >= 0) & (ids < n)
  at, place = ids[there].unique(return_inverse=True)
  want = torch.zeros(at.shape[0], dtype=torch.float64, device="cuda").index_add_(0, place, grad[there, 0].double())
  assert torch.equal(got[at].double(), want)
  got[at] = 0
  for part in got.view(torch.int32).split(1 << 28):
    assert not part.any()


def test_gradient_of_as_many_ids_as_there_may_be():
  from cuhnsw_amd import rows
  t, n = 1 << 30, 70_001
  print("ids", t, flush=True)
  g = torch.Generator(device="cuda").manual_seed(1)
  ids = torch.randint(-1, n, (t,), generator=g, device="cuda", dtype=torch.int32)   # about 15 000 places a row, 240 stretches of 64
  grad = torch.randint(0, 8, (t,), generator=g, device="cuda", dtype=torch.int8).float().view(t, 1)  # (sums below 2^24 are exact)
  want = torch.zeros(n + 1, dtype=torch.float64, device="cuda")
  for i, x in zip(ids.split(1 << 26), grad.split(1 << 26)):
    want.index_add_(0, i.long() + 1, x[:, 0].double())
  assert float(want.max()) < 1 << 24
  got = rows.lookup_grad(grad, ids, n)
  assert torch.equal(got[:, 0].double(), want[1:])
  ones = rows.lookup_grad(torch.ones(1, 1, device="cuda").expand(t, 1), ids, n)
  count = torch.zeros(n + 1, dtype=torch.float64, device="cuda")
  for i in ids.split(1 << 26):
    count.index_add_(0, i.long() + 1, torch.ones(1, dtype=torch.float64, device="cuda").expand(i.shape[0]))
  assert torch.equal(ones[:, 0].double(), count[1:])
