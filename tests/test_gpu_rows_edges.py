"""Calls of the operators on rows that are allowed and rare, on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_states_without_elements_beside_others():
  from cuhnsw_amd import rows
  parents = torch.tensor([[1, 1, 0], [2, -1, 0]], dtype=torch.int32, device="cuda")
  full = torch.randn(2, 3, 7, device="cuda")
  empty, hollow, moved = rows.reorder_states([torch.zeros(2, 3, 0, device="cuda"), torch.zeros(2, 3, 2, 0, 3, device="cuda"), full], parents)
  assert empty.shape == (2, 3, 0) and hollow.shape == (2, 3, 2, 0, 3)
  for b in range(2):
    for j in range(3):
      p = int(parents[b, j])
      assert torch.equal(moved[b, j], full[b, p] if p >= 0 else torch.zeros(7, device="cuda"))


@pytest.mark.parametrize("dist_type", ["dot", "l2"])
def test_search_of_more_queries_than_one_product_takes(dist_type):
  from cuhnsw_amd import rows
  nq = 0xfffff0 + 17
  packed = rows.pack(torch.tensor([[7.0], [-7.0], [0.0]], device="cuda"))     # (exact: the scale is one, a row of zeros stays one)
  q = (torch.arange(nq, device="cuda") % 15 - 7).float()[:, None]
  with pytest.raises(RuntimeError, match="too many queries"):
    packed.scores(q)
  ids, dist, found = packed.search_knn(q, 2, dist_type)
  rows_there = torch.tensor([7.0, -7.0, 0.0], device="cuda")
  kinds = torch.arange(-7, 8, device="cuda").float()[:, None]
  key = -(kinds * rows_there) if dist_type == "dot" else (kinds - rows_there) ** 2
  order = key.sort(dim=1, stable=True)
  at = torch.arange(nq, device="cuda") % 15
  assert torch.equal(ids.long(), order.indices[at, :2]) and torch.equal(dist, order.values[at, :2]) and (found == 2).all()
