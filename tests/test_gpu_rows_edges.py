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
