"""Which kernel a product with rows in 4 bits goes to, asked without a GPU: the sizes that the tests on the GPU rely on."""
import ctypes

import pytest

from cuhnsw_amd import capi


def _plan(*sizes):
  out = (ctypes.c_int * 4)()
  assert capi.load().cuhnsw_packed_scores_plan(*sizes, out) == 0
  return tuple(out)


@pytest.mark.parametrize("query_type", [0, 1, 2])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_sizes_that_the_kernels_are_tested_at_reach_them(group, query_type):
  for d in (20, 33, 64, 96, 101, 130, 200, 300, 960, 1024):
    for n, nq, tiles in ((24_577, 17, 2), (16_385, 33, 3), (12_801, 64, 4)):
      assert _plan(n, d, group, query_type, nq)[0] == tiles
      assert _plan(n, d, group, query_type, 1)[0] == _plan(n, d, group, query_type, 16)[0] == 0
  for n, nq, plan in ((100_001, 97, (4, 2)), (40_001, 250, (4, 2)), (50_001, 400, (4, 7)), (2000, 3000, (4, 3))):
    assert _plan(n, 96, group, query_type, nq)[:2] == plan


def test_products_of_bad_sizes_have_no_plan():
  out = (ctypes.c_int * 4)()
  for sizes in ((0, 8, 32, 0, 1), (5, 0, 32, 0, 1), (5, 8, 0, 0, 1), (5, 8, 32, 3, 1), (5, 8, 32, 0, 0)):
    assert capi.load().cuhnsw_packed_scores_plan(*sizes, out) == -1
  assert capi.load().cuhnsw_packed_scores_plan(5, 8, 32, 0, 1, None) == -1


def test_a_lookup_drops_no_tangent():
  """A table of forward-mode differentiation does not require a gradient: its tangent would be lost without a word."""
  torch = pytest.importorskip("torch")
  from torch.autograd import forward_ad

  from cuhnsw_amd import rows
  ids = torch.zeros(1, dtype=torch.int64)
  with forward_ad.dual_level():
    for table in (torch.zeros(4, 3), torch.zeros(4, 3, requires_grad=True)):
      with pytest.raises(ValueError, match="forward-mode"):
        rows.lookup(forward_ad.make_dual(table, torch.ones(4, 3)), ids)
    with pytest.raises(ValueError, match="on the GPU"):    # (one without a tangent is not refused for it)
      rows.lookup(torch.zeros(4, 3), ids)
  with pytest.raises(ValueError, match="forward-mode"):
    torch.func.jvp(lambda x: rows.lookup(x, ids), (torch.zeros(4, 3),), (torch.ones(4, 3),))
