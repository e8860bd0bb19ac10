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


def test_views_that_are_still_to_be_negated_or_conjugated_are_refused():
  """What is in their memory is not what they stand for."""
  torch = pytest.importorskip("torch")
  from cuhnsw_amd import rows
  late = torch.zeros(2, 4, 64, dtype=torch.complex64).conj()
  negated = late.imag
  assert negated.is_neg() and late.is_conj()
  ids, parents = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 4, dtype=torch.int32)
  flat = torch.zeros(4, dtype=torch.complex64).conj().imag
  for call in (lambda: rows.lookup(negated[0], ids), lambda: rows.lookup_grad(negated[0, :2], ids, 3), lambda: rows.pack(negated[0]),
               lambda: rows.select_beams(negated, None, 1), lambda: rows.select_beams(torch.zeros(2, 4, 64), negated[:, :, 0], 1),
               lambda: rows.reorder_states([negated], parents), lambda: rows.reorder_states([late], parents)):
    with pytest.raises(ValueError, match="still to be negated"):
      call()
  assert flat.is_neg()
  packed = object.__new__(rows.PackedRows)
  packed.num_rows, packed.num_dims = 4, 64
  for call in (lambda: packed.scores(negated[0]), lambda: packed.scores(torch.zeros(1, 64), bias=flat), lambda: packed.search_knn(negated[0], 1)):
    with pytest.raises(ValueError, match="still to be negated"):
      call()


def test_states_without_elements_are_contiguous():
  torch = pytest.importorskip("torch")
  from cuhnsw_amd import rows
  for shape in ((2, 3, 2, 0, 3), (2, 3, 0), (2, 3, 5, 0)):
    with pytest.raises(ValueError, match="on the GPU"):
      rows.reorder_states([torch.zeros(shape)], torch.zeros(2, 3, dtype=torch.int32))


def test_scratch_memory_of_a_gradient_does_not_grow_with_the_rows_more_than_it_has_to():
  """Sorted ids, sums of long stretches, counts: by the ids.  By the rows: where those of every workgroup begin, four rows or more."""
  l = capi.load()
  few, many = (l.cuhnsw_lookup_grad_workspace(5000, n, 8) for n in (1 << 20, 1 << 30))
  assert 0 < many - few <= (1 << 30) + (1 << 20)     # (the counts have more digits)
