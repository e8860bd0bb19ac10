"""Rows in 4 bits and products with them, on the GPU, against plain statements in 64 bits."""
import numpy as np
import pytest
import torch

import rows_reference as ref
from helpers import gauss_mixture, integer_vectors

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _codes(n, d, group, offsets, scale_type=torch.float16, seed=0):
  """Random codes, all sixteen of them, with scales and offsets of mixed sizes; the places behind the last element hold anything."""
  g = torch.Generator().manual_seed(seed)
  width, groups = 16 * -(-d // 32), -(-d // group)
  codes = torch.randint(0, 256, (n, width), generator=g, dtype=torch.int64).to(torch.uint8)
  scales = (torch.rand(n, groups, generator=g) * 0.1 + 0.001).to(scale_type)
  lows = (torch.randn(n, groups, generator=g) * 0.3).to(scale_type) if offsets else None
  return codes.cuda(), scales.cuda(), None if lows is None else lows.cuda()


def _check(packed, q, alpha=1.0, bias=None, dtype=None):
  got = packed.scores(q, alpha=alpha, bias=bias, dtype=dtype)
  want, bound = ref.scores(q, packed.codes, packed.scales, packed.offsets, packed.num_dims, packed.group, float(np.float32(alpha)), bias)
  assert got.shape == want.shape and got.dtype == (dtype or q.dtype)
  off = (got.cpu().double() - want).abs()
  assert (off <= bound + ref.stored(want.abs() + bound, got.dtype)).all(), float((off - bound).max())
  return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("n, d, nq", [
    (1, 1, 1), (15, 32, 1), (17, 33, 2), (100, 50, 1), (1000, 50, 17), (333, 96, 5), (64, 128, 16), (129, 101, 33), (50, 129, 3), (2051, 960, 4),
    (70, 4096, 1), (300, 1024, 65), (513, 200, 130)])
def test_scores(n, d, nq, group, offsets, dtype):
  from cuhnsw_amd import rows
  print("scores", n, d, nq, group, offsets, dtype, flush=True)
  packed = rows.PackedRows(*_codes(n, d, group, offsets), num_dims=d, group=group)
  q = torch.randn(nq, d, generator=torch.Generator().manual_seed(nq)).to(dtype).cuda()
  bias = torch.randn(n, generator=torch.Generator().manual_seed(5)).cuda()
  _check(packed, q)
  _check(packed, q, alpha=-1.75, bias=bias)
  _check(packed, q, bias=bias, dtype=torch.float32)


@pytest.mark.parametrize("n, d, nq", [(7, 64, 257), (3000, 64, 300), (100_003, 50, 1), (100_003, 50, 3), (40_000, 960, 1), (5000, 2048, 70)])
def test_scores_of_larger_sizes(n, d, nq):
  from cuhnsw_amd import rows
  print("scores", n, d, nq, flush=True)
  for offsets, group, dtype in ((False, 32, torch.float32), (True, 64, torch.bfloat16), (False, 128, torch.float16)):
    packed = rows.PackedRows(*_codes(n, d, group, offsets), num_dims=d, group=group)
    _check(packed, torch.randn(nq, d, generator=torch.Generator().manual_seed(nq)).to(dtype).cuda())


@pytest.mark.parametrize("nq", [1, 20, 90])
def test_scores_with_bfloat16_scales_and_strided_queries(nq):
  from cuhnsw_amd import rows
  codes, scales, lows = _codes(200, 70, 32, True, torch.bfloat16)
  packed = rows.PackedRows(codes, scales * 1e6, lows * 1e6, num_dims=70, group=32)
  base = torch.randn(nq, 163, device="cuda")
  _check(packed, base[:, 5:75])
  assert torch.equal(packed.scores(base[0, 5:75]), packed.scores(base[:1, 5:75])[0])
  assert packed.scores(torch.empty(0, 70, device="cuda")).shape == (0, 200)
  _check(packed, torch.randn(1, 70, device="cuda").expand(nq, 70))


@pytest.mark.parametrize("nq", [1, 18, 70])
@pytest.mark.parametrize("dtype", TYPES)
def test_queries_that_are_tiny_large_zero_or_not_finite(nq, dtype):
  from cuhnsw_amd import rows
  packed = rows.PackedRows(*_codes(100, 130, 64, True), num_dims=130, group=64)
  q = torch.randn(nq, 130, generator=torch.Generator().manual_seed(2)).cuda()
  sizes = (1.0, 1e-3, 1e3, 0.0) if dtype == torch.float16 else (1e-37, 1e-30, 1e30, 1.0, 0.0)
  for i in range(nq):
    q[i] *= sizes[i % len(sizes)]
  q = q.to(dtype)
  _check(packed, q, dtype=torch.float32)
  clean = packed.scores(q)
  for value in (float("inf"), float("nan"), -float("inf")):
    spoilt = q.clone()
    spoilt[nq // 2, 57] = value
    got = packed.scores(spoilt)
    assert not torch.isfinite(got[nq // 2]).any()
    others = torch.arange(nq) != nq // 2
    assert torch.equal(got[others.cuda()], clean[others.cuda()])


def test_elements_of_very_different_sizes():
  """One element a million times the others, where the row's own element is zero: the others' sum is still there."""
  from cuhnsw_amd import rows
  codes, scales, _ = _codes(64, 256, 32, False)
  codes[:, 20] = 0x88                                # elements 40 and 41 are zero
  packed = rows.PackedRows(codes, scales, num_dims=256, group=32)
  for nq in (1, 33):
    q = torch.randn(nq, 256, generator=torch.Generator().manual_seed(3)).cuda()
    q[:, 40] = 1e6
    _check(packed, q)
    _check(packed, q.bfloat16(), dtype=torch.float32)


def test_scores_are_written_where_they_belong_and_nowhere_else():
  from cuhnsw_amd import cuhnsw_bind, rows
  n, d, nq = 77, 50, 19
  packed = rows.PackedRows(*_codes(n, d, 32, False), num_dims=d, group=32)
  q = torch.randn(nq, d, device="cuda")
  want = packed.scores(q)
  out = torch.full((nq + 2, 100), 7.0, device="cuda")
  size = cuhnsw_bind.packed_scores_workspace(n, d, 32, 0, nq)
  work = torch.empty(size + 1, dtype=torch.uint8, device="cuda")
  cuhnsw_bind.packed_scores(packed.codes.data_ptr(), packed.scales.data_ptr(), 0, 1, n, d, 32, q.data_ptr(), 0, d, nq, 1.0, 0,
                            out[1].data_ptr(), 0, 100, work.data_ptr(), size, 0, torch.cuda.current_stream().cuda_stream)
  assert torch.equal(out[1:-1, :n], want)
  assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[1:-1, n:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("n, d, group", [(1, 1, 32), (100, 50, 32), (33, 101, 64), (500, 128, 128), (65, 130, 128), (1000, 960, 64)])
def test_pack(n, d, group, offsets, dtype):
  """Every element is within half a step of what was packed; the step is the scale, which is rounded, and the extremes of a
  group may fall outside the sixteen values by what the scale and the offset were rounded by (2^-11 relative)."""
  from cuhnsw_amd import rows
  x = (torch.randn(n, d, generator=torch.Generator().manual_seed(d)) * 3).to(dtype)
  x = x.abs() if offsets else x
  wide = torch.cat([x, x], 1).cuda()
  packed = rows.pack(wide[:, :d], group=group, offsets=offsets)
  assert torch.equal(packed.codes, rows.pack(x.cuda().contiguous(), group=group, offsets=offsets).codes)
  got = sum(ref.unpack(packed.codes, packed.scales, packed.offsets, d, group))
  step = packed.scales.cpu().double().repeat_interleave(group, 1)[:, :d]
  slack = step * (0.5 + 16 * 2.0 ** -11) + (0 if packed.offsets is None else packed.offsets.cpu().double().abs().repeat_interleave(group, 1)[:, :d] * 2.0 ** -10)
  assert ((got - x.double()).abs() <= slack + 2.0 ** -20).all()
  assert ((packed.unpack().cpu().double() - got).abs() <= got.abs() * 2.0 ** -23 + step * 2.0 ** -20).all()


def test_pack_of_constant_and_of_large_rows():
  from cuhnsw_amd import rows
  x = torch.zeros(4, 64, device="cuda")
  x[1], x[2], x[3] = 5.0, -3.0, 1e30
  assert (rows.pack(x, offsets=True).unpack()[:3] == x[:3]).all()
  packed = rows.pack(x)
  assert torch.isfinite(packed.unpack()).all() and (packed.unpack()[0] == 0).all()
  assert (rows.pack(x, scale_dtype=torch.bfloat16).unpack()[3] / 1e30 - 1).abs().max() < 2.0 ** -8


@pytest.mark.parametrize("dist_type", ["dot", "l2"])
def test_search_of_packed_rows(dist_type):
  """On integers (a scale of one) everything is exact: ids, ties and distances are those of a plain search."""
  from cuhnsw_amd import rows
  n, d = 5000, 24
  x = torch.from_numpy(integer_vectors(n, d, seed=1, hi=5))
  x[:, 0], x[:, 1] = 7, -7     # (every group's largest magnitude: the scale is one)
  packed = rows.pack(x.cuda())
  assert (packed.unpack().cpu() == x).all()
  q = torch.from_numpy(integer_vectors(40, d, seed=2, hi=5)) - 2
  key = -(q.double() @ x.double().t()) if dist_type == "dot" else ((q.double()[:, None] - x.double()[None]) ** 2).sum(2)
  order = key.sort(dim=1, stable=True)
  ids, dist, found = packed.search_knn(q.cuda(), 100, dist_type)
  assert (ids.cpu() == order.indices[:, :100]).all() and (dist.cpu().double() == order.values[:, :100]).all() and (found == 100).all()
  one = packed.search_knn(q[3].cuda(), 7, dist_type)
  assert torch.equal(one[0], ids[3:4, :7])
  few = rows.pack(x[:5].cuda(), labels=torch.arange(5, device="cuda") + 2 ** 40)
  ids, dist, found = few.search_knn(q.cuda(), 8, dist_type)
  assert (found == 5).all() and (ids[:, :5] >= 2 ** 40).all() and (ids[:, 5:] == -1).all() and torch.isinf(dist[:, 5:]).all()


@pytest.mark.parametrize("dist_type", ["dot", "l2"])
def test_packed_rows_of_an_index(dist_type):
  from cuhnsw_amd import CuHNSW
  x = gauss_mixture(4000, 50, seed=8, normalise=dist_type == "dot") + (0 if dist_type == "dot" else 4)
  x = x.astype(np.float32)
  h = CuHNSW({"py_log_level": 1, "heuristic_coef": 0.0, "dist_type": dist_type})
  h.set_data(x)
  packed = h.pack_rows()
  from cuhnsw_amd import rows
  other = rows.pack(torch.from_numpy(x).cuda(), offsets=dist_type == "l2")
  assert torch.equal(packed.codes, other.codes) and torch.equal(packed.scales, other.scales) and packed.labels is None
  h.build()
  q = gauss_mixture(200, 50, seed=9, normalise=False)
  exact = packed.search_knn(torch.from_numpy(q).cuda(), 10, dist_type)[0].cpu().numpy()
  nns = h.search_knn(q, 10, 300)[0]
  shared = np.mean([len(set(a) & set(b)) / 10 for a, b in zip(exact, nns)])
  assert shared > 0.5      # the neighbours of rows in 4 bits are mostly those of the rows


def test_scores_in_a_graph_and_on_another_stream():
  from cuhnsw_amd import rows
  packed = rows.PackedRows(*_codes(3000, 200, 32, True), num_dims=200, group=32)
  for nq in (1, 40):
    q = torch.randn(nq, 200, device="cuda")
    packed.scores(q)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
      graph = torch.cuda.CUDAGraph()
      with torch.cuda.graph(graph):
        out = packed.scores(q)
      graphs.append((graph, out))
    for _ in range(4):
      q.normal_()
      for graph, _ in graphs:
        graph.replay()
      want = packed.scores(q)
      torch.cuda.synchronize()
      for _, out in graphs:
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      late = q * 3
      out = packed.scores(late)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, packed.scores(q * 3))


def test_more_rows_than_one_launch_packs():
  from cuhnsw_amd import rows
  n = (1 << 29) + 5
  x = torch.empty(n, 1, dtype=torch.float16, device="cuda").fill_(3.5)
  x[-5:, 0] = torch.tensor([0.0, -7.0, 1.0, 14.0, -0.5], device="cuda")
  packed, last = rows.pack(x), rows.pack(x[-5:])
  assert torch.equal(packed.codes[-5:], last.codes) and torch.equal(packed.scales[-5:], last.scales)
  assert (packed.scales[:-5] == 0.5).all() and (packed.codes[:-5, 0] == 15).all() and not packed.codes[:-5, 1:].any()


def test_search_of_no_rows():
  from cuhnsw_amd import rows
  packed = rows.pack(torch.zeros(0, 40, device="cuda"))
  for dist_type in ("dot", "l2"):
    ids, dist, found = packed.search_knn(torch.ones(3, 40, device="cuda"), 4, dist_type)
    assert (ids == -1).all() and (dist == float("inf")).all() and (found == 0).all() and ids.shape == dist.shape == (3, 4)


def test_search_by_length_in_a_graph_first_and_on_another_stream_then():
  """The rows' lengths are made when they are first wanted: not to be kept from a capture, and there for every stream."""
  from cuhnsw_amd import rows
  g = torch.Generator().manual_seed(2)
  packed, q = rows.pack(torch.randn(5000, 96, generator=g).cuda()), torch.randn(6, 96, generator=g).cuda()
  want = rows.PackedRows(packed.codes, packed.scales, num_dims=96).search_knn(q, 5, "l2")
  packed.scores(q)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = packed.search_knn(q, 5, "l2")
  other = torch.cuda.Stream()
  other.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(other):
    eager = packed.search_knn(q, 5, "l2")
  here = packed.search_knn(q, 5, "l2")
  torch.cuda.synchronize()
  for _ in range(3):
    for x in out:
      x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c, d in zip(out, want, eager, here):
      assert torch.equal(a, b) and torch.equal(c, b) and torch.equal(d, b)
