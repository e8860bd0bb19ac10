"""Rows by id and the gradient of that, on the GPU, against plain statements in 64 bits: types, odd sizes, strides, ids outside the
table, one id many times, other streams, graphs, and the index's own vectors."""
import numpy as np
import pytest
import torch

import rows_reference as ref
from helpers import gauss_mixture

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _table(n, d, dtype, seed=0, stride=0):
  g = torch.Generator().manual_seed(seed)
  x = torch.randn(n, d + stride, generator=g).to(dtype).cuda()
  return x[:, :d]


def _ids(n, shape, seed=1, dtype=torch.int64, outside=True):
  g = torch.Generator().manual_seed(seed)
  low, high = (-2, n + 2) if outside else (0, n)
  return torch.randint(low, max(high, low + 1), shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, shape, stride", [
    (1, 1, (1,), 0), (3, 1, (7,), 0), (100, 50, (8,), 0), (77, 101, (33,), 0), (64, 96, (5, 7), 0), (31, 128, (64,), 8), (40, 50, (9,), 3),
    (500, 960, (1001,), 0), (1000, 1024, (300,), 0), (9, 2050, (11,), 0), (20, 33, (2, 3, 4), 31), (10, 24, (0,), 0), (2000, 200, (70000,), 0)])
def test_lookup(n, d, shape, stride, dtype):
  from cuhnsw_amd import rows
  table, ids = _table(n, d, dtype, stride=stride), _ids(n, shape)
  for scale in (1.0, 0.37):
    for out_type in {dtype, torch.float32}:
      print("lookup", n, d, shape, stride, dtype, scale, out_type, flush=True)
      out = rows.lookup(table, ids.int() if scale == 1.0 else ids, scale=scale, dtype=out_type)
      assert out.shape == (*shape, d) and out.dtype == out_type
      want = ref.lookup(table, ids, float(np.float32(scale)))
      assert ((out.cpu().double() - want).abs() <= want.abs() * ref.HALF32 + ref.stored(want, out_type)).all()
      if scale == 1.0:
        assert (out.cpu().double() == want).all()


def test_lookup_in_an_empty_table_and_of_special_values():
  from cuhnsw_amd import rows
  out = rows.lookup(torch.empty(0, 5, device="cuda"), _ids(3, (4,)))
  assert (out == 0).all() and out.shape == (4, 5)
  table = torch.tensor([[float("nan"), float("inf"), -float("inf"), -0.0, 1e-40, 3e38]], device="cuda")
  out = rows.lookup(table, torch.tensor([0, 1, -1], device="cuda"))
  assert out[0].isnan()[0] and (out[0, 1:] == table[0, 1:]).all() and (out[1:] == 0).all()
  half = rows.lookup(table.bfloat16(), torch.tensor([0], device="cuda"))
  assert half[0].isnan()[0] and (half[0, 1:] == table.bfloat16()[0, 1:]).all()


def test_an_id_is_compared_in_64_bits():
  from cuhnsw_amd import rows
  table = _table(5, 8, torch.float32)
  ids = torch.tensor([2 ** 32 + 1, -(2 ** 32) + 1, 1, 2 ** 62], device="cuda")
  out = rows.lookup(table, ids)
  assert (out[[0, 1, 3]] == 0).all() and (out[2] == table[1]).all()
  grad = rows.lookup_grad(torch.ones(4, 8, device="cuda"), ids, 5)
  assert grad.sum() == 8 and (grad[1] == 1).all()


def test_the_place_of_a_row_passes_32_bits():
  from cuhnsw_amd import rows
  n, d = 2_200_000, 1024   # 2.25 G elements
  table = torch.zeros(n, d, dtype=torch.float16, device="cuda")
  at = torch.tensor([n - 1, 5, n - 70_000], device="cuda")
  table[at] = torch.arange(3 * d, device="cuda").reshape(3, d).half()
  assert (rows.lookup(table, at) == table[at]).all()
  g = torch.randn(3, d, device="cuda").half()
  grad = rows.lookup_grad(g, at, n)
  assert (grad[at] == g).all()
  grad[at] = 0
  assert not grad.view(torch.int16).any()


def _check_grad(grad, ids, n, scale, dtype):
  from cuhnsw_amd import rows
  got = rows.lookup_grad(grad, ids, n, scale, dtype)
  want, bound = ref.lookup_grad(grad, ids, n, float(np.float32(scale)))
  off = (got.cpu().double() - want).abs()
  assert got.dtype == dtype and got.shape == (n, grad.shape[-1])
  assert (off <= bound + ref.stored(want.abs() + bound, dtype)).all()
  again = rows.lookup_grad(grad, ids, n, scale, dtype)
  assert torch.equal(got, again)
  return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, t", [
    (1, 1, 1), (1, 50, 3000), (5, 7, 0), (3, 33, 100), (100, 50, 8), (1000, 50, 1000), (77, 101, 2047), (77, 101, 2048), (77, 101, 2049), (5000, 96, 5000),
    (300, 128, 20000), (2, 960, 4100), (4097, 24, 70001), (131, 1024, 9000), (200_000, 24, 6000), (9, 2050, 130), (3_000_000, 2, 5000)])
def test_gradient(n, d, t, dtype):
  g = torch.Generator().manual_seed(n + t)
  grad = torch.randn(t, d, generator=g).to(dtype).cuda()
  print("gradient", n, d, t, dtype, flush=True)
  _check_grad(grad, _ids(n, (t,), seed=t), n, 0.7, dtype)


@pytest.mark.parametrize("t", [1, 64, 65, 500, 2048, 2049, 5000, 66_000])
@pytest.mark.parametrize("law", ["one", "two", "none", "runs", "frequent"])
def test_gradient_of_ids_that_come_often(t, law):
  n, d = 1000, 40
  at = torch.arange(t)
  ids = {"one": torch.full((t,), 7), "two": at % 2 * 999, "none": torch.full((t,), -1), "runs": at // 63 % n,
         "frequent": torch.where(at % 3 == 0, 5, at * 7919 % n)}[law].cuda()
  grad = torch.randn(t, d, generator=torch.Generator().manual_seed(t)).cuda()
  print("gradient of", law, t, flush=True)
  for dtype in (torch.float32, torch.bfloat16):
    _check_grad(grad, ids, n, 1.0, dtype)
  _check_grad(grad.half(), ids.int(), n, 3.0, torch.float16)


def test_gradient_takes_strided_and_expanded_gradients():
  ids = _ids(50, (300,))
  base = torch.randn(300, 64, device="cuda")
  for grad in (base[:, :40], base[:, ::2], torch.ones(1, 30, device="cuda").expand(300, 30), base.t().contiguous().t()[:, :33]):
    _check_grad(grad, ids, 50, 1.0, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(dtype):
  from cuhnsw_amd import rows
  table = _table(300, 50, dtype).clone().requires_grad_(True)
  ids = _ids(300, (40, 7))
  out = rows.lookup(table, ids, scale=0.5)
  w = torch.randn(out.shape, device="cuda").to(dtype)
  (out * w).sum().backward()
  want, bound = ref.lookup_grad(w, ids, 300, 0.5)
  assert table.grad.dtype == dtype
  assert ((table.grad.cpu().double() - want).abs() <= bound + ref.stored(want.abs() + bound, dtype)).all()
  wide = rows.lookup(table, ids, scale=0.5, dtype=torch.float32)
  g, = torch.autograd.grad(wide, table, w.float())
  assert g.dtype == dtype
  assert ((g.cpu().double() - want).abs() <= bound + ref.stored(want.abs() + bound, dtype)).all()
  with pytest.raises(RuntimeError):   # once
    g, = torch.autograd.grad(rows.lookup(table, ids), table, w.requires_grad_(True), create_graph=True)
    g.sum().backward()


def test_gradient_against_differences():
  """The loss is linear in the table, so differences at any step are exact but for rounding: 64-bit sums of float32 results."""
  from cuhnsw_amd import rows
  table = torch.randn(20, 6, device="cuda").requires_grad_(True)
  ids = torch.tensor([3, 3, -1, 19, 0, 3, 25], device="cuda")
  w = torch.randn(7, 6, device="cuda")

  def loss(x):
    return (rows.lookup(x, ids, scale=1.5).double() * w.double()).sum()

  loss(table).backward()
  with torch.no_grad():
    for v, k in ((3, 0), (3, 5), (19, 2), (0, 1), (7, 3)):
      up = table.clone()
      up[v, k] += 1.0
      # a lookup is one rounding of about 2^-24 of values under 16; three of them, with weights under 5, and the step's own
      assert abs((loss(up) - loss(table)) / (up[v, k] - table[v, k]).double() - table.grad[v, k].double()) < 3 * 5 * 16 * 2.0 ** -23


def test_lookup_on_another_stream():
  from cuhnsw_amd import rows
  table, ids = _table(3000, 128, torch.float32), _ids(3000, (5000,))
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    late = table * 2.0   # (only this stream knows when it is done)
    out = rows.lookup(late, ids)
    grad = rows.lookup_grad(out, ids, 3000)
  torch.cuda.current_stream().wait_stream(side)
  assert (out.cpu().double() == ref.lookup(table, ids, 2.0)).all()
  want, bound = ref.lookup_grad(out, ids, 3000, 1.0)
  assert ((grad.cpu().double() - want).abs() <= bound + ref.stored(want, torch.float32)).all()


@pytest.mark.parametrize("t", [300, 9000])
def test_lookup_and_gradient_in_a_graph(t):
  """Captured once, replayed with other data, beside eager calls that use scratch memory of their own."""
  from cuhnsw_amd import rows
  n, d = 700, 48
  table, ids = _table(n, d, torch.float32).clone(), _ids(n, (t,))
  grad = torch.randn(t, d, device="cuda")
  rows.lookup(table, ids), rows.lookup_grad(grad, ids, n)
  torch.cuda.synchronize()
  graphs = []
  for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      outs = rows.lookup(table, ids, scale=2.0), rows.lookup_grad(grad, ids, n, 0.5)
    graphs.append((graph, outs))
  for turn in range(4):
    ids.copy_(_ids(n, (t,), seed=turn + 10))
    table.normal_()
    grad.normal_()
    for graph, _ in graphs:
      graph.replay()
    want = rows.lookup(table, ids, scale=2.0), rows.lookup_grad(grad, ids, n, 0.5)
    torch.cuda.synchronize()
    for _, outs in graphs:
      assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("half", [False, True])
def test_items_of_an_index(half, tmp_path):
  from cuhnsw_amd import CuHNSW
  x = gauss_mixture(3000, 50, seed=3)
  h = CuHNSW({"py_log_level": 1, "heuristic_coef": 0.0})
  if half:
    h.obj.set_tunable("fp16_storage", 1)
  h.set_data(x)
  held = x.astype(np.float16).astype(np.float32) if half else x
  items = [7, 0, 2999, 7]
  assert (h.get_items(items) == held[items]).all()
  assert (h.get_items(items, scale=0.5) == held[items] * np.float32(0.5)).all()
  assert h.get_items([]).shape == (0, 50)
  with pytest.raises(RuntimeError, match="outside the index"):
    h.get_items([3000])
  h.build()
  many = np.arange(0, 3000, 7)
  for got, want in zip(h.search_items(many, 10, 100), h.search_knn(held[many], 10, 100)):
    assert (got == want).all()
  with pytest.raises(RuntimeError, match="outside the index"):
    h.search_items([3000], 1, 10)


def test_items_of_a_loaded_index_go_by_label(tmp_path):
  from cuhnsw_amd import CuHNSW
  x = gauss_mixture(500, 24, seed=5)
  h = CuHNSW({"py_log_level": 1, "heuristic_coef": 0.0, "max_m": 8, "max_m0": 16})
  h.set_data(x)
  h.build()
  path = str(tmp_path / "a.idx")
  h.save_index(path)
  raw = bytearray(open(path, "rb").read())
  header, record, label_at = 96, 4 + 16 * 4 + 24 * 4 + 8, 4 + 16 * 4 + 24 * 4
  labels = np.random.default_rng(0).permutation(500) * 3 + 11
  for i, label in enumerate(labels):
    at = header + i * record + label_at
    assert int.from_bytes(raw[at:at + 8], "little") == i     # (the file's layout is what this test takes it to be)
    raw[at:at + 8] = int(label).to_bytes(8, "little")
  open(path, "wb").write(raw)
  h.load_index(path)
  items = labels[[3, 499, 0]]
  assert (h.get_items(items) == x[[3, 499, 0]]).all()
  nns, dist, found = h.search_items(items, 5, 50)
  for got, want in zip((nns, dist, found), h.search_knn(x[[3, 499, 0]], 5, 50)):
    assert (got == want).all()
  assert (nns[:, 0] == items).all() or (dist[:, 0] <= dist[:, 1]).all()
  with pytest.raises(RuntimeError, match="no item has the label 12"):
    h.get_items([12])
  packed = h.pack_rows()
  assert (packed.labels.cpu().numpy() == labels).all()
