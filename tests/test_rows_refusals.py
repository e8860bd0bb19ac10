"""What the operators on rows refuse, checked without a GPU: wrong shapes, types and sizes before anything looks at the device,
tensors that are not on one, and the C ABI's own checks."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from cuhnsw_amd import capi, rows  # noqa: E402


def _table(*shape, dtype=torch.float32):
  return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call, kind, message", [
    (lambda: rows.lookup([1.0], torch.zeros(1, dtype=torch.int64)), TypeError, "table is a tensor"),
    (lambda: rows.lookup(_table(4), torch.zeros(1, dtype=torch.int64)), ValueError, "table has 1 dimensions"),
    (lambda: rows.lookup(_table(4, 3, dtype=torch.float64), torch.zeros(1, dtype=torch.int64)), ValueError, "type torch.float64"),
    (lambda: rows.lookup(_table(4, 3), torch.zeros(1)), ValueError, "ids has the type"),
    (lambda: rows.lookup(_table(4, 3), torch.zeros(1, dtype=torch.int16)), ValueError, "ids has the type"),
    (lambda: rows.lookup(_table(4, 3), torch.zeros(1, dtype=torch.int64), scale="2"), TypeError, "scale is a number"),
    (lambda: rows.lookup(_table(4, 3), torch.zeros(1, dtype=torch.int64), scale=torch.ones(1)), TypeError, "scale is a number"),
    (lambda: rows.lookup(_table(4, 3), torch.zeros(1, dtype=torch.int64), dtype=torch.float16), ValueError, "the table's type"),
    (lambda: rows.lookup(_table(4, 0), torch.zeros(1, dtype=torch.int64)), ValueError, "empty"),
    (lambda: rows.lookup(_table(4, 3), torch.zeros(1, dtype=torch.int64)), ValueError, "on the GPU"),
    (lambda: rows.lookup_grad(_table(2, 3), torch.zeros(3, dtype=torch.int64), 4), ValueError, "shape"),
    (lambda: rows.lookup_grad(_table(2, 3), torch.zeros(2, dtype=torch.int64), -1), ValueError, "num_rows"),
    (lambda: rows.lookup_grad(_table(2, 3, dtype=torch.float16), torch.zeros(2, dtype=torch.int64), 4, dtype=torch.float32), ValueError, "float32"),
    (lambda: rows.lookup_grad(_table(2, 3), torch.zeros(2, dtype=torch.int64), 4), ValueError, "on the GPU"),
    (lambda: rows.pack(_table(4, 3), group=48), ValueError, "32, 64 or 128"),
    (lambda: rows.pack(_table(4, 3), scale_dtype=torch.float32), ValueError, "scales are"),
    (lambda: rows.pack(_table(4, 0)), ValueError, "empty"),
    (lambda: rows.pack(_table(4, 3)), ValueError, "on the GPU"),
    (lambda: rows.select_beams(_table(2, 3), None, 1), ValueError, "dimensions"),
    (lambda: rows.select_beams(_table(2, 3, 5), None, 0), ValueError, "between 1 and 256"),
    (lambda: rows.select_beams(_table(2, 3, 5), None, 257), ValueError, "between 1 and 256"),
    (lambda: rows.select_beams(_table(2, 40, 300), None, 200), ValueError, "at most 4096"),
    (lambda: rows.select_beams(_table(2, 0, 5), None, 1), ValueError, "no beams"),
    (lambda: rows.select_beams(_table(2, 3, 10)[:, :, ::2], None, 1), ValueError, "contiguous"),
    (lambda: rows.select_beams(_table(2, 3, 5), _table(2, 4), 1), ValueError, "beams have the shape"),
    (lambda: rows.select_beams(_table(2, 3, 5), None, 1, finished=torch.zeros(2, 3, dtype=torch.bool), end=0), ValueError, "what they gathered"),
    (lambda: rows.select_beams(_table(2, 3, 5), _table(2, 3), 1, finished=torch.zeros(2, 3, dtype=torch.bool)), ValueError, "token that ends"),
    (lambda: rows.select_beams(_table(2, 3, 5), _table(2, 3), 1, finished=torch.zeros(2, 3, dtype=torch.bool), end=5), ValueError, "token that ends"),
    (lambda: rows.select_beams(_table(2, 3, 5), _table(2, 3), 1), ValueError, "on the GPU"),
    (lambda: rows.reorder_states(_table(2, 3, 5), torch.zeros(2, 3, dtype=torch.int32)), TypeError, "list of tensors"),
    (lambda: rows.reorder_states([_table(2, 3, 5)], torch.zeros(2, 3, dtype=torch.int64)), ValueError, "parents has the type"),
    (lambda: rows.reorder_states([_table(3, 3, 5)], torch.zeros(2, 3, dtype=torch.int32)), ValueError, "states have the shape"),
    (lambda: rows.reorder_states([_table(2, 3, 5), _table(2, 4, 5)], torch.zeros(2, 3, dtype=torch.int32)), ValueError, "states have the shape"),
    (lambda: rows.reorder_states([_table(2, 3, 5, 4).transpose(2, 3)], torch.zeros(2, 3, dtype=torch.int32)), ValueError, "contiguous"),
    (lambda: rows.reorder_states([_table(2, 3, 5)], torch.zeros(2, 3, dtype=torch.int32)), ValueError, "on the GPU"),
])
def test_wrong_arguments_are_refused(call, kind, message):
  with pytest.raises(kind, match=message):
    call()


def test_packed_rows_check_their_parts():
  codes, scales = torch.zeros(5, 32, dtype=torch.uint8), torch.zeros(5, 2, dtype=torch.float16)

  def make(codes=codes, scales=scales, offsets=None, num_dims=50, group=32, labels=None):
    return rows.PackedRows(codes, scales, offsets, num_dims=num_dims, group=group, labels=labels)

  for message, args in [("32, 64 or 128", dict(group=16)), ("are 64 bytes a row", dict(num_dims=100, scales=torch.zeros(5, 4, dtype=torch.float16))),
                        ("scales have the shape", dict(group=64)), ("scales has the type", dict(scales=scales.float())),
                        ("offsets has the type", dict(offsets=scales.bfloat16())), ("shape of scales", dict(offsets=scales[:4])),
                        ("positive", dict(num_dims=0)), ("one label a row", dict(labels=torch.zeros(4, dtype=torch.int64))),
                        ("contiguous", dict(scales=torch.zeros(2, 5, dtype=torch.float16).t())), ("on the GPU", {})]:
    with pytest.raises(ValueError, match=message):
      make(**args)
  with pytest.raises(ValueError, match="codes has the type"):
    make(codes=codes.int())


def test_scratch_sizes():
  l = capi.load()
  for args in ((0, 5, 3), (5, 0, 3), (5, 5, 0), (-1, 5, 3)):
    assert l.cuhnsw_lookup_grad_workspace(*args) == 0
  assert l.cuhnsw_lookup_grad_workspace(2048, 1000, 50) == 0    # (few ids need none)
  assert l.cuhnsw_lookup_grad_workspace(100000, 1183514, 50) >= 100000 * 8
  assert l.cuhnsw_select_beams_workspace(0, 0, 1, 1, 1) == 0
  assert l.cuhnsw_select_beams_workspace(3, 1, 1, 1, 1) == 0
  assert l.cuhnsw_select_beams_workspace(0, 3, 4, 1000, 8) >= 3 * 4 * 8


@pytest.mark.skipif(capi.has_device(), reason="checks the no-GPU error path")
def test_calls_without_a_gpu_say_so(tmp_path):
  l = capi.load()
  buf = ctypes.create_string_buffer(4096)
  at = ctypes.addressof(buf)
  assert l.cuhnsw_lookup_rows(at, 0, 4, 3, 3, at, 0, 2, 1.0, at, 0, None) == -1
  assert b"no HIP device" in l.cuhnsw_last_error(None)
  assert l.cuhnsw_select_beams(at, 0, 5, 5, 1, 1, 5, None, None, 0, 1, 1, at, at, at, at, 4096, None) == -1
  assert b"no HIP device" in l.cuhnsw_last_error(None)
  import numpy as np
  from cuhnsw_amd import CuHNSW
  h = CuHNSW({"py_log_level": 1})
  h.set_data(np.ones((4, 3), np.float32))
  for call in (lambda: h.get_items([0]), lambda: h.search_items([0], 1, 1), lambda: h.obj.get_labels()):
    with pytest.raises(RuntimeError, match="no HIP device"):
      call()


def test_items_are_whole_numbers_that_fit():
  import numpy as np
  from cuhnsw_amd import CuHNSW
  h = CuHNSW({"py_log_level": 1})
  h.set_data(np.ones((4, 3), np.float32))
  for items in ([0.5], [[0, 1]], [-1], [1 << 31], "a"):
    with pytest.raises(ValueError):
      h.get_items(items)
