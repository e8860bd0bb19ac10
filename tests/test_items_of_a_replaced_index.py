"""Two threads may share an index: what one of them made room for is not written to by the sizes of the other's."""
import ctypes
import threading

import numpy as np
import pytest

from cuhnsw_amd import CuHNSW, capi


class Replaced:
  """A binding whose index another thread replaces at the worst moment: right after `when` was asked for (with vectors, or by a
  call of its own)."""

  def __init__(self, obj, when, data):
    self.obj, self.when, self.data = obj, when, data

  def __getattr__(self, name):
    call = getattr(self.obj, name)
    if name != self.when:
      return call

    def then_replaced(*args):
      answer = call(*args)
      if callable(self.data):
        self.data()
      else:
        self.obj.set_data(self.data)
      return answer
    return then_replaced


def _index(rows, dims, **opt):
  h = CuHNSW({"py_log_level": 1, **opt})
  h.set_data(np.arange(rows * dims, dtype=np.float32).reshape(rows, dims))
  return h


@pytest.mark.parametrize("dims", [2, 300])
def test_items_of_an_index_that_was_replaced_meanwhile(dims):
  h = _index(4, 3)
  h.obj = Replaced(h.obj, "num_dims", np.zeros((4, dims), np.float32))
  with pytest.raises(RuntimeError, match="replaced meanwhile: %d elements a vector, not 3" % dims):
    h.get_items([0, 3])


def test_c_calls_compare_what_the_result_was_made_for():
  l = capi.load()
  e = capi.Engine()
  e.set_data(np.zeros((4, 3), np.float32))
  room = (ctypes.c_longlong * 8)(*[7] * 8)
  items = (ctypes.c_int * 2)(0, 1)
  assert l.cuhnsw_get_items(e._h, items, 2, 4, 1.0, room) == -1
  assert b"replaced meanwhile: 3 elements a vector, not 4" in l.cuhnsw_last_error(e._h)
  for num in (3, 5, 0):
    assert l.cuhnsw_get_labels(e._h, num, room) == -1
    assert b"replaced meanwhile: 4 rows, not %d" % num in l.cuhnsw_last_error(e._h)
  assert list(room) == [7] * 8


@pytest.mark.parametrize("rows, dims, message", [(5, 3, "4 rows, not 5"), (3, 3, "4 rows, not 3"), (4, 2, "3 elements a vector, not 2")])
def test_packing_compares_what_the_room_was_made_for(rows, dims, message):
  l = capi.load()
  e = capi.Engine()
  e.set_data(np.zeros((4, 3), np.float32))
  room = np.full(1024, 7, np.uint8)
  at = (room.ctypes.data + 15) // 16 * 16
  deleted = ctypes.c_int(7)
  assert l.cuhnsw_pack_items(e._h, rows, dims, 32, at, at + 256, None, 1, at + 512, ctypes.addressof(deleted), None) == -1
  assert b"replaced meanwhile: " + message.encode() in l.cuhnsw_last_error(e._h)
  assert (room == 7).all() and deleted.value == 7


@pytest.mark.gpu
def test_items_while_another_thread_replaces_the_index():
  """Every answer is of one of the two indexes, or the call fails and says why."""
  data = [np.random.default_rng(s).standard_normal((n, d), dtype=np.float32) for s, (n, d) in enumerate(((300, 24), (500, 700)))]
  h = CuHNSW({"py_log_level": 1})
  h.set_data(data[0])
  over, wrong = threading.Event(), []

  def replace():
    for turn in range(60):
      h.set_data(data[(turn + 1) % 2])
    over.set()

  items, answers = np.arange(0, 300, 3), 0
  thread = threading.Thread(target=replace)
  thread.start()
  while not over.is_set():
    try:
      got = h.get_items(items)
    except RuntimeError as exc:
      assert "replaced meanwhile" in str(exc)
      continue
    answers += 1
    if not any(got.shape[1] == x.shape[1] and (got == x[items]).all() for x in data):
      wrong.append(got)
  thread.join()
  assert not wrong and answers > 0


@pytest.mark.gpu
@pytest.mark.parametrize("when", ["num_data", "num_dims"])
@pytest.mark.parametrize("rows, dims", [(1000, 24), (300, 200), (100, 24), (300, 8)])
def test_packed_rows_of_an_index_that_was_replaced_meanwhile(rows, dims, when):
  pytest.importorskip("torch")
  h = _index(300, 24)
  obj, h.obj = h.obj, Replaced(h.obj, when, np.ones((rows, dims), np.float32))
  if when == "num_data" and rows == 300:     # (seen before anything was made: the new index's)
    assert h.pack_rows().num_dims == dims
  else:
    with pytest.raises(RuntimeError, match="replaced meanwhile"):
      h.pack_rows()
  h.obj = obj
  assert h.pack_rows().num_rows == rows


@pytest.mark.gpu
def test_labels_of_packed_rows_are_their_own(oracle, tmp_path):
  """An index of the same sizes takes the place of the packed one: its labels, or its deleted elements, are not the packed rows'."""
  pytest.importorskip("torch")
  n, d = 300, 24
  x = np.random.default_rng(1).standard_normal((n, d), dtype=np.float32)
  ix = oracle.OracleIndex("dot").build(x, np.zeros(n, np.int32), 8, 16, 40, 0.4)
  plain, marked, named = (str(tmp_path / name) for name in ("plain.idx", "marked.idx", "named.idx"))
  ix.save(plain)
  ix.mark_deleted([3, 8])
  ix.save(marked)
  raw = bytearray(open(plain, "rb").read())
  record, label_at = 4 + 16 * 4 + d * 4 + 8, 4 + 16 * 4 + d * 4
  for i in range(n):
    at = 96 + i * record + label_at
    assert int.from_bytes(raw[at:at + 8], "little") == i
    raw[at:at + 8] = (2 * i + 100).to_bytes(8, "little")
  open(named, "wb").write(raw)
  h = CuHNSW({"py_log_level": 1, "max_m": 8, "max_m0": 16})
  obj = h.obj
  h.load_index(named)
  h.obj = Replaced(obj, "pack_items", lambda: obj.load_index(plain.encode()))
  packed = h.pack_rows()
  assert packed.labels.tolist() == [2 * i + 100 for i in range(n)]
  h.obj = obj
  h.load_index(marked)
  with pytest.raises(RuntimeError, match="deleted elements"):
    h.pack_rows()
  h.load_index(plain)
  h.obj = Replaced(obj, "num_deleted", lambda: obj.load_index(marked.encode()))
  with pytest.raises(RuntimeError, match="deleted elements"):
    h.pack_rows()
