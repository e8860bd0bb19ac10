"""Two threads may share an index: what one of them made room for is not written to by the sizes of the other's."""
import ctypes
import threading

import numpy as np
import pytest

from cuhnsw_amd import CuHNSW, capi


class Replaced:
  """A binding whose index another thread replaces at the worst moment: right after `when` was asked for."""

  def __init__(self, obj, when, data):
    self.obj, self.when, self.data = obj, when, data

  def __getattr__(self, name):
    call = getattr(self.obj, name)
    if name != self.when:
      return call

    def then_replaced(*args):
      answer = call(*args)
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
