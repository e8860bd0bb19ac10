"""Operators on tables of learned vectors that are on the GPU, as torch tensors: what a user of the index needs next to it.

  lookup(table, ids, scale)        rows by id, differentiable: queries made of items, a model's input embedding
  pack(vectors) -> PackedRows      rows in 4 bits with a scale per group of elements
  PackedRows.scores(queries)       products with every row: the exact form of what a search answers approximately
  PackedRows.search_knn(...)       the best rows of all, as CuHNSW.search_knn returns them
  select_beams(scores, ...)        the best candidates over beams and vocabulary; over one beam: the nearest neighbours
  reorder_states(states, parents)  the beams' states in their new order

Every call runs on its tensors' device and torch's current stream there, does not wait for the GPU, takes its scratch
memory from torch, and may be captured into a graph (pack_index waits, and may not; PackedRows.norms waits once).  lookup
is differentiable, the others are not: their results carry no gradient and no tangent, whatever their inputs do.  Wrong
arguments are a ValueError (a TypeError where the kind of object is wrong); what the native library refuses is a RuntimeError with its message, as everywhere in this package.
There is no CPU form.

torch ships its own copy of the HIP runtime: it has to be imported before this package's native library is loaded, or
the process holds two runtimes that do not know each other's memory.
"""
import sys

if "torch" not in sys.modules and "cuhnsw_amd.cuhnsw_bind" in sys.modules:
  raise ImportError("cuhnsw_amd.rows: import torch before cuhnsw_amd (two HIP runtimes would be loaded otherwise)")

import ctypes
import numbers

import numpy as np
import torch

try:
  from cuhnsw_amd import cuhnsw_bind as _native
except ImportError as exc:  # pragma: no cover
  raise ImportError("cuhnsw_amd: the native extension is missing (%s); build it with `python -m cuhnsw_amd.build`" % exc) from exc


def _one_hip_runtime():
  """Whether torch and the native library call the same one (not where torch was imported after the library was loaded)."""
  def runtime_of(module):
    return ctypes.cast(ctypes.CDLL(module.__file__).hipGetDeviceCount, ctypes.c_void_p).value
  try:
    return runtime_of(torch._C) == runtime_of(_native)
  except AttributeError:  # (a torch without HIP)
    return True


if not _one_hip_runtime():
  raise ImportError("cuhnsw_amd.rows: import torch before cuhnsw_amd (two HIP runtimes are loaded)")

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_GROUPS = (32, 64, 128)


def _check(ok, message, *args):
  if not ok:
    raise ValueError(message % args)


def _tensor(x, name, dims=None, types=_TYPES):
  if not isinstance(x, torch.Tensor):
    raise TypeError("%s is a tensor, not %s" % (name, type(x).__name__))
  _check(dims is None or x.dim() == dims, "%s has %s dimensions, %s are wanted", name, x.dim(), dims)
  _check(x.dtype in types, "%s has the type %s: %s is wanted", name, x.dtype, " or ".join(str(t) for t in types))
  _check(not x.is_neg(), "%s is a view that is still to be negated (resolve_neg)", name)


def _rows(x, name):
  """The row stride of a matrix whose rows are contiguous, whatever lies between them (an expanded one's is 0)."""
  _check(x.shape[1] <= 1 or x.stride(1) == 1, "the elements of one row of %s have to be contiguous", name)
  return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _same_device(first, *others):
  """The number of the GPU that all of the tensors are on."""
  device = first.get_device()
  _check(device >= 0, "the tensors have to be on the GPU")
  for x in others:
    _check(x is None or x.get_device() == device, "the tensors are on different devices")
  return device


def _number(x, name):
  if type(x) is not float:
    if not isinstance(x, numbers.Real) or isinstance(x, bool):
      raise TypeError("%s is a number, not %s" % (name, type(x).__name__))
    x = float(x)
  return x


# (the native calls take the device's number and make it the current one while they launch; the handle of torch's current
# stream is asked for without the object around it where that is possible: together a few microseconds a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _workspace(size, like):
  return like.new_empty(size, dtype=torch.uint8) if size else None


def _address(x):
  return 0 if x is None else x.data_ptr()


# -------------------------------------------------------------------------------------------------- lookup
_IDS = {torch.int32: 0, torch.int64: 1}


def _flat(ids):
  ids = ids if ids.dim() == 1 else ids.reshape(-1)
  return ids if ids.is_contiguous() else ids.contiguous()


def _lookup(table, stride, flat, scale, dtype, device):
  dims = table.shape[1]
  out = table.new_empty((flat.shape[0], dims), dtype=dtype)
  _native.lookup_rows(table.data_ptr(), _TYPES[table.dtype], table.shape[0], stride, dims, flat.data_ptr(), _IDS[flat.dtype],
                      flat.shape[0], scale, out.data_ptr(), _TYPES[dtype], device, _raw_stream(device))
  return out


_tangent = torch.autograd.forward_ad.unpack_dual


def _grad_workspace(flat, num_rows, dims):
  return _native.lookup_grad_workspace(flat.shape[0], num_rows, dims)


def _lookup_grad(grad, flat, num_rows, dims, scale, dtype, size, device):
  stride = dims
  if not grad.is_contiguous():
    grad = grad.reshape(-1, dims)
    if dims > 1 and grad.stride(1) != 1:
      grad = grad.contiguous()
    stride = _rows(grad, "grad")
  out = grad.new_empty((num_rows, dims), dtype=dtype)
  work = grad.new_empty(size, dtype=torch.uint8) if size else None
  _native.lookup_rows_grad(grad.data_ptr(), _TYPES[grad.dtype], stride, flat.data_ptr(), _IDS[flat.dtype], flat.shape[0], num_rows, dims, scale,
                           out.data_ptr(), _TYPES[dtype], work.data_ptr() if size else 0, size, device, _raw_stream(device))
  return out


class _Lookup(torch.autograd.Function):
  """(What can be found out in the forward pass is: the backward pass runs on autograd's own thread, where Python is slow.)"""

  @staticmethod
  def forward(ctx, table, stride, flat, shape, scale, dtype, device):
    num_rows, dims = table.shape
    ctx.save_for_backward(flat)
    ctx.rest = num_rows, dims, scale, table.dtype, _grad_workspace(flat, num_rows, dims), device
    out = _lookup(table, stride, flat, scale, dtype, device)
    return out if shape is None else out.view(shape)

  @staticmethod
  def backward(ctx, grad):
    if torch.is_grad_enabled():  # (a graph of the gradient is wanted: one that says that it cannot be had)
      return _Lookup.backward_of_once(ctx, grad)
    return _lookup_grad(grad, *ctx.saved_tensors, *ctx.rest), None, None, None, None, None, None

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward_of_once(ctx, grad):
    return _lookup_grad(grad, *ctx.saved_tensors, *ctx.rest), None, None, None, None, None, None


def lookup(table, ids, scale=1.0, dtype=None):
  """scale * table[ids], zeros where an id is outside [0, len(table)) (padded places: -1).

  table: [rows, dims], float32, float16 or bfloat16, rows contiguous; ids: int32 or int64 of any shape; the result, of
  shape [*ids.shape, dims], has the table's type or is float32.  Products are taken in 32 bits and rounded once.
  Differentiable with respect to table (once, and in reverse: a table with a forward-mode tangent is refused): see
  lookup_grad.  Where a backward pass is captured into a graph, no eager graph over the same table may be alive (its leaf
  belongs to another stream then, which torch would wait for)."""
  _tensor(table, "table", 2)
  _tensor(ids, "ids", types=_IDS)
  scale = _number(scale, "scale")
  dtype = dtype or table.dtype
  _check(dtype is table.dtype or dtype is torch.float32, "the result has the table's type or is float32")
  _check(table.shape[1] > 0, "the table's rows are empty")
  stride = _rows(table, "table")
  _check(_tangent(table).tangent is None, "lookup has no forward-mode derivative")
  device = _same_device(table, ids)
  flat, shape = _flat(ids), None if ids.dim() == 1 else (*ids.shape, table.shape[1])
  if table.requires_grad and torch.is_grad_enabled():
    return _Lookup.apply(table, stride, flat, shape, scale, dtype, device)
  out = _lookup(table, stride, flat, scale, dtype, device)
  return out if shape is None else out.view(shape)


def lookup_grad(grad, ids, num_rows, scale=1.0, dtype=None):
  """The gradient of lookup with respect to its table: [num_rows, dims], row v the sum of scale * grad[t] over the places
  t with ids[t] = v.

  grad: [*ids.shape, dims]; at most 2^30 ids and 2^31 - 2 rows.  The sums are formed in 32 bits, in an order that depends on the sizes and the
  ids alone, and rounded once to
  `dtype` (grad's own, or any where grad is float32): the same inputs give the same bits."""
  _tensor(grad, "grad")
  _tensor(ids, "ids", types=_IDS)
  scale = _number(scale, "scale")
  dtype = dtype or grad.dtype
  _check(dtype in _TYPES and (grad.dtype in (dtype, torch.float32)), "the gradient of a %s table is of that type or float32", dtype)
  _check(grad.dim() == ids.dim() + 1 and grad.shape[:-1] == ids.shape, "grad has the shape [*ids.shape, dims]")
  _check(grad.shape[-1] > 0, "the rows of grad are empty")
  _check(isinstance(num_rows, int) and num_rows >= 0, "num_rows is a whole number that is not negative")
  device, flat, dims = _same_device(grad, ids), _flat(ids), grad.shape[-1]
  return _lookup_grad(grad, flat, num_rows, dims, scale, dtype, _grad_workspace(flat, num_rows, dims), device)


# -------------------------------------------------------------------------------------------- rows in 4 bits
_SCALES = {torch.float16: 1, torch.bfloat16: 2}


class PackedRows:
  """Rows held in 4 bits: element k of row n is scales[n][k // group] * (code - 8) or, with offsets,
  scales[n][k // group] * code + offsets[n][k // group].

  codes: uint8 [rows, 16 * ceil(num_dims / 32)], element 2 i in the low half of byte i (what is behind num_dims elements is
  not looked at); scales, offsets: float16 or bfloat16 [rows, ceil(num_dims / group)]; group: 32, 64 or 128.  The tensors are
  used as they are, not copied.  labels: int64 [rows], what search_knn returns instead of row numbers, or None."""

  def __init__(self, codes, scales, offsets=None, *, num_dims, group=32, labels=None):
    _check(isinstance(num_dims, int) and num_dims > 0, "num_dims is a positive whole number")
    _check(group in _GROUPS, "the group is 32, 64 or 128 elements")
    _tensor(codes, "codes", 2, (torch.uint8,))
    _tensor(scales, "scales", 2, _SCALES)
    width, groups = 16 * -(-num_dims // 32), -(-num_dims // group)
    _check(codes.shape[1] == width, "codes of %d elements are %d bytes a row", num_dims, width)
    _check(tuple(scales.shape) == (codes.shape[0], groups), "scales have the shape (%d, %d)", codes.shape[0], groups)
    if offsets is not None:
      _tensor(offsets, "offsets", 2, (scales.dtype,))
      _check(offsets.shape == scales.shape, "offsets have the shape of scales")
    if labels is not None:
      _tensor(labels, "labels", 1, (torch.int64,))
      _check(labels.shape[0] == codes.shape[0], "there is one label a row")
    for name, x in (("codes", codes), ("scales", scales), ("offsets", offsets)):
      _check(x is None or x.is_contiguous(), "%s have to be contiguous", name)
    _check(codes.data_ptr() % 16 == 0, "codes have to be aligned to 16 bytes")
    _same_device(codes, scales, offsets, labels)
    self.codes, self.scales, self.offsets, self.labels = codes, scales, offsets, labels
    self.num_rows, self.num_dims, self.group = codes.shape[0], num_dims, group
    self._norms = None

  def __len__(self):
    return self.num_rows

  def scores(self, queries, alpha=1.0, bias=None, dtype=None):
    """alpha * queries @ rows.T (+ bias): [num_queries, num_rows], of the queries' type or float32.

    queries: [num_queries, num_dims] (or one: [num_dims]), at most 16 777 200, float32, float16 or bfloat16; bias: float32
    [num_rows].  Sums are held in 32 bits; a float32 query as two planes of float16, good to 2^-23 of an element or 2^-39 of its largest
    one.  A query that is not finite gets scores that are not."""
    _tensor(queries, "queries")
    _check(queries.dim() in (1, 2) and queries.shape[-1] == self.num_dims, "queries have the shape [num_queries, %d]", self.num_dims)
    alpha = _number(alpha, "alpha")
    dtype = dtype or queries.dtype
    _check(dtype in (queries.dtype, torch.float32), "the scores have the queries' type or are float32")
    if bias is not None:
      _tensor(bias, "bias", 1, (torch.float32,))
      _check(bias.shape[0] == self.num_rows and bias.is_contiguous(), "bias is contiguous, one value a row")
    device = _same_device(self.codes, queries, bias)
    q = queries if queries.dim() == 2 else queries[None]
    nq, kind = q.shape[0], _TYPES[q.dtype]
    out = q.new_empty((nq, self.num_rows), dtype=dtype)
    size = _native.packed_scores_workspace(self.num_rows, self.num_dims, self.group, kind, nq)
    work = _workspace(size, q)
    _native.packed_scores(self.codes.data_ptr(), self.scales.data_ptr(), _address(self.offsets), _SCALES[self.scales.dtype], self.num_rows,
                          self.num_dims, self.group, q.data_ptr(), kind, _rows(q, "queries"), nq, alpha, _address(bias), out.data_ptr(),
                          _TYPES[dtype], self.num_rows, _address(work), size, device, _raw_stream(device))
    return out if queries.dim() == 2 else out[0]

  def unpack(self):
    """The rows as float32 [num_rows, num_dims]."""
    values = torch.stack((self.codes & 15, self.codes >> 4), dim=2).view(self.num_rows, -1)[:, :self.num_dims].float()
    column = torch.arange(self.num_dims, device=self.codes.device) // self.group
    scales = self.scales.float()[:, column]
    return (values - 8.0) * scales if self.offsets is None else values * scales + self.offsets.float()[:, column]

  def norms(self):
    """Squared lengths of the rows, float32.  Computed and waited for once, for every stream (the rows must not change
    afterwards); inside a capture they belong to the graph and are not kept."""
    if self._norms is None:
      device = self.codes.device
      out = torch.empty(self.num_rows, dtype=torch.float32, device=device)
      step = max(1, (64 << 20) // self.num_dims)
      for low in range(0, self.num_rows, step):
        part = PackedRows(self.codes[low:low + step], self.scales[low:low + step],
                          None if self.offsets is None else self.offsets[low:low + step], num_dims=self.num_dims, group=self.group)
        out[low:low + step] = part.unpack().double().square_().sum(1)
      if torch.cuda.is_current_stream_capturing():
        return out
      torch.cuda.current_stream(device).synchronize()
      self._norms = out
    return self._norms

  def search_knn(self, queries, topk, dist_type="dot"):
    """The topk (up to 256) nearest of all rows: (ids int32, or int64 labels, distances float32, found int32), nearest first and of
    equal ones the lower row first, as CuHNSW.search_knn's: -<q, row> for "dot", squared distances for "l2" (|q|^2 + |row|^2 - 2 <q, row>, of
    which the last two are formed in 32 bits: a distance that is small beside the lengths is as exact as these)."""
    _check(dist_type in ("dot", "l2"), "dist_type is dot or l2, not %s", dist_type)
    _tensor(queries, "queries")
    q = queries if queries.dim() == 2 else queries[None]
    _check(q.dim() == 2 and q.shape[1] == self.num_dims, "queries have the shape [num_queries, %d]", self.num_dims)
    _check(isinstance(topk, int) and 0 < topk <= 256, "topk is between 1 and 256")
    _same_device(self.codes, q)
    if self.num_rows == 0:
      return (q.new_full((q.shape[0], topk), -1, dtype=torch.int32 if self.labels is None else torch.int64),
              q.new_full((q.shape[0], topk), float("inf"), dtype=torch.float32), q.new_zeros(q.shape[0], dtype=torch.int32))
    l2 = dist_type == "l2"
    bias = -self.norms() if l2 else None
    lengths = q.double().square().sum(1, keepdim=True) if l2 else None
    step = max(1, min(1 << 22, (1 << 30) // self.num_rows))  # (scores of at most 4 GiB at a time, and queries that one product takes)
    found = []
    for low in range(0, max(1, q.shape[0]), step):
      part = self.scores(q[low:low + step], alpha=2.0 if l2 else 1.0, bias=bias, dtype=torch.float32)
      found.append(select_beams(part[:, None, :], None, topk, normalise=False))
    best, _, ids = (torch.cat(x) for x in zip(*found)) if len(found) > 1 else found[0]
    there = ids >= 0
    distances = (lengths - best.double()).clamp_min(0.0).float() if l2 else -best
    distances = torch.where(there, distances, float("inf"))
    if self.labels is not None:
      ids = torch.where(there, self.labels[ids.clamp_min(0).long()], -1)
    return ids, distances, there.sum(1, dtype=torch.int32)


def _empty_packed(num_rows, num_dims, group, offsets, scale_dtype, device):
  _check(group in _GROUPS, "the group is 32, 64 or 128 elements")
  _check(scale_dtype in _SCALES, "scales are float16 or bfloat16")
  groups = -(-num_dims // group)
  codes = torch.empty(num_rows, 16 * -(-num_dims // 32), dtype=torch.uint8, device=device)
  scales = torch.empty(num_rows, groups, dtype=scale_dtype, device=device)
  return codes, scales, torch.empty_like(scales) if offsets else None


def pack(vectors, group=32, offsets=False, scale_dtype=torch.float16, labels=None):
  """The nearest PackedRows of finite vectors [rows, dims] (float32, float16 or bfloat16): per group scale = largest magnitude
  / 7, or with offsets (for vectors that are not centred) scale = span / 15 and offset = the smallest."""
  _tensor(vectors, "vectors", 2)
  _check(vectors.shape[1] > 0, "the vectors are empty")
  stride = _rows(vectors, "vectors")
  _check(group in _GROUPS, "the group is 32, 64 or 128 elements")
  _check(scale_dtype in _SCALES, "scales are float16 or bfloat16")
  device = _same_device(vectors)
  n, d = vectors.shape
  codes, scales, lows = _empty_packed(n, d, group, offsets, scale_dtype, vectors.device)
  _native.pack_rows(vectors.data_ptr(), _TYPES[vectors.dtype], stride, n, d, group, codes.data_ptr(), scales.data_ptr(), _address(lows),
                    _SCALES[scale_dtype], device, _raw_stream(device))
  return PackedRows(codes, scales, lows, num_dims=d, group=group, labels=labels)


def pack_index(index, group=32, offsets=False, scale_dtype=torch.float16):
  """PackedRows of the vectors that a CuHNSW index holds (CuHNSW.pack_rows).  Rows of a loaded index keep its labels; an index
  with deleted elements is refused, since its rows are all returned here."""
  obj = index.obj

  def refuse_deleted(count):
    if count > 0:
      raise RuntimeError("pack_rows: the index holds deleted elements")

  refuse_deleted(obj.num_deleted())
  n, d = obj.num_data(), obj.num_dims()
  _check(n > 0, "pack_rows: no vectors (call set_data or load_index first)")
  _check(torch.cuda.is_available(), "no HIP device available: this call needs a GPU")
  device = torch.device("cuda", torch.cuda.current_device())
  codes, scales, lows = _empty_packed(n, d, group, offsets, scale_dtype, device)
  # (one call, so that all of it is of one index: another thread may replace it, and where the sizes differ the call fails)
  labels, deleted = obj.pack_items(n, d, group, codes.data_ptr(), scales.data_ptr(), _address(lows), _SCALES[scale_dtype],
                                   _raw_stream(device.index))
  refuse_deleted(deleted)
  plain = np.array_equal(labels, np.arange(n))
  return PackedRows(codes, scales, lows, num_dims=d, group=group, labels=None if plain else torch.from_numpy(labels).to(device))


# ------------------------------------------------------------------------------------------------- selection
def select_beams(scores, beams, num, normalise=True, finished=None, end=None):
  """The `num` (1 to 256) best candidates of every batch entry over its beams and the vocabulary: (totals float32, parents
  int32, tokens int32), each [batch, num], best first.

  scores: [batch, beams, values], float32, float16 or bfloat16; beams: float32 [batch, beams], what the beams have gathered, or
  None (zeros).  A candidate's total is beams + scores, with normalise beams + log_softmax(scores); totals are compared in 64
  bits, equal ones go to the lower beam, then the larger score, then the lower token.  Masked places hold -infinity (a NaN counts as
  one): they are never chosen, and where too few candidates are left the rest says -infinity, -1, -1.  With normalise, where a
  score is +infinity (and log_softmax is a NaN) only the beam's n infinite ones are candidates, each with total beams - log(n).
  finished: bool [batch, beams] or None: a finished beam has one candidate, token `end`, with what it gathered.

  A beam's own candidates stand in the order of their scores; log_softmax is good to about 2^-20, and candidates of different
  beams that are nearer to each other may stand in either order.  The same call gives the same answer to the last bit; how a
  row's sum of exponentials is split depends on the sizes, so that a row's totals can differ in their last bits between batches
  of different sizes."""
  _tensor(scores, "scores", 3)
  _check(isinstance(num, int) and 0 < num <= 256, "num is between 1 and 256")
  b, k, v = scores.shape
  _check(k > 0 and v > 0, "there are no beams or no values")
  _check(k <= 1024, "%d beams: at most 1024", k)
  _check(k * min(num, v) <= 4096, "%d beams and %d candidates: at most 4096 together", k, num)
  _check(v == 1 or scores.stride(2) == 1, "the values of one beam have to be contiguous")
  if beams is not None:
    _tensor(beams, "beams", 2, (torch.float32,))
    _check(tuple(beams.shape) == (b, k), "beams have the shape (%d, %d)", b, k)
  if finished is not None:
    _tensor(finished, "finished", 2, (torch.bool,))
    _check(tuple(finished.shape) == (b, k), "finished has the shape (%d, %d)", b, k)
    _check(beams is not None, "finished beams need what they gathered (beams)")
    _check(isinstance(end, int) and 0 <= end < v, "finished beams need the token that ends a sequence (end)")
  device = _same_device(scores, beams, finished)
  beams = None if beams is None else beams.contiguous()
  finished = None if finished is None else finished.contiguous()
  totals = scores.new_empty((b, num), dtype=torch.float32)
  parents = scores.new_empty((b, num), dtype=torch.int32)
  tokens = scores.new_empty((b, num), dtype=torch.int32)
  kind = _TYPES[scores.dtype]
  size = _native.select_beams_workspace(kind, b, k, v, num)
  work = _workspace(size, scores)
  _native.select_beams(scores.data_ptr(), kind, scores.stride(0), scores.stride(1), b, k, v, _address(beams), _address(finished),
                       0 if end is None else end, int(bool(normalise)), num, totals.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                       _address(work), size, device, _raw_stream(device))
  return totals, parents, tokens


def reorder_states(states, parents):
  """What the beams remember, in their new order: for every tensor [batch, beams, ...] of states a new one [batch, picked, ...]
  whose entry [b][j] is the old one's [b][parents[b][j]], zeros where that is outside [0, beams).

  states: a list of tensors of any type, one beam's state contiguous; parents: int32 [batch, picked] (select_beams')."""
  _tensor(parents, "parents", 2, (torch.int32,))
  if isinstance(states, torch.Tensor):
    raise TypeError("states is a list of tensors")
  states = list(states)
  if not states:
    return []
  b, picked = parents.shape
  k = states[0].shape[1] if isinstance(states[0], torch.Tensor) and states[0].dim() >= 2 else 0
  outs, sizes, strides_b, strides_k = [], [], [], []
  for x in states:
    if not isinstance(x, torch.Tensor):
      raise TypeError("states is a list of tensors")
    _check(not (x.is_neg() or x.is_conj()), "a state is a view that is still to be negated or conjugated (resolve_neg, resolve_conj)")
    shape, stride, size = x.shape, x.stride(), x.element_size()
    _check(len(shape) >= 2 and shape[0] == b and shape[1] == k and k > 0, "states have the shape [batch, beams, ...]: %s with %d batch entries",
           tuple(shape), b)
    expected, empty = 1, x.numel() == 0
    for i in range(len(shape) - 1, 1, -1):
      _check(empty or shape[i] == 1 or stride[i] == expected, "one beam's state has to be contiguous")
      expected *= shape[i]
    sizes.append(expected * size)
    strides_b.append(stride[0] * size)
    strides_k.append(stride[1] * size)
  _check(b * picked <= 65535, "at most 65535 states in all")
  device = _same_device(parents, *states)
  outs = [x.new_empty((b, picked, *x.shape[2:])) for x in states]
  _native.reorder_states([x.data_ptr() for x in states], [x.data_ptr() for x in outs], strides_b, strides_k, sizes, parents.data_ptr(),
                         parents.stride(0), parents.stride(1), b, k, picked, device, _raw_stream(device))
  return outs
