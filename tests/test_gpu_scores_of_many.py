"""Products with rows in 4 bits by the kernel for many queries, on the GPU, against plain statements in 64 bits.

Every test says which kernel its call goes to: a rule that changes cannot empty it."""
import ctypes

import pytest
import torch

from rows_reference import HALF32, stored

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# rows and queries that this kernel takes (384 pairs or more of 128 rows and 16 queries): two, three and four tiles of queries at a time
SIZES = [(24_577, 17), (16_385, 33), (12_801, 64)]
TILES = {17: 2, 33: 3, 64: 4}


def _plan(n, d, group, dtype, nq):
  """(tiles of queries at a time or 0, blocks of them, wavefronts that share a row, laid out by the workgroups)"""
  from cuhnsw_amd import capi
  out = (ctypes.c_int * 4)()
  assert capi.load().cuhnsw_packed_scores_plan(n, d, group, TYPES.index(dtype), nq, out) == 0
  return tuple(out)


def _rows(n, d, group, offsets, scale_type=torch.float16, seed=0, size=1.0):
  """Random codes, all sixteen of them, with scales and offsets of mixed sizes; the places behind the last element hold anything."""
  from cuhnsw_amd import rows
  g = torch.Generator(device="cuda").manual_seed(seed)
  groups = -(-d // group)
  codes = torch.randint(0, 256, (n, 16 * -(-d // 32)), generator=g, device="cuda", dtype=torch.uint8)
  scales = ((torch.rand(n, groups, generator=g, device="cuda") * 0.1 + 0.001) * size).to(scale_type)
  lows = (torch.randn(n, groups, generator=g, device="cuda") * 0.3 * size).to(scale_type) if offsets else None
  return rows.PackedRows(codes, scales, lows, num_dims=d, group=group)


def _queries(nq, d, dtype=torch.float32, seed=1):
  return torch.randn(nq, d, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _terms(packed):
  """(code term, offset term) of the rows in 64 bits, whose sum they are."""
  k = torch.arange(packed.num_dims, device="cuda")
  c = ((packed.codes[:, k // 2] >> (4 * (k % 2)).to(torch.uint8)) & 15).double()
  scales = packed.scales.double()[:, k // packed.group]
  if packed.offsets is None:
    return (c - 8.0) * scales, torch.zeros_like(scales)
  return c * scales, packed.offsets.double()[:, k // packed.group]


def _want(packed, terms, q, alpha, bias):
  """(scores, bound): as rows_reference.scores, on the GPU.  Every product and every addition of a sum in 32 bits over d elements,
  their groups and what surrounds them, 2^-24 each of the sum of magnitudes; the queries' own representation, 2^-22 relative (in
  the 16 steps) and 2^-38 of the query's largest element."""
  a, b = terms
  x, size = q.double(), a.abs() + b.abs()
  y = alpha * (x @ (a + b).t().contiguous())
  bound = abs(alpha) * (x.abs() @ size.t().contiguous())
  most = abs(alpha) * x.abs().amax(1, keepdim=True) * size.sum(1)[None]
  if bias is not None:
    y, bound = y + bias.double(), bound + bias.double().abs()
  steps = packed.num_dims - (-packed.num_dims // packed.group) + 16
  return y, steps * HALF32 * bound * 1.001 + most * 2.0 ** -38


def _check(packed, terms, q, alpha=1.0, bias=None, dtype=None):
  got = packed.scores(q, alpha=alpha, bias=bias, dtype=dtype)
  want, bound = _want(packed, terms, q, alpha, bias)
  assert got.shape == want.shape and got.dtype == (dtype or q.dtype)
  off = (got.double() - want).abs()
  assert (off <= bound + stored(want.abs() + bound, got.dtype)).all(), float((off - bound).max())
  return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("n, nq", SIZES)
def test_scores_of_many(n, nq, offsets, group, dtype):
  """Rows of one to 32 units of 32 elements: less than a chunk, a chunk, several with and without a rest, groups that end inside one."""
  bias = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
  for d in (20, 33, 64, 96, 101, 130, 200, 960, 1024):
    print("many", n, d, nq, group, offsets, dtype, flush=True)
    assert _plan(n, d, group, dtype, nq)[0] == TILES[nq]
    packed, q = _rows(n, d, group, offsets, seed=d), _queries(nq, d, dtype, seed=d)
    terms = _terms(packed)
    plain = _check(packed, terms, q)
    _check(packed, terms, q, alpha=-1.75, bias=bias)
    wide = _check(packed, terms, q, dtype=torch.float32)
    assert torch.equal(wide.to(dtype), plain)      # (a sum in 32 bits, rounded once)
    assert torch.equal(packed.scores(q), plain)    # (and the same bits again)


@pytest.mark.parametrize("n, nq, plan", [(3000, 300, (4, 1)), (20_011, 130, (3, 1)), (100_001, 97, (4, 2)), (40_001, 250, (4, 2)), (50_001, 400, (4, 7)),
                                         (2000, 3000, (4, 3)), (12_800, 79, (3, 1)), (12_927, 80, (3, 1))])
@pytest.mark.parametrize("d, group, offsets, dtype", [(96, 32, True, torch.float32), (96, 64, False, torch.bfloat16), (200, 32, True, torch.float16),
                                                      (210, 128, True, torch.bfloat16), (50, 32, True, torch.float32)])
def test_blocks_of_queries_one_after_the_other(n, nq, plan, d, group, offsets, dtype):
  """Workgroups that go from one block of queries to the next, the last of which has fewer tiles, and a last tile that is not full."""
  print("blocks", n, nq, d, group, offsets, dtype, flush=True)
  assert _plan(n, d, group, dtype, nq)[:2] == plan
  packed, q = _rows(n, d, group, offsets), _queries(nq, d, dtype)
  _check(packed, _terms(packed), q, alpha=2.0, bias=torch.randn(n, device="cuda"), dtype=torch.float32)


@pytest.mark.parametrize("n, nq", SIZES)
@pytest.mark.parametrize("d, group", [(70, 32), (300, 64)])
def test_bfloat16_scales_and_strided_queries(n, nq, d, group):
  assert _plan(n, d, group, torch.float32, nq)[0] == TILES[nq]
  packed = _rows(n, d, group, True, torch.bfloat16, size=1e6)
  terms = _terms(packed)
  base = _queries(nq, 2 * d + 23)
  _check(packed, terms, base[:, 5:5 + d])                       # (rows that begin at any address)
  _check(packed, terms, base.bfloat16()[:, 3:3 + d])
  _check(packed, terms, _queries(1, d).expand(nq, d))
  assert torch.equal(packed.scores(base[:, 5:5 + d]), packed.scores(base[:, 5:5 + d].contiguous()))


@pytest.mark.parametrize("dtype, out_type", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                             (torch.float16, torch.float32)])
@pytest.mark.parametrize("n, nq, wider", [(24_577, 17, 37), (16_385, 33, 1), (12_801, 64, 0), (12_863, 61, 129), (12_927, 50, 2)])
def test_scores_are_written_where_they_belong_and_nowhere_else(n, nq, wider, dtype, out_type):
  from cuhnsw_amd import cuhnsw_bind
  d, group = 130, 32
  assert _plan(n, d, group, dtype, nq)[0] > 0
  packed, q = _rows(n, d, group, True), _queries(nq, d, dtype)
  want = packed.scores(q, dtype=out_type)
  out = torch.full((nq + 2, n + wider), 7.0, device="cuda", dtype=out_type)
  size = cuhnsw_bind.packed_scores_workspace(n, d, group, TYPES.index(dtype), nq)
  work = torch.full((size + 256,), 77, dtype=torch.uint8, device="cuda")
  cuhnsw_bind.packed_scores(packed.codes.data_ptr(), packed.scales.data_ptr(), packed.offsets.data_ptr(), 1, n, d, group, q.data_ptr(),
                            TYPES.index(dtype), d, nq, 1.0, 0, out[1].data_ptr(), TYPES.index(out_type), n + wider, work.data_ptr(), size, 0,
                            torch.cuda.current_stream().cuda_stream)
  assert torch.equal(out[1:-1, :n], want)
  assert (out[0] == 7).all() and (out[-1] == 7).all() and (out[1:-1, n:] == 7).all() and (work[size:] == 77).all()


@pytest.mark.parametrize("n, nq", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_queries_that_are_tiny_large_or_zero(n, nq, dtype):
  d, group = 130, 64
  assert _plan(n, d, group, dtype, nq)[0] == TILES[nq]
  packed, q = _rows(n, d, group, True), _queries(nq, d)
  sizes = (1.0, 1e-3, 1e3, 0.0) if dtype == torch.float16 else (1e-37, 1e-30, 1e30, 1.0, 0.0)
  q *= torch.tensor([sizes[i % len(sizes)] for i in range(nq)], device="cuda")[:, None]
  _check(packed, _terms(packed), q.to(dtype), dtype=torch.float32)


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("n, nq", SIZES)
def test_in_a_graph_and_on_another_stream(n, nq, offsets):
  d = 200
  assert _plan(n, d, 32, torch.bfloat16, nq)[0] == TILES[nq]
  packed, q = _rows(n, d, 32, offsets), _queries(nq, d, torch.bfloat16)
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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("n, d, nq, split", [(300, 200, 40, 2), (500, 300, 3, 4), (200, 500, 5, 4), (70_000, 700, 1, 4), (100_001, 300, 2, 4), (9001, 520, 37, 8)])
def test_few_queries_whose_rows_are_shared(n, d, nq, split, offsets, dtype):
  """The other kernel, with two, four and eight wavefronts that share the elements of a row, the last of which may have none."""
  print("few", n, d, nq, offsets, dtype, flush=True)
  for group in (32, 128):
    assert _plan(n, d, group, dtype, nq) == (0, 1, split, int(nq <= 2))
    packed, q = _rows(n, d, group, offsets), _queries(nq, d, dtype)
    terms = _terms(packed)
    plain = _check(packed, terms, q)
    _check(packed, terms, q, alpha=-1.75, bias=torch.randn(n, device="cuda"), dtype=torch.float32)
    assert torch.equal(packed.scores(q, dtype=torch.float32).to(dtype), plain)
    assert torch.equal(packed.scores(q), plain)


@pytest.mark.parametrize("n, nq", SIZES)
@pytest.mark.parametrize("d, group", [(20, 32), (96, 32), (130, 64), (200, 32), (300, 128), (960, 32), (1024, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_query_that_is_not_finite_spoils_no_other(n, nq, d, group, dtype):
  """The last query of a tile holds it, in the row's last group: what stands behind that group, in a chunk that it does not
  fill, is nobody's."""
  print("not finite", n, nq, d, group, dtype, flush=True)
  assert _plan(n, d, group, dtype, nq)[0] == TILES[nq]
  for offsets in (False, True):
    packed, q = _rows(n, d, group, offsets), _queries(nq, d, dtype)
    clean = packed.scores(q)
    assert torch.isfinite(clean).all()
    others = torch.arange(nq, device="cuda") != 15
    for value in (float("inf"), float("nan")):
      spoilt = q.clone()
      spoilt[15, d - 1] = value
      got = packed.scores(spoilt)
      assert not torch.isfinite(got[15]).any()
      assert torch.equal(got[others], clean[others])
