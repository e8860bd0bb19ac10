"""Products with rows in 4 bits by the kernel for many queries, on the GPU, against plain statements in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# rows and queries that this kernel takes (384 pairs or more of 128 rows and 16 queries): two, three and four tiles of queries at a time
SIZES = [(24_577, 17), (16_385, 33), (12_801, 64)]


def _rows(n, d, group, offsets, scale_type=torch.float16, seed=0):
  """Random codes, all sixteen of them, with scales and offsets of mixed sizes; the places behind the last element hold anything."""
  from cuhnsw_amd import rows
  g = torch.Generator(device="cuda").manual_seed(seed)
  groups = -(-d // group)
  codes = torch.randint(0, 256, (n, 16 * -(-d // 32)), generator=g, device="cuda", dtype=torch.uint8)
  scales = (torch.rand(n, groups, generator=g, device="cuda") * 0.1 + 0.001).to(scale_type)
  lows = (torch.randn(n, groups, generator=g, device="cuda") * 0.3).to(scale_type) if offsets else None
  return rows.PackedRows(codes, scales, lows, num_dims=d, group=group)


def _queries(nq, d, dtype=torch.float32, seed=1):
  return torch.randn(nq, d, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("n, nq", SIZES)
@pytest.mark.parametrize("d, group", [(20, 32), (96, 32), (130, 64), (200, 32), (300, 128), (960, 32), (1024, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_query_that_is_not_finite_spoils_no_other(n, nq, d, group, dtype):
  """The last query of a tile holds it, in the row's last group: what stands behind that group, in a chunk that it does not
  fill, is nobody's."""
  print("not finite", n, nq, d, group, dtype, flush=True)
  packed, q = _rows(n, d, group, True), _queries(nq, d, dtype)
  clean = packed.scores(q)
  assert torch.isfinite(clean).all()
  others = torch.arange(nq, device="cuda") != 15
  for value in (float("inf"), float("nan")):
    spoilt = q.clone()
    spoilt[15, d - 1] = value
    got = packed.scores(spoilt)
    assert not torch.isfinite(got[15]).any()
    assert torch.equal(got[others], clean[others])
