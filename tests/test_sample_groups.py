"""sample with top_k up to 128, which looks for the first k among what the k-th largest maximum of parts of the row bounds:
vocabularies whose parts do not come out even, and rows with fewer tokens than that."""
import math

import pytest
import torch

from tests.test_sample import definition, rows

SIZES = [1, 3, 63, 64, 65, 127, 128, 129, 255, 257, 300, 509, 511, 513, 1021, 2047, 2049, 3000, 4097, 8193, 11000, 16385, 32768,
         33000, 50257, 65537, 128256, 151936, 256000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", SIZES)
def test_first_tokens_of_every_vocabulary(v, dtype):
  """Every k around the number of parts, one row and several, with ties in bfloat16."""
  import recurrentgemma_b200 as rg
  logits, _, g = rows(v, 40, v, dtype)
  for k in (1, 2, 50, 63, 64, 65, 100, 125, 126, 127, 128, 129):
    u = torch.rand((40,), generator=g, device="cuda")
    got = rg.sample(logits, u, top_k=k, top_p=0.99, temperature=3.0)
    some = torch.tensor([0, 17, 39], device="cuda")
    assert torch.equal(got[some], definition(logits[some], u[some], top_k=k, top_p=0.99, temperature=3.0)), k
    assert torch.equal(rg.sample(logits[:1], u[:1], top_k=k, top_p=0.99, temperature=3.0), got[:1]), k


@pytest.mark.gpu
@pytest.mark.parametrize("v", [200, 513, 5000, 33000, 256000])
def test_parts_of_a_row_without_a_token(v):
  """Rows of -inf and NaN but for a few places, side by side or far apart, at the ends too."""
  import recurrentgemma_b200 as rg
  logits = torch.full((6, v), -math.inf, device="cuda")
  logits[1::2, ::3] = math.nan
  g = torch.Generator(device="cuda").manual_seed(v)
  for m, places in enumerate([[v - 1], [0, v - 1], list(range(60)), list(range(v - 70, v)), list(range(0, v, v // 100)),
                              list(range(1, v, v // 140))]):
    logits[m, places] = torch.randn(len(places), generator=g, device="cuda")
  for k in (1, 50, 100, 128):
    for u in (0.0, 0.4, 1.0 - 2.0 ** -24):
      uniforms = torch.full((6,), u, device="cuda")
      assert torch.equal(rg.sample(logits, uniforms, top_k=k), definition(logits, uniforms, top_k=k)), (k, u)


@pytest.mark.gpu
def test_settings_of_rows_below_their_range():
  """Only numbers are refused on the host: in a tensor a top_p below 0 keeps one token, a min_p below 0 all, one above 1 the
  largest, a temperature below 0 is greedy and a top_k below 0 keeps all."""
  import recurrentgemma_b200 as rg
  logits, u, _ = rows(7, 6, 5000, torch.float32)
  logits[3] = logits[3].round()                      # (ties at the top)
  logits[4, 7], logits[4, 1900] = math.inf, math.inf
  row = lambda v: torch.full((6,), v, device="cuda")                             # noqa: E731
  best = definition(logits, u, temperature=0.0)
  for k in (0, 50, 3000):
    assert torch.equal(rg.sample(logits, u, top_k=k, top_p=row(-0.5)), best)
    assert torch.equal(rg.sample(logits, u, top_k=k, top_p=row(-math.inf)), best)
  assert torch.equal(rg.sample(logits, u, temperature=row(-1.0)), best)
  every = rg.sample(logits, u)
  assert torch.equal(rg.sample(logits, u, min_p=row(-2.0)), every)
  assert torch.equal(rg.sample(logits, u, top_k=torch.full((6,), -9, dtype=torch.int32, device="cuda")), every)
  assert torch.equal(rg.sample(logits, u, min_p=row(7.0)), rg.sample(logits, u, min_p=1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [31, 5000, 50257])
def test_temperatures_of_any_size(v, dtype):
  import recurrentgemma_b200 as rg
  logits, u, _ = rows(v, 5, v, dtype)
  logits[1, ::2] = torch.finfo(dtype).min
  logits[2, 3], logits[2, 9] = torch.finfo(dtype).max, torch.finfo(dtype).min
  logits[3, ::3] = -math.inf
  logits[4] = logits[4].abs() * -1e-3
  logits[4, 11] = 0.0
  for t in (1e-45, 1e-38, 1e-30, 1e-3, 300.0, 1e30, 3e38, math.inf):
    for settings in ({}, dict(top_k=20), dict(top_p=0.7), dict(top_k=300, top_p=0.9, min_p=0.5)):
      assert torch.equal(rg.sample(logits, u, temperature=t, **settings),
                         definition(logits, u, temperature=t, **settings)), (t, settings)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [1000, 50257, 256000, 2 ** 18 + 5, 2 ** 20])
def test_rounding_of_the_weights(v):
  """Against weights in 64 bits, not rounded to the kernel's: each of the kernel's is within one multiple of 2^-44 (-43, -42)
  of them, so that a sum is within v of those.  Where no border is nearer than that the token is the same.  (v borders twice
  2 v units wide in a sum of some hundred: a row in two hundred at 2^20 tokens, fewer below; one of sixteen may be left out.)"""
  import recurrentgemma_b200 as rg
  unit = 2.0 ** -(44 if v <= 2 ** 18 else 43 if v <= 2 ** 19 else 42)
  logits, u, _ = rows(v, 16, v, torch.float32)
  order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
  sorted_logits = torch.gather(logits, 1, order).double()
  far = 2.0 * v * unit                                # (a border's sum, and the target, which is a share of another sum)
  for t, p in ((1.0, 1.0), (2.5, 1.0), (1.0, 0.9), (0.7, 0.5)):
    share = float(torch.tensor(p, dtype=torch.float32))
    w = torch.exp((sorted_logits - sorted_logits[:, :1]) / float(torch.tensor(t, dtype=torch.float32)))
    upto = torch.cumsum(w, -1)
    sure = torch.ones(16, dtype=torch.bool, device="cuda")
    if p < 1.0:
      target = share * upto[:, -1:]
      sure &= (upto - target).abs().min(-1).values > far
      w = torch.where(upto - w < target, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    upto = torch.cumsum(w, -1)
    target = u.double()[:, None] * upto[:, -1:]
    sure &= (upto - target).abs().min(-1).values > far
    want = (upto <= target).sum(-1).int()
    got = rg.sample(logits, u, temperature=t, top_p=p)
    assert torch.equal(got[sure], want[sure])
    assert sure.sum() >= 15
