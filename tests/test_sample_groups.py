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
