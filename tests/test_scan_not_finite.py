"""selective_scan of values that are not finite, and of decay factors that pass the largest float32."""
import math

import pytest
import torch

from tests.test_state_space import scan_case, scan_definition, within

DTYPES = [torch.float32, torch.bfloat16]


def same_kind(got, want):
  """NaN where the definition has NaN, the same infinity where it has one, a number elsewhere."""
  got = got.double()
  assert torch.equal(got.isnan(), want.isnan())
  assert torch.equal(torch.where(got.isinf(), got, 0.0), torch.where(want.isinf(), want, 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,n", [(2, 1, 1), (2, 1, 12), (70, 1, 3), (70, 1, 12), (70, 1, 13), (2, 1, 200), (2, 3, 1), (2, 40, 3),
                                   (2, 40, 12), (2, 40, 21), (2, 40, 50), (1, 40, 100), (1, 20, 200), (2, 40, 16)])
def test_infinite_inputs(b, t, n, dtype):
  """An infinite x or dt, and NaN, in channels of their own: the states are what the definition has, outputs are finite where
  it has finite ones (and then those), for numbers of states that no register or lane count divides, too."""
  import recurrentgemma_b200 as rg
  e = 2560 if b > 8 else 40
  case = scan_case(n + t, b, t, e, n, dtype)
  # one sign of b, c and d, so that infinite terms sum to an infinite output in any order
  case["b"], case["c"], case["d"] = (case[k].abs() + 0.125 for k in ("b", "c", "d"))
  at = t // 2
  case["x"][0, at, 1], case["x"][0, at, 2] = math.inf, -math.inf
  case["dt"][0, at, 5], case["dt"][0, at, 6], case["x"][0, at, 7], case["dt"][0, at, 9] = (
      math.inf, -math.inf, math.nan, math.nan)
  case["z"][..., :12] = case["z"][..., :12].abs() + 0.125
  y, state = rg.selective_scan(**case)
  want, held, bound, bound_state = scan_definition(**case)
  assert want[0, at, 1] == math.inf and want.isnan().any()
  assert torch.equal(y.isfinite(), want.isfinite())
  same_kind(state, held)
  fine, fine_state = want.isfinite(), held.isfinite()
  within(torch.where(fine, y, 0.0), torch.where(fine, want, 0.0), torch.where(fine, bound, 0.0), dtype)
  within(torch.where(fine_state, state, 0.0), torch.where(fine_state, held, 0.0), torch.where(fine_state, bound_state, 0.0),
         torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,n", [(2, 1, 16), (2, 1, 5), (70, 1, 16), (2, 40, 16), (2, 40, 3), (1, 40, 21)])
@pytest.mark.parametrize("state", [False, True])
def test_a_decay_without_end_in_front_of_nothing(b, t, n, state, dtype):
  """A factor of e^100 on the first token of a document, or of a call without a state, has nothing to multiply."""
  import recurrentgemma_b200 as rg
  e = 2560 if b > 8 else 40
  case = scan_case(n + t, b, t, e, n, dtype, state=state, bias=False)
  case["dt"] = case["dt"].abs() * 0.01
  case["dt"][:, ::7] = 100.0
  case["a"][:] = 1.0
  if state or t > 1:
    case["segment_pos"] = (torch.arange(t, device="cuda") % 7).int().repeat(b, 1)
  y, state = rg.selective_scan(**case, softplus=False)
  want, held, bound, bound_state = scan_definition(**case, softplus=False)
  within(y, want, bound, dtype)
  within(state, held, bound_state, torch.float32)
