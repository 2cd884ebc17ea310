"""How near selective_scan comes to its definition in 64 bits, beyond the bounds that hold for every input."""
import math

import pytest
import torch

U = 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n", [(torch.float32, 16), (torch.float32, 3), (torch.bfloat16, 4)])
@pytest.mark.parametrize("t", [1, 2, 40])
def test_growth_up_to_the_largest_float(t, n, dtype):
  """A decay factor of 2^126 to 2^128 is a float32: the state that it multiplies is too.  The argument, up to 88.7, is
  rounded three times (the product with log2(e), that constant, the product with the step), the rest is 8 units."""
  import recurrentgemma_b200 as rg
  e = 16
  x = torch.zeros((1, t, e), dtype=dtype, device="cuda")
  dt = torch.zeros_like(x)
  dt[:, 0] = 1.0
  bc = torch.zeros((1, t, 1, n), dtype=dtype, device="cuda")
  power = torch.linspace(126.0, 127.99, e, device="cuda")
  a = (power * math.log(2.0))[:, None].repeat(1, n)
  state = torch.full((1, e, n), 0.37, device="cuda")
  got = rg.selective_scan(x, dt, a, bc, bc, state=state, softplus=False)[1]
  want = torch.exp(a.double()) * state.double()
  assert (want < torch.finfo(torch.float32).max).all()
  assert torch.isfinite(got).all()
  assert ((got.double() - want).abs() <= (3 * 88.8 + 8) * U * want).all()
