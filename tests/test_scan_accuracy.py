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


def off(got, want):
  """Relative to 64 bits, in the 2-norm."""
  return ((got.double() - want).norm() / want.norm()).item()


def off_each(got, want):
  """Relative to each value in 64 bits, root mean square; what is 0 there is 0."""
  assert (got[want == 0] == 0).all()
  return torch.where(want == 0, 0.0, (got.double() - want) / want).square().mean().sqrt().item()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [2, 33])
def test_steps_in_float32(t):
  """Steps softplus(dt) of 1e-4 to 0.3, seen in states that forget all else: the exponential (0.45 u rms), the logarithm
  (0.7 u) and two products (0.42 u each) make 1.0 u; half as much again is allowed."""
  import recurrentgemma_b200 as rg
  g = torch.Generator(device="cuda").manual_seed(t)
  e, n = 2560, 16
  dt = -1.0 - 8.0 * torch.rand((1, t, e), generator=g, device="cuda")
  x = torch.randn((1, t, e), generator=g, device="cuda")
  b, c = (torch.randn((1, t, 1, n), generator=g, device="cuda") for _ in range(2))
  a = torch.full((e, n), -1e7, device="cuda")
  got = rg.selective_scan(x, dt, a, b, c)[1]
  want = (torch.log1p(torch.exp(dt[:, -1].double())) * x[:, -1].double())[:, :, None] * b[:, -1].double()
  assert off_each(got, want) <= 1.5 * U


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 16, 21])
def test_decay_factors_in_float32(n):
  """States whose decay factors are 1/2 to 1.  A term of k steps ago has passed k factors and k multiply-adds, and weighs
  with the square of its decay: 1.4 steps on average.  So of the squares of the errors (rms, in u) 1.4 times a factor's
  (0.45 the exponential, 0.2 each the argument and the rate times log2(e)) and a multiply-add's (0.42), and once those of the
  two products that a term is (0.42): 1.0 u in all.  A fifth more is allowed."""
  import recurrentgemma_b200 as rg
  g = torch.Generator(device="cuda").manual_seed(n)
  t, e = 40, 2560
  dt = math.log(2.0) * torch.rand((1, t, e), generator=g, device="cuda")
  x = torch.randn((1, t, e), generator=g, device="cuda")
  b = torch.randn((1, t, 1, n), generator=g, device="cuda")
  a = torch.full((e, n), -1.0, device="cuda")
  got = rg.selective_scan(x, dt, a, b, b, softplus=False)[1]
  want = torch.zeros((1, e, n), dtype=torch.float64, device="cuda")
  for i in range(t):
    step = dt[:, i].double()
    want = torch.exp(-step)[:, :, None] * want + (step * x[:, i].double())[:, :, None] * b[:, i].double()
  assert off(got, want) <= 1.2 * U


def layer(seed, b, t, e, n, dtype, gate=True):
  """Steps of 1e-3 to 1e-1, decay rates of about 1 to n, as trained layers have them."""
  g = torch.Generator(device="cuda").manual_seed(seed)
  normal = lambda *s: torch.randn(s, generator=g, device="cuda")                 # noqa: E731
  step = torch.exp(torch.rand(e, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
  return dict(x=normal(b, t, e).to(dtype), dt=(0.5 * normal(b, t, e)).to(dtype),
              a=-(torch.arange(1, n + 1, device="cuda") * torch.exp(0.2 * normal(e, n))),
              b=normal(b, t, 1, n).to(dtype), c=normal(b, t, 1, n).to(dtype), d=0.5 * normal(e),
              z=normal(b, t, e).to(dtype) if gate else None, dt_bias=step + torch.log(-torch.expm1(-step)))


def token_by_token(case, dtype):
  """The formula in `dtype`, a token after the other: (y, state)."""
  x, dt, a, b, c, d, z, bias = (None if case[k] is None else case[k].to(dtype)
                                for k in ("x", "dt", "a", "b", "c", "d", "z", "dt_bias"))
  step = dt + bias
  step = torch.where(step > 0, step, 0.0) + torch.log1p(torch.exp(-step.abs()))
  h = x.new_zeros(x.shape[0], *a.shape)
  y = torch.empty_like(x)
  for i in range(x.shape[1]):
    now = step[:, i, :, None]
    h = torch.exp(now * a) * h + now * x[:, i, :, None] * b[:, i]
    y[:, i] = (h * c[:, i]).sum(-1) + d * x[:, i]
  return (y if z is None else y * (z / (1.0 + torch.exp(-z)))), h


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 8, 16, 21, 48])
@pytest.mark.parametrize("gate", [True, False])
def test_sequences_in_float32_are_as_exact_as_the_formula(n, gate):
  """No further from 64 bits, outputs and states, than the formula in float32 with its library's functions."""
  import recurrentgemma_b200 as rg
  case = layer(n, 2, 700, 320, n, torch.float32, gate)
  want, plain = token_by_token(case, torch.float64), token_by_token(case, torch.float32)
  got = rg.selective_scan(**case)
  for k, p, w in zip(got, plain, want):
    assert off(k, w) <= off(p, w)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 4])
def test_states_of_bfloat16_sequences(n):
  """Up to 4 states are as exact as the formula in float32 makes them of the same bfloat16 inputs."""
  import recurrentgemma_b200 as rg
  case = layer(n, 2, 700, 320, n, torch.bfloat16)
  want, plain = token_by_token(case, torch.float64), token_by_token(case, torch.float32)
  assert off(rg.selective_scan(**case)[1], want[1]) <= off(plain[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,b,t,e,n", [
    (torch.float32, 2, 700, 320, 1), (torch.float32, 2, 700, 320, 16), (torch.float32, 2, 700, 320, 21),
    (torch.float32, 1, 300, 40, 200), (torch.bfloat16, 2, 700, 320, 3), (torch.bfloat16, 2, 700, 320, 4),
    (torch.float32, 64, 60, 5120, 16), (torch.bfloat16, 300, 60, 5120, 4)])         # (many sequences a thread)
def test_single_steps_are_as_exact_as_the_formula(dtype, b, t, e, n):
  """Steps that overwrite their state, one after the other: states no further from 64 bits than the formula in float32; the
  same rule as for a sequence in one call.  Float32 outputs within a tenth of that: sums of 200 states are eight products
  in turn (a rounding of the i-th counts i/8 of one of the whole sum: 4.5 in all) joined five times, 9.5 roundings of the
  sum's size where the formula's sum by halves has 8, and the square root of 9.5/8 is 1.09."""
  import recurrentgemma_b200 as rg
  case = layer(n + t, b, t, e, n, dtype)
  want, plain = token_by_token(case, torch.float64), token_by_token(case, torch.float32)
  state, y = torch.zeros(b, e, n, device="cuda"), torch.empty_like(case["x"])
  for i in range(t):
    now = {k: v[:, i:i + 1] if k in ("x", "dt", "b", "c", "z") else v for k, v in case.items()}
    y[:, i:i + 1] = rg.selective_scan(**now, state=state, inplace=True)[0]
  assert off(state, want[1]) <= off(plain[1], want[1])
  if dtype == torch.float32:
    assert off(y, want[0]) <= 1.1 * off(plain[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("b,t", [(1, 1), (64, 1), (2, 35)])
def test_gate_in_float32(b, t):
  """y = d x silu(z) of z from -20 to 20: five roundings (0.42 u rms each) and an exponential of 0.5 u make 1.1 u, half as
  much again is allowed; gates of 0, of 200 either way, infinite ones and NaN give what the formula gives."""
  import recurrentgemma_b200 as rg
  e, n = 5120, 16
  case = layer(b + t, b, t, e, n, torch.float32)
  g = torch.Generator(device="cuda").manual_seed(b + t)
  case["z"] = 40.0 * torch.rand(case["x"].shape, generator=g, device="cuda") - 20.0
  case["c"] = torch.zeros_like(case["c"])
  z = case["z"].double()
  got = rg.selective_scan(**case)[0]
  assert off_each(got, case["d"].double() * case["x"].double() * z / (1.0 + torch.exp(-z))) <= 1.6 * U
  case["z"][..., :6] = torch.tensor([0.0, -200.0, 200.0, math.inf, -math.inf, math.nan], device="cuda")
  got = rg.selective_scan(**case)[0][..., :6]
  want = (case["d"] * case["x"] * (case["z"] / (1.0 + torch.exp(-case["z"]))))[..., :6]
  assert torch.equal(got.isnan(), want.isnan()) and torch.allclose(got.nan_to_num(), want.nan_to_num(), rtol=1e-6, atol=1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("lo,hi", [(1e-5, 1e-4), (1e-4, 1e-3), (1e-3, 1e-2), (1e-2, 1e-1)])
def test_slow_states_of_bfloat16_calls(lo, hi, single):
  """1000 steps of states with decay rates of lo to hi a step, in bfloat16, where the factors are the hardware's.  Up to 1e-2
  no further off than the formula in float32.  Beyond, the mean error of a factor (13e-9 at most) counts as often as a term
  is old, 1 / (2 lo) steps, and its random part with the multiply-add's (0.69 u) by the root of that: 6.5e-7 and 2.9e-7."""
  import recurrentgemma_b200 as rg
  t, e, n = 1000, 320, 16
  g = torch.Generator(device="cuda").manual_seed(3)
  case = layer(4, 1, t, e, n, torch.bfloat16, False)
  case["dt"] = (0.5 + torch.rand((1, t, e), generator=g, device="cuda")).bfloat16()
  case["a"] = -torch.exp(torch.rand((e, n), generator=g, device="cuda") * math.log(hi / lo) + math.log(lo))
  state = torch.randn((1, e, n), generator=g, device="cuda")

  def formula(dtype):
    h, (x, dt, a, b) = state.to(dtype), (case[k].to(dtype) for k in ("x", "dt", "a", "b"))
    for i in range(t):
      h = torch.exp(dt[:, i, :, None] * a) * h + (dt[:, i] * x[:, i])[:, :, None] * b[:, i]
    return h
  want, plain, got = formula(torch.float64), formula(torch.float32), state.clone()
  for i in range(0, t, 1 if single else t):
    part = {k: case[k][:, i:i + 1] if single else case[k] for k in ("x", "dt", "b", "c")}
    rg.selective_scan(**part, a=case["a"], state=got, softplus=False, inplace=True)
  assert off(got, want) <= (off(plain, want) if hi <= 1e-2 else math.hypot(6.5e-7, 2.9e-7))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [3, 16, 21])
def test_steps_of_no_time_leave_the_states(n, dtype):
  """A step of 0, given or as softplus of -infinity, is a factor of exactly 1 and puts nothing in."""
  import recurrentgemma_b200 as rg
  for t in (1, 45):
    case = layer(n, 70, t, 640, n, dtype)
    state = torch.randn((70, 640, n), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda")
    for dt, softplus in ((0.0, False), (-math.inf, True)):
      case["dt"] = torch.full_like(case["dt"], dt)
      given = {**case, "dt_bias": None} if not softplus else case
      assert torch.equal(rg.selective_scan(**given, state=state, softplus=softplus)[1], state)
