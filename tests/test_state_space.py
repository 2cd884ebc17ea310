"""causal_conv and selective_scan against their definitions in 64 bits, and what they refuse.

Tolerances count roundings.  A float32 operation is off by u = 2^-24 of its value, the hardware exponential by 4 u and
2 u of its argument's size; a bfloat16 output by 2^-8 of itself.

  causal_conv     the sum of W products and a bias: (W + 2) u of the sum of magnitudes; silu moves that by at
                  most 1.1 times it and adds (10 + 2 |v|) u of itself.
  selective_scan  a state's term has passed t steps, each off by 6 u (the exponential, the multiply-add, and
                  the argument's and the step's roundings, which count D |a| times and decay by exp(D |a|)):
                  with the sum over N states, the step (16 u) and silu (10 u + 2 |z| u, |z| below 8) at
                  most (6 T + N + 64) u of the sum of the magnitudes of all terms.
"""
import math

import pytest
import torch

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def half_step(dtype):
  return torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else U


def within(got, want, bound, dtype):
  """Every element of `got` within its bound and one rounding of `want`."""
  assert got.dtype == dtype and got.shape == want.shape
  off = (got.double() - want).abs()
  allowed = bound + half_step(dtype) * (want.abs() + bound) + 1e-37
  assert torch.isfinite(got.double()).all()
  worst = (off / allowed).max().item() if off.numel() else 0.0
  assert worst <= 1.0, f"{worst:.2f} times the bound"


def generator(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def positions(g, b, t, doc, dtype=torch.int64):
  """Documents of random length, some of one token; a row may begin inside one."""
  pos = torch.arange(t, device="cuda").repeat(b, 1)
  starts = torch.rand((b, t), generator=g, device="cuda") < 1.0 / doc
  begin = torch.cummax(torch.where(starts, pos, torch.full_like(pos, -3)), dim=1).values
  return (pos - begin).to(dtype)


# ---- causal_conv ----------------------------------------------------------------------------------
def conv_case(seed, b, t, e, taps, dtype, doc=0, state=True, bias=True, part=False):
  g = generator(seed)
  normal = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)       # noqa: E731
  x = normal(b, t, 2 * e + 1)[..., 1:e + 1] if part else normal(b, t, e)
  pos = positions(g, b, t, doc) if doc else None
  return dict(x=x, w=normal(taps, e), b=normal(e) if bias else None, segment_pos=pos,
              state=normal(b, taps - 1, e) if state else None)


def conv_definition(x, w, b=None, segment_pos=None, state=None, activation="silu"):
  """(y, state, bound) in 64 bits, token by token."""
  (bs, t, e), taps = x.shape, w.shape[0]
  held = x.new_zeros((bs, taps - 1, e), dtype=torch.float64) if state is None else state.double()
  y, bound = (x.new_zeros((bs, t, e), dtype=torch.float64) for _ in range(2))
  for i in range(t):
    if segment_pos is not None:
      held = torch.where((segment_pos[:, i] == 0)[:, None, None], 0.0, held)
    window = torch.cat([held, x[:, i:i + 1].double()], 1)
    terms = window * w.double()
    v = terms.sum(1) + (0.0 if b is None else b.double())
    size = terms.abs().sum(1) + (0.0 if b is None else b.double().abs())
    y[:, i] = v * torch.sigmoid(v) if activation else v
    bound[:, i] = 1.1 * (taps + 2) * U * size + (10 + 2 * v.abs()) * U * y[:, i].abs() * bool(activation)
    held = window[:, 1:]
  return y, held, bound


CONV = [
    # b, t, e, taps, doc, state, bias, part of a wider tensor
    (1, 1, 8, 4, 0, True, True, False),
    (3, 1, 24, 2, 0, True, False, False),
    (2, 1, 33, 3, 0, True, True, True),
    (2, 2, 16, 4, 0, True, True, False),
    (2, 3, 16, 4, 2, True, True, False),
    (1, 5, 7, 4, 0, False, True, False),
    (2, 16, 40, 4, 5, True, True, False),
    (2, 17, 40, 3, 2, True, False, True),
    (3, 67, 130, 2, 4, False, True, False),
    (1, 70, 2560, 4, 9, True, True, False),
    (5, 700, 2560, 4, 40, True, True, False),      # large enough for sixteen rows a thread
    (2, 1000, 5121, 4, 40, True, True, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,e,taps,doc,state,bias,part", CONV)
def test_causal_conv(b, t, e, taps, doc, state, bias, part, dtype):
  import recurrentgemma_b200 as rg
  case = conv_case(t + e, b, t, e, taps, dtype, doc, state, bias, part)
  for activation in ("silu", None):
    y, new = rg.causal_conv(**case, activation=activation)
    want, held, bound = conv_definition(**case, activation=activation)
    within(y, want, bound, dtype)
    assert torch.equal(new.double(), held)
  again, none = rg.causal_conv(**case, activation=None, return_state=False)
  assert none is None and torch.equal(again, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cuts", [(1,) * 9, (0, 3, 1, 5), (2, 7), (8, 1)])
def test_causal_conv_in_chunks(cuts, dtype):
  """A prompt in chunks, the state passed on in place, gives what one call gives."""
  import recurrentgemma_b200 as rg
  case = conv_case(5, 3, sum(cuts), 48, 4, dtype, doc=4)
  y, new = rg.causal_conv(**case)
  state, at, parts = case["state"].clone(), 0, []
  for n in cuts:
    part, back = rg.causal_conv(case["x"][:, at:at + n], case["w"], case["b"],
                                segment_pos=case["segment_pos"][:, at:at + n], state=state, inplace=True)
    assert back is state
    parts.append(part)
    at += n
  assert torch.equal(torch.cat(parts, 1), y) and torch.equal(state, new)


# ---- selective_scan -------------------------------------------------------------------------------
def scan_case(seed, b, t, e, n, dtype, groups=1, doc=0, state=True, z=True, d=True, bias=True, part=False):
  g = generator(seed)
  normal = lambda *s: torch.randn(s, generator=g, device="cuda")                 # noqa: E731
  rows = lambda: (normal(b, t, 3 * e + 2)[..., e + 1:2 * e + 1] if part else normal(b, t, e)).to(dtype)  # noqa: E731
  bc = normal(b, t, 2 * groups * n + 5).to(dtype)[..., 5:] if part else normal(b, t, 2 * groups * n).to(dtype)
  bb, cc = (bc[..., k * groups * n:(k + 1) * groups * n].unflatten(-1, (groups, n)) for k in (0, 1))
  if not part:
    bb, cc = bb.contiguous(), cc.contiguous()
  return dict(x=rows(), dt=rows(), b=bb, c=cc, z=rows() if z else None,
              a=-torch.exp(normal(e, n)), d=normal(e) if d else None,
              dt_bias=normal(e) - 3.0 if bias else None,
              segment_pos=positions(g, b, t, doc, torch.int32) if doc else None,
              state=normal(b, e, n) if state else None)


def scan_definition(x, dt, a, b, c, d=None, z=None, dt_bias=None, segment_pos=None, state=None, softplus=True):
  """(y, state, bound of y, bound of the state) in 64 bits, token by token."""
  bs, t, e = x.shape
  groups, n = b.shape[2:]
  x, dt, z = (None if v is None else v.double() for v in (x, dt, z))
  b, c = (v.double().repeat_interleave(e // groups, 2) for v in (b, c))
  step = dt + (0.0 if dt_bias is None else dt_bias.double())
  if softplus:
    step = torch.where(step > 0, step, 0.0) + torch.log1p(torch.exp(-step.abs()))
  h = x.new_zeros(bs, e, n) if state is None else state.double()
  size = h.abs()
  y, bound = torch.empty_like(x), torch.empty_like(x)
  units = (6 * t + n + 64) * U
  for i in range(t):
    if segment_pos is not None:
      keep = (segment_pos[:, i] != 0)[:, None, None]
      h, size = torch.where(keep, h, 0.0), torch.where(keep, size, 0.0)
    decay = torch.exp(step[:, i, :, None] * a.double())
    put = step[:, i, :, None] * x[:, i, :, None] * b[:, i]
    h, size = decay * h + put, decay * size + put.abs()
    y[:, i] = (h * c[:, i]).sum(-1)
    bound[:, i] = (size * c[:, i].abs()).sum(-1)
    if d is not None:
      y[:, i] += d.double() * x[:, i]
      bound[:, i] += (d.double() * x[:, i]).abs()
  if z is not None:
    gate = z * torch.sigmoid(z)
    y, bound = y * gate, bound * gate.abs()
  return y, h, units * bound, units * size


SCAN = [
    # b, t, e, n, groups, doc, options
    (1, 1, 8, 16, 1, 0, {}),
    (3, 1, 40, 16, 1, 0, dict(z=False)),
    (2, 1, 33, 5, 1, 0, dict(part=True)),
    (4, 1, 64, 128, 2, 0, {}),
    (2, 1, 12, 200, 1, 1, dict(d=False, bias=False)),
    (70, 1, 2560, 16, 1, 0, {}),
    (67, 1, 2570, 9, 2, 3, dict(part=True)),
    (131, 1, 300, 130, 1, 0, dict(z=False)),
    (256, 1, 5120, 16, 1, 2, {}),                  # many sequences a thread
    (300, 1, 5132, 8, 2, 0, dict(state=False)),
    (256, 1, 5120, 7, 1, 0, {}), (256, 1, 200, 200, 1, 0, {}),         # the same without vectors, with eight states a lane
    (1, 2, 8, 1, 1, 0, {}),
    (2, 31, 64, 16, 2, 7, {}),
    (2, 32, 36, 16, 1, 0, dict(state=False)),
    (2, 33, 30, 16, 3, 3, dict(part=True)),
    (1, 100, 130, 4, 1, 20, dict(z=False, d=False, bias=False, state=False)),
    (2, 70, 100, 8, 2, 11, dict(part=True)),
    (2, 64, 24, 21, 1, 9, dict(z=False)),
    (1, 65, 40, 64, 2, 30, {}),
    (1, 40, 20, 100, 1, 8, {}),
    (2, 35, 10, 256, 1, 8, dict(part=True)),
    (3, 257, 2560, 16, 1, 60, {}),
    (9, 90, 5120, 16, 1, 0, {}),
    (1, 50, 1024, 16, 1, 20, {}), (1, 50, 4096, 16, 1, 20, {}),        # every shape that a number of states has
    (8, 40, 5120, 8, 1, 30, {}), (2, 40, 5120, 30, 2, 30, dict(part=True)), (4, 40, 5120, 32, 1, 0, {}),
    (2, 40, 2560, 64, 1, 30, {}), (2, 40, 5120, 60, 1, 30, {}), (1, 40, 5120, 128, 2, 30, {}),
    (3, 700, 5120, 16, 1, 90, {}),                 # more blocks of channels than CTAs: chunks of time
    (2, 1031, 5120, 24, 2, 200, dict(part=True)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,e,n,groups,doc,options", SCAN)
def test_selective_scan(b, t, e, n, groups, doc, options, dtype):
  import recurrentgemma_b200 as rg
  case = scan_case(t + e + n, b, t, e, n, dtype, groups, doc, **options)
  y, state = rg.selective_scan(**case)
  want, held, bound, bound_state = scan_definition(**case)
  within(y, want, bound, dtype)
  within(state, held, bound_state, torch.float32)
  again, none = rg.selective_scan(**case, return_state=False)
  assert none is None and torch.equal(again, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_scan_given_steps(dtype):
  """softplus=False takes dt as the step, and a may be any number: a state that grows, one that stays."""
  import recurrentgemma_b200 as rg
  case = scan_case(3, 2, 40, 24, 16, dtype, doc=9)
  case["dt"] = case["dt"].abs() * 0.1
  case["dt_bias"] = None
  case["a"][:, 0], case["a"][:, 1] = 0.0, 0.3
  y, state = rg.selective_scan(**case, softplus=False)
  want, held, bound, bound_state = scan_definition(**case, softplus=False)
  within(y, want, bound, dtype)
  within(state, held, bound_state, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_scan_steps_of_any_size(dtype):
  """Steps from 1e-20 to 1e4: the softplus keeps its relative precision below, and lets go of the state above."""
  import recurrentgemma_b200 as rg
  case = scan_case(4, 1, 60, 32, 16, dtype, z=False, d=False, bias=False)
  case["dt"] = torch.linspace(-46.0, 60.0, 60, device="cuda")[None, :, None].expand(1, 60, 32).to(dtype)
  case["dt"] = torch.where(case["dt"] > 50, case["dt"] * 200, case["dt"])
  y, state = rg.selective_scan(**case)
  want, held, bound, bound_state = scan_definition(**case)
  within(y, want, bound, dtype)
  within(state, held, bound_state, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [16, 21])
@pytest.mark.parametrize("cuts", [(1,) * 7, (0, 33, 1, 6), (64, 2)])
def test_selective_scan_in_chunks(cuts, n, dtype):
  """Chunks and single tokens that pass the state on in place reach what the definition gives for all."""
  import recurrentgemma_b200 as rg
  case = scan_case(6, 3, sum(cuts), 40, n, dtype, groups=2, doc=5)
  state, at, parts = case["state"].clone(), 0, []
  for m in cuts:
    part = {k: v[:, at:at + m] if k in ("x", "dt", "b", "c", "z", "segment_pos") else v for k, v in case.items()}
    y, back = rg.selective_scan(**{**part, "state": state}, inplace=True)
    assert back is state
    parts.append(y)
    at += m
  want, held, bound, bound_state = scan_definition(**case)
  within(torch.cat(parts, 1), want, bound, dtype)
  within(state, held, bound_state, torch.float32)


@pytest.mark.gpu
def test_document_start_drops_what_is_not_finite():
  """Whatever a finished document left in the state or the taps, the next one does not see it."""
  import recurrentgemma_b200 as rg
  for t in (1, 40):
    case = scan_case(7, 2, t, 16, 16, torch.float32)
    case["segment_pos"] = torch.arange(t, device="cuda").repeat(2, 1)
    case["state"][:] = math.inf
    case["state"][:, ::2] = math.nan
    clean = rg.selective_scan(**{**case, "state": None})
    got = rg.selective_scan(**case)
    assert all(torch.equal(p, q) for p, q in zip(got, clean))
    conv = conv_case(8, 2, t, 16, 4, torch.float32)
    conv["segment_pos"] = case["segment_pos"]
    conv["state"][:] = math.nan
    clean = rg.causal_conv(**{**conv, "state": None})
    got = rg.causal_conv(**conv)
    assert all(torch.equal(p, q) for p, q in zip(got, clean))


@pytest.mark.gpu
def test_empty():
  """No tokens: the state moves on as it is; no sequences, no channels: nothing."""
  import recurrentgemma_b200 as rg
  case = scan_case(9, 2, 0, 16, 16, torch.bfloat16)
  y, state = rg.selective_scan(**case)
  assert y.shape == (2, 0, 16) and torch.equal(state, case["state"])
  assert not rg.selective_scan(**{**case, "state": None})[1].any()
  conv = conv_case(10, 2, 0, 16, 4, torch.bfloat16)
  y, state = rg.causal_conv(**conv)
  assert y.shape == (2, 0, 16) and torch.equal(state, conv["state"])
  assert rg.causal_conv(**conv_case(10, 0, 4, 16, 4, torch.bfloat16))[0].shape == (0, 4, 16)
  assert rg.selective_scan(**scan_case(9, 0, 3, 16, 16, torch.bfloat16))[1].shape == (0, 16, 16)


@pytest.mark.gpu
def test_long_rows_pass_32_bit_offsets():
  """More than 2^31 elements behind the first token: the last row's values are as those of the row alone."""
  import recurrentgemma_b200 as rg
  wide = torch.empty((2, 3, 400_000_000), dtype=torch.bfloat16, device="cuda")
  x = wide[..., :64].normal_()
  case = conv_case(11, 2, 3, 64, 4, torch.bfloat16)
  got, want = (rg.causal_conv(v, case["w"], case["b"], state=case["state"]) for v in (x, x.contiguous()))
  assert all(torch.equal(p, q) for p, q in zip(got, want))
  scan = scan_case(12, 2, 3, 64, 16, torch.bfloat16)
  got, want = (rg.selective_scan(**{**scan, "x": v, "z": v, "dt": v}) for v in (x, x.contiguous()))
  assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
def test_refusals():
  import recurrentgemma_b200 as rg
  conv = conv_case(13, 2, 4, 16, 4, torch.bfloat16)
  for change, error in [
      (dict(x=conv["x"].cpu()), RuntimeError), (dict(x=conv["x"].half()), TypeError),
      (dict(w=conv["w"].float()), TypeError), (dict(w=conv["w"][:1]), rg.RgkError),
      (dict(w=conv["w"].repeat(2, 1), state=None), rg.RgkError), (dict(w=conv["w"][:, :8]), AssertionError),
      (dict(b=conv["b"][:8]), AssertionError), (dict(state=conv["state"][:, 1:]), AssertionError),
      (dict(state=conv["state"].float()), TypeError), (dict(activation="gelu"), ValueError),
      (dict(segment_pos=torch.zeros(2, 3, device="cuda")), AssertionError),
      (dict(state=None, inplace=True), ValueError),
      (dict(state=conv["state"].transpose(0, 1).contiguous().transpose(0, 1), inplace=True), ValueError)]:
    if change.get("w") is not None and change["w"].shape[0] == 1:
      change["state"] = conv["state"][:, :0]
    with pytest.raises(error):
      rg.causal_conv(**{**conv, **change})
  scan = scan_case(14, 2, 4, 16, 16, torch.bfloat16, groups=2)
  big = scan_case(14, 1, 2, 4, 257, torch.bfloat16)
  with pytest.raises(rg.RgkError, match="257"):
    rg.selective_scan(**big)
  for change, error in [
      (dict(x=scan["x"].cpu()), RuntimeError), (dict(x=scan["x"].double()), TypeError),
      (dict(dt=scan["dt"][:, 1:]), AssertionError), (dict(dt=scan["dt"].float()), TypeError),
      (dict(b=scan["b"][:, :, :1]), AssertionError), (dict(z=scan["z"].float()), TypeError),
      (dict(a=scan["a"].bfloat16()), TypeError), (dict(a=scan["a"][:, :8]), AssertionError),
      (dict(d=scan["d"].bfloat16()), TypeError), (dict(dt_bias=scan["dt_bias"][1:]), AssertionError),
      (dict(state=scan["state"].bfloat16()), TypeError), (dict(state=scan["state"][:1]), AssertionError),
      (dict(b=scan["b"][:, :, :, :0], c=scan["c"][:, :, :, :0], a=scan["a"][:, :0], state=None), rg.RgkError),
      (dict(state=None, inplace=True), ValueError)]:
    with pytest.raises(error):
      rg.selective_scan(**{**scan, **change})


def test_refusals_of_the_library():
  """What the C calls refuse, before any device is touched."""
  import ctypes
  from recurrentgemma_b200 import _lib, build
  build.build_library()
  lib = _lib.load()

  def conv(x=16, w=16, state=None, b=1, t=4, e=8, taps=4, act=1, dtype=1, y=16, pos_dtype=0, pos=None):
    return lib.rgk_causal_conv(x, t * e, e, pos, pos_dtype, w, None, state, b, t, e, taps, act, dtype, y, None, None)
  assert conv(x=None) == conv(w=None) == conv(y=None) == conv(act=2) == conv(dtype=2) == conv(b=-1) == -1
  assert conv(pos=16, pos_dtype=3) == -1
  assert conv(taps=1) == conv(taps=5) == conv(b=70000) == conv(e=1 << 21) == conv(t=1 << 31) == -2
  assert conv(x=17) == conv(state=17) == -3
  assert conv(b=0) == conv(t=0) == conv(e=0) == 0

  def scan(b=1, t=4, e=8, groups=1, n=16, dtype=1, y=16, ws=(None, 0), **of):
    p = _lib.RgkScanInputs(**{**{k: 16 for k in ("x", "dt", "b", "c", "a")}, **of})
    return lib.rgk_selective_scan(ctypes.byref(p), None, 0, None, b, t, e, groups, n, dtype, y, None, *ws, None, None)
  assert scan(x=None) == scan(a=None) == scan(c=None) == scan(y=None) == scan(dtype=7) == scan(t=-1) == -1
  assert scan(n=0) == scan(n=257) == scan(groups=3) == scan(groups=0) == scan(b=70000) == -2
  assert b"70000" in lib.rgk_last_error()
  assert scan(x=17) == scan(a=18) == scan(d=18) == -3
  assert scan(ws=(256, lib.rgk_selective_scan_workspace_bytes() - 1)) == -6 and scan(ws=(66, 1 << 30)) == -3
  assert lib.rgk_selective_scan(None, None, 0, None, 1, 4, 8, 1, 16, 1, 16, None, None, 0, None, None) == -1
  assert scan(b=0) == scan(t=0) == scan(e=0) == 0
