"""sample against its definition in 64 bits: the same token, always.  Weights are multiples of 2^-44 of the largest,
in the definition too: sums of them are exact in 64 bits, and what the exponential is off by (2^-46 of itself) moves
one of them by one such step at most.  Uniform numbers have 24 bits and are not chosen to lie that near to a border."""
import math

import pytest
import torch

DTYPES = [torch.float32, torch.bfloat16]


def definition(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
  """Token by token, a row at a time, in 64 bits; settings held in float32."""
  f32 = lambda v, m: float(torch.tensor(v[m].item() if torch.is_tensor(v) else v, dtype=torch.float32))  # noqa: E731
  out = []
  for m in range(logits.shape[0]):
    l = torch.where(logits[m].isnan(), -math.inf, logits[m].double()).cpu()
    t, p, least, u = (f32(v, m) for v in (temperature, top_p, min_p, uniforms))
    k = int(top_k[m]) if torch.is_tensor(top_k) else top_k
    values, order = torch.sort(l, descending=True, stable=True)
    if values[0] == -math.inf or not t > 0:
      out.append(int(order[0]) if values[0] > -math.inf else 0)
      continue
    w = torch.exp((values - values[0]) / t)
    w[values == values[0]] = 1.0
    w[values == -math.inf] = 0.0
    unit = 2.0 ** (44 if len(l) <= 2 ** 18 else 43 if len(l) <= 2 ** 19 else 42)
    w = torch.round(w * unit) / unit
    if k > 0:
      w[k:] = 0.0
    if p < 1.0:
      before = torch.cumsum(w, 0) - w
      exact = torch.cat([torch.zeros(1, dtype=torch.float64), torch.cumsum(w, 0)[:-1]])
      assert torch.allclose(before, exact, rtol=0, atol=1e-6)
      keep = exact < p * w.sum()
      keep[0] = True
      w = torch.where(keep, w, 0.0)
    w[w < least] = 0.0
    kept = torch.zeros_like(w)
    kept[order] = w
    upto = torch.cumsum(kept, 0)
    out.append(int((upto <= u * upto[-1]).sum()))
  return torch.tensor(out, dtype=torch.int32, device=logits.device)


def rows(seed, m, v, dtype, std=3.0):
  g = torch.Generator(device="cuda").manual_seed(seed)
  logits = (torch.randn((m, v), generator=g, device="cuda") * std).to(dtype)
  return logits, torch.rand((m,), generator=g, device="cuda"), g


SETTINGS = [
    {}, dict(temperature=0.0), dict(temperature=0.05), dict(temperature=40.0), dict(top_k=1), dict(top_k=2),
    dict(top_k=40), dict(top_k=128), dict(top_k=129), dict(top_k=3000, top_p=0.9), dict(top_k=10**6), dict(top_p=0.0), dict(top_p=0.5), dict(top_p=0.95), dict(top_p=0.9999),
    dict(min_p=0.1), dict(min_p=1.0), dict(top_k=100, top_p=0.7, min_p=0.02, temperature=1.3),
    dict(top_p=0.9, temperature=6.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("m,v", [(1, 1), (3, 2), (2, 31), (4, 256), (3, 257), (2, 4097), (2, 50001), (9, 32000)])
def test_sample(m, v, settings, dtype):
  import recurrentgemma_b200 as rg
  logits, uniforms, _ = rows(m + v, m, v, dtype)
  got = rg.sample(logits, uniforms, **settings)
  assert got.dtype == torch.int32
  assert torch.equal(got, definition(logits, uniforms, **settings))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 40, 300])
def test_sample_large_vocabulary(m, dtype):
  """Rows of the model's vocabulary with settings of their own; one row alone gives what it gives among others."""
  import recurrentgemma_b200 as rg
  logits, uniforms, g = rows(m, m, 256_000, dtype, std=2.0)
  r = lambda: torch.rand((m,), generator=g, device="cuda")                       # noqa: E731
  settings = dict(temperature=2.0 * r() * (r() > 0.1), top_p=1.1 * r() + 0.2, min_p=0.1 * r() * (r() > 0.5),
                  top_k=torch.randint(-1, 3000, (m,), generator=g, dtype=torch.int32, device="cuda"))
  settings["top_k"] *= torch.rand((m,), generator=g, device="cuda") > 0.5
  got = rg.sample(logits, uniforms, **settings)
  some = range(0, m, max(1, m // 12))
  pick = torch.tensor(list(some), device="cuda")
  want = definition(logits[pick], uniforms[pick], **{k: v[pick] for k, v in settings.items()})
  assert torch.equal(got[pick], want)
  for i in list(some)[:6]:
    alone = rg.sample(logits[i:i + 1], uniforms[i:i + 1], **{k: v[i:i + 1] for k, v in settings.items()})
    assert torch.equal(alone, got[i:i + 1])


@pytest.mark.gpu
@pytest.mark.parametrize("v", [2 ** 18, 2 ** 18 + 1, 2 ** 20])
def test_sample_largest_vocabularies(v):
  import recurrentgemma_b200 as rg
  logits, uniforms, _ = rows(v, 2, v, torch.float32)
  for settings in ({}, dict(top_k=100, top_p=0.9), dict(temperature=30.0, top_p=0.5), dict(top_k=v // 4, top_p=0.9)):
    assert torch.equal(rg.sample(logits, uniforms, **settings), definition(logits, uniforms, **settings)), settings


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_special_rows(dtype):
  """Rows of one value, of two, with infinities, NaN and masked places of the type's lowest value."""
  import recurrentgemma_b200 as rg
  v = 5000
  low = torch.finfo(dtype).min
  logits, uniforms, _ = rows(1, 17, v, dtype)
  logits[0] = 0.0
  logits[1] = -math.inf
  logits[2] = math.nan
  logits[3, :] = -math.inf
  logits[3, 77] = 3.0
  logits[4, ::3] = math.nan
  logits[5, 100:] = low
  logits[6] = low
  logits[7, 5], logits[7, 900] = math.inf, math.inf
  logits[8] = 0.0
  logits[8, 1::2] = -0.0
  logits[9] = torch.where(torch.arange(v, device="cuda") % 7 == 0, 2.0, 1.0)
  logits[10, 50:] = -math.inf
  logits[11] = -70000.0
  logits[12, :] = logits[12, 0]
  logits[13, 1:] = -math.inf
  logits[14] = -math.inf
  logits[14, v - 1] = low
  logits[15, 1000:1300] += 20.0                       # the likely ones side by side
  logits[16, :40], logits[16, 2500:2600] = 9.0, 9.0   # and equal
  for settings in SETTINGS:
    for u in (0.0, 0.3, 0.5, 1.0 - 2.0 ** -24):
      uniforms[:] = u
      assert torch.equal(rg.sample(logits, uniforms, **settings), definition(logits, uniforms, **settings)), (settings, u)


@pytest.mark.gpu
def test_sample_follows_the_distribution():
  """Evenly spread uniform numbers give every token its share."""
  import recurrentgemma_b200 as rg
  n = 4096
  logits = torch.log(torch.tensor([0.1, 0.2, 0.05, 0.4, 0.25], device="cuda"))[None].repeat(n, 1)
  u = (torch.arange(n, device="cuda") + 0.5) / n
  for settings, shares in [({}, [0.1, 0.2, 0.05, 0.4, 0.25]), (dict(top_k=2), [0, 0, 0, 0.4 / 0.65, 0.25 / 0.65]),
                           (dict(top_p=0.8), [0, 0.2 / 0.85, 0, 0.4 / 0.85, 0.25 / 0.85]),
                           (dict(min_p=0.3), [0, 0.2 / 0.85, 0, 0.4 / 0.85, 0.25 / 0.85]),
                           (dict(temperature=0.5), [v * v / 0.275 for v in (0.1, 0.2, 0.05, 0.4, 0.25)])]:
    count = torch.bincount(rg.sample(logits, u, **settings).long(), minlength=5)
    for c, share in zip(count.tolist(), shares):
      assert abs(c - share * n) <= 1.01        # a share's ends fall between two of the numbers


@pytest.mark.gpu
def test_sample_uniforms_out_of_range():
  """Numbers outside [0, 1) and NaN take the first or the last kept token."""
  import recurrentgemma_b200 as rg
  logits = torch.zeros((5, 100), device="cuda")
  logits[:, :3], logits[:, 90:] = -math.inf, -math.inf
  u = torch.tensor([-1.0, 1.0, 2.0, math.nan, math.inf], device="cuda")
  assert rg.sample(logits, u).tolist() == [3, 89, 89, 3, 89]


@pytest.mark.gpu
def test_sample_layouts():
  """Rows of a wider tensor, unaligned ones, leading dimensions, an output of the caller's."""
  import recurrentgemma_b200 as rg
  wide, uniforms, _ = rows(3, 6, 1003, torch.bfloat16)
  part = wide[:, 1:1000]
  want = rg.sample(part.contiguous(), uniforms, top_p=0.9)
  assert torch.equal(want, definition(part, uniforms, top_p=0.9))
  out = torch.full((6,), -1, dtype=torch.int32, device="cuda")
  assert rg.sample(part, uniforms, top_p=0.9, out=out) is out and torch.equal(out, want)
  assert torch.equal(rg.sample(part.unflatten(0, (2, 3)), uniforms.view(2, 3), top_p=0.9), want.view(2, 3))
  assert torch.equal(rg.sample(part.t().contiguous().t(), uniforms, top_p=0.9), want)
  assert rg.sample(wide[:0], uniforms[:0]).shape == (0,)
  assert rg.sample(wide[0], uniforms[0], top_p=0.9).shape == ()


@pytest.mark.gpu
def test_sample_refusals():
  import recurrentgemma_b200 as rg
  logits, u, _ = rows(4, 3, 100, torch.float32)
  for args, kw, error in [
      ((logits.cpu(), u), {}, RuntimeError), ((logits, u.cpu()), {}, RuntimeError), ((logits.half(), u), {}, TypeError),
      ((logits, u.double()), {}, TypeError), ((logits, u[:2]), {}, AssertionError),
      ((logits, u), dict(temperature=-1.0), ValueError), ((logits, u), dict(temperature=math.nan), ValueError),
      ((logits, u), dict(top_p=-0.1), ValueError), ((logits, u), dict(min_p=1.5), ValueError),
      ((logits, u), dict(min_p=-0.5), ValueError), ((logits, u), dict(top_k=u), TypeError),
      ((logits, u), dict(top_p=u.double()), TypeError), ((logits, u), dict(top_p=u[:2]), AssertionError),
      ((logits, u), dict(out=torch.zeros(3, dtype=torch.int64, device="cuda")), AssertionError),
      ((torch.zeros((1, 2**20 + 1), device="cuda"), u[:1]), {}, rg.RgkError),
      ((logits[:, :0], u), {}, rg.RgkError)]:
    with pytest.raises(error):
      rg.sample(*args, **kw)


def test_refusals_of_the_library():
  """What the C call refuses, before any device is touched."""
  import ctypes
  from recurrentgemma_b200 import _lib, build
  build.build_library()
  lib = _lib.load()

  def call(x=16, m=1, v=100, dtype=0, u=16, out=16, settings=True, **of):
    p = _lib.RgkSampleSettings(**of)
    return lib.rgk_sample(x, m, v, v, dtype, u, ctypes.byref(p) if settings else None, out, None)
  assert call(x=None) == call(u=None) == call(out=None) == call(dtype=2) == call(m=-1) == call(v=0) == -1
  assert call(settings=False) == -1
  assert call(v=2**20 + 1) == -2 and b"2^20" in lib.rgk_last_error()
  assert call(x=18) == call(u=18) == call(top_k=18) == -3
  assert call(m=0) == 0
