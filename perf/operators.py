"""Operator cases: the calls around a selective state space layer and the draw of the next token.

A case is a dict of plain values whose "op" says which operator it calls:

  conv     causal_conv: the short causal convolution with its activation; seq 1 is a decode step
  scan     selective_scan: the selective state space recurrence; seq 1 is a decode step
  sample   sample: one token per row of logits, by temperature, top-k, top-p and min-p

`run` computes a case in its plain form, elementary torch operations in float32 (float64 where cumulated
weights decide a token), or, where `own` is set, by the calls of this package.  Widths are those of the 2B
preset (2560) and twice it, as such layers have; the vocabulary is the preset's 256000.
"""
import math

import torch

own = False

VOCAB = 256_000
MOST = 8 * 4096 * 5120                       # elements of the largest activation


def listed():
  return [
      # The convolution of a layer over a full prefill batch; its input is one half of a projection's output.
      dict(name="conv_prefill", op="conv", dtype="bfloat16", batch=8, seq=4096, width=5120, taps=4,
           doc=0, state=False, half=True),
      # A continued chunk of packed documents in float32, odd in length and width, three taps.
      dict(name="conv_packed", op="conv", dtype="float32", batch=3, seq=1237, width=2565, taps=3,
           doc=200, state=True, half=False),
      # The convolution of one token for 64 sequences.
      dict(name="conv_step", op="conv", dtype="bfloat16", batch=64, seq=1, width=5120, taps=4, doc=0,
           state=True, half=True),
      # The recurrence of a layer over a full prefill batch.
      dict(name="scan_prefill", op="scan", dtype="bfloat16", batch=8, seq=4096, width=5120, states=16,
           groups=1, doc=0, state=False, gate=True),
      # One interactive prompt.
      dict(name="scan_prompt", op="scan", dtype="bfloat16", batch=1, seq=2048, width=5120, states=16,
           groups=1, doc=0, state=False, gate=True),
      # Numerics work: float32, a continued chunk of packed documents, two groups, an odd number of states.
      dict(name="scan_packed", op="scan", dtype="float32", batch=2, seq=777, width=2560, states=21,
           groups=2, doc=150, state=True, gate=False),
      # One token of one sequence: the smallest call of a decode loop.
      dict(name="scan_step_one", op="scan", dtype="bfloat16", batch=1, seq=1, width=5120, states=16,
           groups=1, doc=0, state=True, gate=True),
      # One token for a full serving batch: the states are read and written.
      dict(name="scan_step_batch", op="scan", dtype="bfloat16", batch=256, seq=1, width=5120, states=16,
           groups=1, doc=0, state=True, gate=True),
      # The next token of one chat.
      dict(name="sample_one", op="sample", dtype="bfloat16", rows=1, vocab=VOCAB, temperature=0.8,
           top_k=50, top_p=0.95, min_p=0.0, mixed=False),
      # A serving batch with nucleus sampling on float32 logits.
      dict(name="sample_nucleus", op="sample", dtype="float32", rows=256, vocab=VOCAB, temperature=1.0,
           top_k=0, top_p=0.9, min_p=0.02, mixed=False),
      # Rollouts for evaluation: the whole distribution.
      dict(name="sample_whole", op="sample", dtype="bfloat16", rows=64, vocab=VOCAB, temperature=1.0,
           top_k=0, top_p=1.0, min_p=0.0, mixed=False),
      # A small odd vocabulary, every row with settings of its own, greedy ones among them.
      dict(name="sample_mixed", op="sample", dtype="float32", rows=33, vocab=32_003, temperature=0.9,
           top_k=40, top_p=0.8, min_p=0.05, mixed=True),
  ]


def _log(rng, lo, hi):
  """An integer spread over [lo, hi] by its logarithm."""
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(["conv", "scan", "scan", "sample"])
  dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
  if op == "sample":
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, VOCAB),
                temperature=round(rng.uniform(0.3, 2.0), 3), top_k=rng.choice([0, _log(rng, 1, 1000)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                min_p=rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)]), mixed=rng.random() < 0.5)
  width = rng.choice([2560, 5120, _log(rng, 64, 5120)])
  step = rng.random() < 0.3
  batch = _log(rng, 1, 256 if step else 8)
  seq = 1 if step else _log(rng, 2, min(16384, MOST // 2 // (width * batch)))
  case = dict(op=op, dtype=dtype, batch=batch, seq=seq, width=width,
              doc=0 if step else rng.choice([0, _log(rng, 16, 2048)]), state=step or rng.random() < 0.5)
  if op == "conv":
    return dict(case, taps=rng.choice([2, 3, 4, 4]), half=rng.random() < 0.5)
  return dict(case, states=rng.choice([16, 16, rng.randint(1, 32)]),
              groups=2 if width % 2 == 0 and rng.random() < 0.3 else 1, gate=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------
# What a program has in hand before the call
# ------------------------------------------------------------------------------------------------
def _positions(g, batch, seq, doc, state):
  """Positions of rows packed with documents of mean length `doc`; a continued chunk begins inside one.
  None where every row is one document."""
  if not doc:
    return None
  pos = torch.arange(seq, dtype=torch.int64, device="cuda").repeat(batch, 1)
  starts = torch.rand((batch, seq), generator=g, device="cuda") < 1.0 / doc
  starts[:, 0] = not state
  begin = torch.cummax(torch.where(starts, pos, torch.full_like(pos, -7)), dim=1).values
  return pos - begin


def prepare(case, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  dt = getattr(torch, case["dtype"])

  def normal(*shape, std=1.0, dtype=dt):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)

  def uniform(*shape):
    return torch.rand(shape, generator=g, device="cuda")

  s = {"op": case["op"]}
  if case["op"] == "sample":
    m, v = case["rows"], case["vocab"]
    # a broad bulk and some tens of likely tokens a row, capped as the model caps its logits
    logits = normal(m, v, std=2.0, dtype=torch.float32)
    likely = torch.randint(0, v, (m, 64), generator=g, device="cuda")
    # (where two of them are one token, the larger value: inputs of one seed are the same each time)
    logits.scatter_reduce_(1, likely, 4.0 + 10.0 * uniform(m, 64), "amax", include_self=False)
    s["logits"] = (30.0 * torch.tanh(logits / 30.0)).to(dt)
    s["uniforms"] = uniform(m)
    settings = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
    if case["mixed"]:                        # every request of a batch comes with its own
      settings["temperature"] = settings["temperature"] * (0.5 + uniform(m)) * (uniform(m) > 0.1)
      settings["top_k"] = torch.randint(0, 2 * case["top_k"] + 1, (m,), generator=g, dtype=torch.int32,
                                        device="cuda")
      settings["top_p"] = 1.0 - (1.0 - case["top_p"]) * 2.0 * uniform(m)
      settings["min_p"] = case["min_p"] * 2.0 * uniform(m)
    s["settings"] = settings
    return s
  b, t, e = case["batch"], case["seq"], case["width"]
  s["pos"] = _positions(g, b, t, case["doc"], case["state"])
  if case["op"] == "conv":
    taps = case["taps"]
    s["x"] = normal(b, t, 2 * e)[..., :e] if case["half"] else normal(b, t, e)
    s["w"], s["b"] = normal(taps, e, std=0.5), normal(e, std=0.1)
    s["state"] = normal(b, taps - 1, e) if case["state"] else None
    return s
  n, groups = case["states"], case["groups"]
  s["x"], s["dt"] = normal(b, t, e), normal(b, t, e, std=0.5)
  # steps of 1e-3 to 1e-1 behind the softplus, decay rates of 1 to N
  step = torch.exp(uniform(e) * math.log(100.0) + math.log(1e-3))
  s["dt_bias"] = step + torch.log(-torch.expm1(-step))
  s["a"] = -(torch.arange(1, n + 1, device="cuda") * torch.exp(normal(e, n, std=0.2, dtype=torch.float32)))
  # b and c are parts of one projection's output, behind the 160 columns that the step comes from
  bc = normal(b, t, 160 + 2 * groups * n)
  s["b"], s["c"] = (bc[..., 160 + k * groups * n:160 + (k + 1) * groups * n].unflatten(-1, (groups, n))
                    for k in (0, 1))
  s["d"] = normal(e, std=0.5, dtype=torch.float32)
  s["z"] = normal(b, t, 2 * e)[..., e:] if case["gate"] else None
  s["state"] = normal(b, e, n, std=0.3, dtype=torch.float32) if case["state"] else None
  return s


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------
def run(s):
  if own:
    return _own(s)
  if s["op"] == "conv":
    return _conv(s["x"], s["w"], s["b"], s["pos"], s["state"])
  if s["op"] == "scan":
    return _scan(s["x"], s["dt"], s["a"], s["b"], s["c"], s["d"], s["z"], s["dt_bias"], s["pos"],
                 s["state"])
  return _sample(s["logits"], s["uniforms"], **s["settings"])


def _own(s):
  import recurrentgemma_b200 as rg
  if s["op"] == "conv":
    return rg.causal_conv(s["x"], s["w"], s["b"], segment_pos=s["pos"], state=s["state"])
  if s["op"] == "scan":
    return rg.selective_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], d=s["d"], z=s["z"],
                             dt_bias=s["dt_bias"], segment_pos=s["pos"], state=s["state"])
  return rg.sample(s["logits"], s["uniforms"], **s["settings"])


def _silu(v):
  return v / (1.0 + torch.exp(-v))


def _conv(x, w, b, pos, state):
  """Causal depthwise convolution and silu; taps and the new state stop at document starts."""
  taps, (batch, seq, width) = w.shape[0], x.shape
  before = x.new_zeros(batch, taps - 1, width) if state is None else state
  rows = torch.cat([before, x], dim=1).float()
  windows = rows.unfold(1, taps, 1)                                 # [B, T, E, W]
  if pos is None:
    last, y = rows[:, seq:], (windows * w.float().T).sum(-1)
  else:
    doc = torch.cumsum(pos == 0, dim=1)
    docs = torch.cat([doc.new_zeros(batch, taps - 1), doc], dim=1)
    same = docs.unfold(1, taps, 1) == doc[..., None]                # [B, T, W]
    y = (windows * w.float().T * same[:, :, None]).sum(-1)
    last = rows[:, seq:] * (docs[:, seq:] == docs[:, -1:])[..., None]
  return _silu(y + b.float()).to(x.dtype), last.to(x.dtype)


def _scan(x, dt, a, b, c, d, z, dt_bias, pos, state):
  """h_t = exp(step a) h_{t-1} + step x b, y = <h, c> + d x, times silu(z): by doubling, every time step
  joined with the one 1, 2, 4, ... before it."""
  (batch, seq, width), (groups, n) = x.shape, b.shape[2:]
  xf = x.float()
  step = dt.float() + dt_bias
  step = torch.where(step > 20.0, step, torch.log1p(torch.exp(step)))
  decay = torch.exp(step[..., None] * a)                            # [B, T, E, N]
  if pos is not None:
    decay = decay * (pos != 0)[:, :, None, None]
  h = (step * xf).view(batch, seq, groups, -1, 1) * b.float()[:, :, :, None]
  h = h.view(batch, seq, width, n)
  if state is not None:
    h[:, 0] += decay[:, 0] * state
  back = 1
  while back < seq:
    h[:, back:] += decay[:, back:] * h[:, :-back]
    decay[:, back:] *= decay[:, :-back].clone()
    back *= 2
  y = (h.view(batch, seq, groups, -1, n) * c.float()[:, :, :, None]).sum(-1).view(batch, seq, width)
  y = y + d * xf
  if z is not None:
    y = y * _silu(z.float())
  return y.to(x.dtype), h[:, -1].clone()


def _column(value, like, dtype):
  """A setting, one for all rows or one for each, as a column (numbers are held in `dtype` first)."""
  if not torch.is_tensor(value):
    value = torch.full(like.shape[:1], value, dtype=dtype, device=like.device)
  return value[:, None]


def _sample(logits, uniforms, temperature, top_k, top_p, min_p):
  """One token per row; cumulated weights in 64 bits, since they decide which."""
  f32, i32 = torch.float32, torch.int32
  temperature, top_p, min_p = (_column(v, logits, f32).double() for v in (temperature, top_p, min_p))
  top_k = _column(top_k, logits, i32)
  x = torch.where(logits.isnan(), -math.inf, logits.double())
  x, order = torch.sort(x, dim=-1, descending=True, stable=True)
  rank = torch.arange(x.shape[1], device=x.device)
  w = torch.where(x == x[:, :1], 1.0, torch.exp((x - x[:, :1]) / temperature))
  w = torch.where((rank < top_k) | (top_k <= 0), w, 0.0)
  upto = torch.cumsum(w, dim=-1)
  within = torch.cat([torch.ones_like(upto[:, :1]), upto[:, :-1] < top_p * upto[:, -1:]], dim=-1) > 0
  w = torch.where((within | (top_p >= 1.0)) & (w >= min_p), w, 0.0)
  upto = torch.cumsum(torch.zeros_like(w).scatter_(1, order, w), dim=-1)
  token = (upto <= uniforms[:, None].double() * upto[:, -1:]).sum(-1)
  greedy = (temperature[:, 0] == 0) | (x[:, 0] == -math.inf)
  return torch.where(greedy, order[:, 0], token).to(i32)


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
  s = prepare(case, seed)
  if case["op"] == "sample":
    return None
  f64 = lambda v: None if v is None else v.double()                 # noqa: E731
  x, pos, state = f64(s["x"]), s["pos"], f64(s["state"])
  batch, seq, width = x.shape
  start = torch.zeros(batch, seq, dtype=torch.bool, device="cuda") if pos is None else pos == 0
  y = torch.empty_like(x)
  if case["op"] == "conv":
    w, bias, taps = f64(s["w"]), f64(s["b"]), case["taps"]
    held = x.new_zeros(batch, taps - 1, width) if state is None else state.clone()
    for t in range(seq):
      held[start[:, t]] = 0.0
      window = torch.cat([held, x[:, t:t + 1]], dim=1)
      y[:, t] = torch.einsum("bwe,we->be", window, w) + bias
      held = window[:, 1:].clone()
    return y * torch.sigmoid(y), held
  per = width // case["groups"]
  a, d, z = f64(s["a"]), f64(s["d"]), f64(s["z"])
  step = torch.logaddexp(s["dt"].double() + s["dt_bias"].double(), x.new_zeros(()))
  h = x.new_zeros(batch, width, case["states"]) if state is None else state.clone()
  for t in range(seq):
    h[start[:, t]] = 0.0
    now = step[:, t, :, None]
    b, c = (v[:, t].double().repeat_interleave(per, dim=1) for v in (s["b"], s["c"]))
    h = h * torch.exp(now * a) + now * x[:, t, :, None] * b
    y[:, t] = (h * c).sum(-1) + d * x[:, t]
  return y if z is None else y * z * torch.sigmoid(z), h


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
  size = 4 if case["dtype"] == "float32" else 2
  if case["op"] == "sample":
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size + case["rows"] * 8, "flops": 4 * n}
  b, t, e = case["batch"], case["seq"], case["width"]
  n, pos, states = b * t * e, b * t * 8 * (case["doc"] > 0), 2 if case["state"] else 1
  if case["op"] == "conv":
    taps = case["taps"]
    return {"bytes": 2 * n * size + pos + ((taps + 1) * e + states * b * (taps - 1) * e) * size,
            "flops": n * (2 * taps + 4)}
  k, groups = case["states"], case["groups"]
  return {"bytes": (3 + case["gate"]) * n * size + 2 * b * t * groups * k * size + pos
          + 4 * (e * (k + 2) + states * b * e * k),
          "flops": n * (7 * k + 8 + 4 * case["gate"])}
