"""The operators of a state space layer and the draw of tokens, run together as a program uses them."""
import pytest
import torch

from tests.test_sample import definition


class Layers:
  """A small state space language model: embedding, convolution, recurrence, logits; float32 or bfloat16."""

  def __init__(self, width=96, states=16, vocab=500, taps=4, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda") * std       # noqa: E731
    self.dtype, self.width, self.states, self.taps = dtype, width, states, taps
    self.table = normal(vocab, width).to(dtype)
    self.w_in = normal(width, 2 * width, std=width ** -0.5).to(dtype)
    self.w_bc = normal(width, width + 2 * states, std=width ** -0.5).to(dtype)
    self.conv_w, self.conv_b = normal(taps, width, std=0.5).to(dtype), normal(width, std=0.1).to(dtype)
    self.a = -torch.exp(normal(width, states, std=0.5))
    self.d, self.dt_bias = normal(width), normal(width) - 3.0

  def states_for(self, b):
    return (torch.zeros(b, self.taps - 1, self.width, dtype=self.dtype, device="cuda"),
            torch.zeros(b, self.width, self.states, device="cuda"))

  def __call__(self, tokens, conv_state, state, segment_pos=None, inplace=False):
    import recurrentgemma_b200 as rg
    x, z = (self.table[tokens.long()] @ self.w_in).chunk(2, dim=-1)            # both strided
    x, conv_state = rg.causal_conv(x, self.conv_w, self.conv_b, segment_pos=segment_pos, state=conv_state,
                                   inplace=inplace)
    dt, b, c = torch.split(x @ self.w_bc, [self.width, self.states, self.states], dim=-1)
    y, state = rg.selective_scan(x, dt, self.a, b[:, :, None], c[:, :, None], d=self.d, z=z,
                                 dt_bias=self.dt_bias, segment_pos=segment_pos, state=state, inplace=inplace)
    return y @ self.table.T, conv_state, state


SETTINGS = dict(temperature=0.9, top_k=50, top_p=0.9, min_p=0.01)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_and_captured_steps(dtype):
  """A prompt, then tokens by a captured step that overwrites its states, against the same steps one by one."""
  import recurrentgemma_b200 as rg
  b, prompt, steps = 3, 37, 12
  m = Layers(dtype=dtype)
  g = torch.Generator(device="cuda").manual_seed(1)
  tokens = torch.randint(0, 500, (b, prompt), generator=g, device="cuda", dtype=torch.int32)
  u = torch.rand((steps, b), generator=g, device="cuda")
  logits, conv0, state0 = m(tokens, *m.states_for(b))
  first = rg.sample(logits[:, -1], u[0], **SETTINGS)
  assert torch.equal(first, definition(logits[:, -1], u[0], **SETTINGS))

  eager, conv, state, token = [first], conv0.clone(), state0.clone(), first
  for i in range(1, steps):
    logits, conv, state = m(token[:, None], conv, state)
    token = rg.sample(logits[:, 0], u[i], **SETTINGS)
    assert torch.equal(token, definition(logits[:, 0], u[i], **SETTINGS))
    eager.append(token)

  conv_s, state_s, token_s, u_s = conv0.clone(), state0.clone(), first.clone(), u[0].clone()

  def step():
    out, _, _ = m(token_s[:, None], conv_s, state_s, inplace=True)
    rg.sample(out[:, 0], u_s, **SETTINGS, out=token_s)
  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    keep = [t.clone() for t in (conv_s, state_s, token_s)]
    step()
    for t, k in zip((conv_s, state_s, token_s), keep):
      t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
      step()
    for i in range(1, steps):
      u_s.copy_(u[i])
      graph.replay()
      assert torch.equal(token_s, eager[i]), i
  torch.cuda.synchronize()
  assert torch.equal(conv_s, conv) and torch.equal(state_s, state)


@pytest.mark.gpu
def test_captured_prompts_on_two_streams():
  """Long calls that cut time into chunks, captured one after the other on one stream and replayed side by side."""
  import recurrentgemma_b200 as rg
  e, t = 5120, 600
  g = torch.Generator(device="cuda").manual_seed(2)
  normal = lambda *s: torch.randn(s, generator=g, device="cuda")               # noqa: E731
  a, bias = -torch.exp(normal(e, 16)), normal(e) - 3.0
  calls = []
  stream = torch.cuda.Stream()
  for k in range(2):
    x, dt = normal(4, t, e).bfloat16(), normal(4, t, e).bfloat16()
    bc = normal(4, t, 2, 16).bfloat16()
    args = (x, dt, a, bc[:, :, :1].contiguous(), bc[:, :, 1:].contiguous())
    want = rg.selective_scan(*args, dt_bias=bias)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
      rg.selective_scan(*args, dt_bias=bias)
      graph = torch.cuda.CUDAGraph()
      with torch.cuda.graph(graph, stream=stream):
        got = rg.selective_scan(*args, dt_bias=bias)
    calls.append((torch.cuda.Stream(), graph, want, got, args))
  for _ in range(5):
    for _, _, _, got, _ in calls:
      for o in got:
        o.zero_()
    torch.cuda.synchronize()
    for own, graph, *_ in calls:
      with torch.cuda.stream(own):
        graph.replay()
    torch.cuda.synchronize()
    for _, _, want, got, _ in calls:
      assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.gpu
def test_long_calls_on_two_streams_at_once():
  import recurrentgemma_b200 as rg
  from tests.test_state_space import scan_case
  cases = [scan_case(seed, 4, 700, 5120, 16, torch.bfloat16) for seed in (5, 6)]
  want = [rg.selective_scan(**c) for c in cases]
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  torch.cuda.synchronize()
  for _ in range(5):
    got = []
    for c, stream in zip(cases, streams):
      with torch.cuda.stream(stream):
        got.append(rg.selective_scan(**c))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for g, w in zip(got, want) for p, q in zip(g, w))


@pytest.mark.gpu
def test_left_padded_batch():
  """Rows of a padded batch (padding at positions of -1, the first token at 0) give what they give alone."""
  m = Layers(dtype=torch.float32)
  g = torch.Generator(device="cuda").manual_seed(3)
  longest, lengths = 45, (45, 1, 20)
  tokens = torch.randint(0, 500, (3, longest), generator=g, device="cuda")
  pos = torch.arange(longest, device="cuda")[None] - longest + torch.tensor(lengths, device="cuda")[:, None]
  logits, conv, state = m(tokens, *m.states_for(3), segment_pos=pos.clip(min=-1))
  for i, n in enumerate(lengths):
    alone = m(tokens[i:i + 1, longest - n:], *m.states_for(1))
    assert (conv[i] - alone[1][0]).abs().max() <= 2.0 ** -12 * alone[1].abs().max()
    # (torch's products of 96 terms may sum in another order for another number of rows: 96 u of the magnitudes' sum, some
    # ten times the result, three of them in a row - 3000 u, below 2^-12)
    for got, want in ((logits[i, longest - n:], alone[0][0]), (state[i], alone[2][0])):
      assert (got - want).abs().max() <= 2.0 ** -12 * want.abs().max()


# ---- Sampler --------------------------------------------------------------------------------------
def _griffin():
  import recurrentgemma_b200 as rg
  kinds = [rg.TemporalBlockType.RECURRENT, rg.TemporalBlockType.RECURRENT, rg.TemporalBlockType.ATTENTION]
  config = rg.GriffinConfig(vocab_size=1000, width=512, mlp_expanded_width=1024, num_heads=2, lru_width=512,
                            embeddings_scale_by_sqrt_dim=True, attention_window_size=64, logits_soft_cap=30.0,
                            block_types=tuple(kinds))
  torch.manual_seed(0)
  return rg.Griffin(config, device="cuda", dtype=torch.bfloat16).eval()


@pytest.mark.gpu
def test_sampler():
  import recurrentgemma_b200 as rg
  model = _griffin()
  g = torch.Generator(device="cuda").manual_seed(4)
  tokens = torch.randint(0, 1000, (3, 20), generator=g, device="cuda", dtype=torch.int32)
  lengths = torch.tensor([20, 3, 11], device="cuda", dtype=torch.int32)
  u = torch.rand((3, 9), generator=g, device="cuda")
  greedy = rg.GreedySampler(model)(tokens, 9, lengths).tokens
  for graph in (True, False):
    assert torch.equal(rg.Sampler(model, temperature=0.0, use_cuda_graph=graph)(tokens, 9, lengths).tokens, greedy)
    assert torch.equal(rg.Sampler(model, top_k=1, use_cuda_graph=graph)(tokens, 9, lengths, uniforms=u).tokens, greedy)
  sampler = rg.Sampler(model, temperature=1.5, top_k=200, top_p=0.95)
  out = sampler(tokens, 9, lengths, return_logits=True, check_status=True, uniforms=u)
  for i in range(9):                          # each token is the draw from the logits of its step
    want = definition(out.logits[:, i], u[:, i], temperature=1.5, top_k=200, top_p=0.95)
    assert torch.equal(out.tokens[:, i], want), i
  assert torch.equal(rg.Sampler(model, temperature=1.5, top_k=200, top_p=0.95, use_cuda_graph=False)(
      tokens, 9, lengths, uniforms=u).tokens, out.tokens)
  # other settings, one for each sequence, through the graph that is there
  sampler.temperature = torch.tensor([0.0, 1.0, 3.0], device="cuda")
  sampler.top_k, sampler.top_p = torch.tensor([0, 5, 900], dtype=torch.int32, device="cuda"), 1.0
  again = sampler(tokens, 9, lengths, return_logits=True, uniforms=u)
  for i in range(9):
    want = definition(again.logits[:, i], u[:, i], temperature=sampler.temperature, top_k=sampler.top_k)
    assert torch.equal(again.tokens[:, i], want), i
  # numbers of its own: the generator decides
  draws = [sampler(tokens, 9, lengths, generator=torch.Generator(device="cuda").manual_seed(s)).tokens for s in (5, 5, 6)]
  assert torch.equal(draws[0], draws[1]) and not torch.equal(draws[0][2], draws[2][2])
  with pytest.raises(AssertionError):
    sampler(tokens, 9, lengths, uniforms=u[:, :8])
  with pytest.raises(TypeError):
    sampler(tokens, 9, lengths, uniforms=u.double())
  sampler.top_p = -1.0
  with pytest.raises(ValueError):
    sampler(tokens, 9, lengths)


@pytest.mark.gpu
def test_outputs_on_another_stream_and_device():
  """Operators follow the current stream, and the device of their tensors where that is not the current one."""
  import recurrentgemma_b200 as rg
  m = Layers()
  tokens = torch.arange(30, device="cuda")[None]
  want = m(tokens, *m.states_for(1))
  stream = torch.cuda.Stream()
  stream.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(stream):
    got = m(tokens, *m.states_for(1))
  stream.synchronize()
  assert all(torch.equal(p, q) for p, q in zip(want, got))
  if torch.cuda.device_count() > 1:
    other = torch.device("cuda", 1)
    logits, u = want[0][:, -1].to(other), torch.full((1,), 0.5, device=other)
    assert rg.sample(logits, u).device == other
