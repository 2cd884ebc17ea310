"""The two operators of a selective state space layer, beside `layers.Conv1D` and `layers.rnn_scan`: its short
causal convolution and its recurrence, for prompts, for continued chunks and for single tokens.

As everywhere in this package: inference only, CUDA only, float32 or bfloat16 with float32 states; a
`segment_pos` of 0 marks the first token of a document, and what lies in front of it does not reach behind it.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from recurrentgemma_b200 import _lib
from recurrentgemma_b200.layers import _pos, _same_dtype

_CONV_ACT = {None: _lib.CONV_ACT_NONE, "silu": _lib.CONV_ACT_SILU}


def _rows(t: torch.Tensor, dims: int) -> torch.Tensor:
  """`t` if its last `dims` dimensions are dense (the kernels take any batch and token stride), else a copy."""
  dense = 1
  for size, stride in zip(reversed(t.shape[-dims:]), reversed(t.stride()[-dims:])):
    if size != 1 and stride != dense:
      return t.contiguous()
    dense *= size
  return t


def _new_state(state: Optional[torch.Tensor], shape, dtype: torch.dtype, dev: torch.device,
               return_state: bool, inplace: bool) -> Optional[torch.Tensor]:
  if not inplace:
    return torch.empty(shape, dtype=dtype, device=dev) if return_state else None
  if state is None:
    raise ValueError("inplace=True needs a state to overwrite")
  if not state.is_contiguous():
    raise ValueError("inplace=True needs a contiguous state")
  return state


def _check_state(state: Optional[torch.Tensor], shape, dtype: torch.dtype) -> None:
  if state is None:
    return
  assert tuple(state.shape) == shape, (tuple(state.shape), shape)
  if state.dtype != dtype:
    raise TypeError(f"the state is {state.dtype}; this operator keeps it in {dtype}")


def causal_conv(
    x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor] = None, *,
    segment_pos: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
    activation: Optional[str] = "silu", return_state: bool = True, inplace: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
  """Depthwise causal convolution over time: (y [B,T,E], new state [B,W-1,E] or None).

  x [B,T,E]; w [W,E] with 2 to 4 taps, the last one on the token itself; b [E] or None; `activation` "silu" or
  None.  `state` holds the W-1 rows in front of x (None: zeros), so that a prompt may come in chunks and a
  decode step is a chunk of one token.  Taps do not reach over a document start; without `segment_pos` x
  begins none.  The new state has the same form, zero in rows that a document start in x hides from what
  comes next.  `inplace` overwrites `state` and returns it (a step that a CUDA graph can replay).
  x may be strided over batch and time, as a part of a wider projection is.
  """
  done = _lib.host().causal_conv(x, w, b, segment_pos, state, activation, return_state, inplace)
  if done is not NotImplemented:
    return done
  return _causal_conv(x, w, b, segment_pos, state, activation, return_state, inplace)


@torch.no_grad()
def _causal_conv(x, w, b, segment_pos, state, activation, return_state, inplace):
  dev = _lib.require_cuda(x, w, b, segment_pos, state)
  dt = _lib.dtype_code(x.dtype)
  assert x.ndim == 3 and w.ndim == 2 and w.shape[1] == x.shape[2], (x.shape, w.shape)
  bs, l, e = x.shape
  taps = w.shape[0]
  if activation not in _CONV_ACT:
    raise ValueError(f"activation {activation!r}: 'silu' or None")
  _same_dtype(x, *(p for p in (w, b) if p is not None))
  assert b is None or b.shape == (e,), (b.shape, e)
  _check_state(state, (bs, taps - 1, e), x.dtype)
  pos = None if segment_pos is None else _pos(segment_pos, bs, l)
  new_state = _new_state(state, (bs, taps - 1, e), x.dtype, dev, return_state, inplace)
  xc, wc = _rows(x, 1), w.contiguous()
  bc = None if b is None else b.contiguous()
  sc = None if state is None else state.contiguous()
  y = torch.empty((bs, l, e), dtype=x.dtype, device=dev)
  with torch.cuda.device(dev):
    _lib.check(_lib.load().rgk_causal_conv(
        xc.data_ptr(), xc.stride(0), xc.stride(1), _lib.ptr(pos), 0 if pos is None else _lib.pos_code(pos),
        wc.data_ptr(), _lib.ptr(bc), _lib.ptr(sc), bs, l, e, taps, _CONV_ACT[activation], dt, y.data_ptr(),
        _lib.ptr(new_state), _lib.stream_ptr(dev)))
  return y, (new_state if return_state else None)


def selective_scan(
    x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, *,
    d: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
    dt_bias: Optional[torch.Tensor] = None, segment_pos: Optional[torch.Tensor] = None,
    state: Optional[torch.Tensor] = None, softplus: bool = True, return_state: bool = True,
    inplace: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
  """The selective state space recurrence: (y [B,T,E] in x.dtype, last state [B,E,N] float32 or None).

    step = softplus(dt + dt_bias)          (dt + dt_bias with softplus=False)
    h_t  = exp(step_t a) h_{t-1} + step_t x_t b_t,    y_t = (<h_t, c_t> + d x_t) silu(z_t)

  x, dt and z (or None) [B,T,E]; b, c [B,T,G,N], channel e using group e // (E // G), N up to 256; a [E,N],
  d [E] and dt_bias [E] float32 (a is the decay rate itself, negative in trained layers).  `state` [B,E,N]
  float32 is h in front of the first token (None: zeros); a decode step is a call with one token.  A document
  start (segment_pos == 0) drops the state in front of it.  `inplace` overwrites `state` and returns it.
  Decay factors and steps are float32 evaluations as exact as the formula's in float32; bfloat16 calls with more than
  4 states take the hardware's exponential for the factors: after 2048 steps their states are 3e-7 off 64 bits
  (2-norm), where float32 calls are 1.5e-7.
  x, dt, z, b and c may be strided over batch and time.  Where x or a step is infinite, y may be NaN instead of
  infinite; the states are as the formula has them.
  """
  done = _lib.host().selective_scan(x, dt, a, b, c, d, z, dt_bias, segment_pos, state, softplus, return_state,
                                    inplace)
  if done is not NotImplemented:
    return done
  return _selective_scan(x, dt, a, b, c, d, z, dt_bias, segment_pos, state, softplus, return_state, inplace)


@torch.no_grad()
def _selective_scan(x, dt, a, b, c, d, z, dt_bias, segment_pos, state, softplus, return_state, inplace):
  dev = _lib.require_cuda(x, dt, a, b, c, d, z, dt_bias, segment_pos, state)
  code = _lib.dtype_code(x.dtype)
  assert x.ndim == 3 and dt.shape == x.shape and (z is None or z.shape == x.shape), (x.shape, dt.shape)
  bs, l, e = x.shape
  assert b.ndim == 4 and b.shape[:2] == (bs, l) and c.shape == b.shape, (b.shape, c.shape)
  groups, n = b.shape[2:]
  assert a.shape == (e, n), (a.shape, (e, n))
  assert groups >= 1 and e % groups == 0, (e, groups)
  for p in (d, dt_bias):
    assert p is None or p.shape == (e,), (p.shape, e)
  _same_dtype(x, *(t for t in (dt, b, c, z) if t is not None))
  for p in (a, d, dt_bias):
    if p is not None and p.dtype != torch.float32:
      raise TypeError(f"a, d and dt_bias are float32 whatever the activations, got {p.dtype}")
  _check_state(state, (bs, e, n), torch.float32)
  pos = None if segment_pos is None else _pos(segment_pos, bs, l)
  # (long calls hand states from chunk to chunk in it, whether it is returned or not)
  new_state = _new_state(state, (bs, e, n), torch.float32, dev, True, inplace)
  held = [None if t is None else _rows(t, 1) for t in (x, dt, z)] + [_rows(t, 2) for t in (b, c)]
  params = [None if p is None else p.contiguous() for p in (a, d, dt_bias)]
  sc = None if state is None else state.contiguous()
  y = torch.empty((bs, l, e), dtype=x.dtype, device=dev)
  p = _lib.RgkScanInputs(
      *(_lib.ptr(t) for t in held),
      *(s for t in held for s in ((0, 0) if t is None else (t.stride(0), t.stride(1)))),
      *(_lib.ptr(t) for t in params), int(softplus))
  with torch.cuda.device(dev):
    lib = _lib.load()
    # (a long call has scratch of its own: captured calls may be replayed side by side)
    ws = (torch.empty(lib.rgk_selective_scan_workspace_bytes(), dtype=torch.uint8, device=dev)
          if l >= _lib.SCAN_CHUNKS_FROM else None)
    _lib.check(lib.rgk_selective_scan(
        ctypes.byref(p), _lib.ptr(pos), 0 if pos is None else _lib.pos_code(pos), _lib.ptr(sc), bs, l, e,
        groups, n, code, y.data_ptr(), new_state.data_ptr(), _lib.ptr(ws), 0 if ws is None else ws.numel(),
        _lib.status_ptr(dev), _lib.stream_ptr(dev)))
  return y, (new_state if return_state else None)
