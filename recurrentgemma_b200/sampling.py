"""Drawing the next token from logits, beside `modules.argmax`."""
from __future__ import annotations

import ctypes
import math
from typing import Dict, Optional, Union

import torch

from recurrentgemma_b200 import _lib


def check_settings(temperature, top_k, top_p, min_p, shape) -> Dict[str, Union[float, int, torch.Tensor]]:
  """The settings by name, if each is a number in its range or a tensor of the given shape and its type."""
  settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
  for name, value in settings.items():
    if torch.is_tensor(value):
      dtype = torch.int32 if name == "top_k" else torch.float32
      if value.dtype != dtype:
        raise TypeError(f"{name} is {value.dtype}: one value for each row is {dtype}")
      assert value.shape == shape, (name, value.shape, shape)
    elif name == "top_k":
      settings[name] = max(-1, min(int(value), 2**31 - 1))
    elif not 0.0 <= value <= (1.0 if name == "min_p" else math.inf):
      raise ValueError(f"{name} {value}: a temperature and top_p are at least 0, min_p is from 0 to 1")
  return settings


def sample(
    logits: torch.Tensor, uniforms: torch.Tensor,
    temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
    top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
  """One token (int32) for every row of logits [..., V], drawn by the row's uniform number in [0, 1).

  Tokens are ordered by logit, largest first, equal ones by index.  Kept are the first `top_k` (0: all); of
  those, with weights exp((logit - largest) / temperature), the shortest prefix with at least `top_p` of their
  weight (1: all); of those the ones with at least `min_p` of the largest weight.  Weights are held as multiples of
  2**-44 (2**-43 above 2**18 tokens, 2**-42 above 2**19), each within one of those.  The token is the first by index up to which the kept weights sum to
  more than `uniforms` times all of them.  Temperature 0 takes the first maximum.
  NaN counts as -inf and neither is ever drawn; a row of nothing else gives 0.

  Each setting is a number, or a tensor with one for each row (float32; `top_k` int32).  `uniforms` is
  float32 [...].  The result does not depend on how many rows are drawn together.  V up to 2**20.
  """
  done = _lib.host().sample(logits, uniforms, temperature, top_k, top_p, min_p, out)
  if done is not NotImplemented:
    return done
  return _sample(logits, uniforms, temperature, top_k, top_p, min_p, out)


@torch.no_grad()
def _sample(logits, uniforms, temperature, top_k, top_p, min_p, out):
  settings = check_settings(temperature, top_k, top_p, min_p, logits.shape[:-1])
  dev = _lib.require_cuda(logits, uniforms, *(s for s in settings.values() if torch.is_tensor(s)), out)
  v = logits.shape[-1]
  if uniforms.dtype != torch.float32:
    raise TypeError(f"uniforms are {uniforms.dtype}, not float32")
  assert uniforms.shape == logits.shape[:-1], (uniforms.shape, logits.shape)
  rows = {n: s.contiguous() if torch.is_tensor(s) else None for n, s in settings.items()}
  numbers = {n: 0 if torch.is_tensor(s) else s for n, s in settings.items()}
  x = logits if logits.ndim == 2 and logits.stride(1) == 1 else logits.contiguous()
  uc = uniforms.contiguous()
  if out is None:
    out = torch.empty(logits.shape[:-1], dtype=torch.int32, device=dev)
  assert out.shape == logits.shape[:-1] and out.dtype == torch.int32 and out.is_contiguous()
  p = _lib.RgkSampleSettings(**{n: _lib.ptr(r) for n, r in rows.items()},
                             **{f"{n}_value": value for n, value in numbers.items()})
  with torch.cuda.device(dev):
    _lib.check(_lib.load().rgk_sample(
        x.data_ptr(), uc.numel(), v, x.stride(0) if x.ndim == 2 else v, _lib.dtype_code(logits.dtype),
        uc.data_ptr(), ctypes.byref(p), out.data_ptr(), _lib.stream_ptr(dev)))
  return out
