"""Drawing the next token from logits, beside `modules.argmax`."""
from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from recurrentgemma_b200 import _lib


def _per_row(name: str, value, dtype: torch.dtype, logits: torch.Tensor) -> Optional[torch.Tensor]:
  """A setting given for each row as a dense tensor; None if it is one number for all."""
  if not torch.is_tensor(value):
    return None
  if value.dtype != dtype:
    raise TypeError(f"{name} is {value.dtype}: one value for each row is {dtype}")
  assert value.shape == logits.shape[:-1], (name, value.shape, logits.shape)
  return value.contiguous()


def sample(
    logits: torch.Tensor, uniforms: torch.Tensor,
    temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
    top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
  """One token (int32) for every row of logits [..., V], drawn by the row's uniform number in [0, 1).

  Tokens are ordered by logit, largest first, equal ones by index.  Kept are the first `top_k` (0: all); of
  those, with weights exp((logit - largest) / temperature) rounded to multiples of 2**-44 (2**-42 from 2**18
  tokens on), the shortest prefix with at least `top_p` of their weight (1: all); of those the ones with at
  least `min_p` of the largest weight.  The token is the first by index up to which the kept weights sum to
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
  settings = (temperature, top_k, top_p, min_p)
  dev = _lib.require_cuda(logits, uniforms, *(s for s in settings if torch.is_tensor(s)), out)
  v = logits.shape[-1]
  if uniforms.dtype != torch.float32:
    raise TypeError(f"uniforms are {uniforms.dtype}, not float32")
  assert uniforms.shape == logits.shape[:-1], (uniforms.shape, logits.shape)
  rows = [_per_row(name, value, torch.int32 if name == "top_k" else torch.float32, logits)
          for name, value in zip(("temperature", "top_k", "top_p", "min_p"), settings)]
  numbers = [value if row is None else 0 for value, row in zip(settings, rows)]
  if not numbers[0] >= 0 or not numbers[2] >= 0 or not 0 <= numbers[3] <= 1:
    raise ValueError(f"temperature {numbers[0]}, top_p {numbers[2]}, min_p {numbers[3]}: a temperature and top_p "
                     "of at least 0, min_p from 0 to 1")
  x = logits if logits.ndim == 2 and logits.stride(1) == 1 else logits.contiguous()
  uc = uniforms.contiguous()
  if out is None:
    out = torch.empty(logits.shape[:-1], dtype=torch.int32, device=dev)
  assert out.shape == logits.shape[:-1] and out.dtype == torch.int32 and out.is_contiguous()
  p = _lib.RgkSampleSettings(*(_lib.ptr(r) for r in rows), float(numbers[0]), min(int(numbers[1]), 2**31 - 1),
                             float(numbers[2]), float(numbers[3]))
  with torch.cuda.device(dev):
    _lib.check(_lib.load().rgk_sample(
        x.data_ptr(), uc.numel(), v, x.stride(0) if x.ndim == 2 else v, _lib.dtype_code(logits.dtype),
        uc.data_ptr(), ctypes.byref(p), out.data_ptr(), _lib.stream_ptr(dev)))
  return out
