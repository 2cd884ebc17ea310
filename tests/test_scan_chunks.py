"""Selective scans that cut time into chunks: a chunk waits for the one before it, so that one must be running already."""
import os
import re

import pytest
import torch

from tests.test_dependent_launches import CSRC, _kernels


def test_every_chunk_is_drawn_by_a_ticket():
  """A CTA's first item too: with items by the CTA's number a started CTA could wait for one that never starts, because
  the waiting ones hold its place."""
  with open(os.path.join(CSRC, "selective_scan.cu")) as f:
    text = re.sub(r"//[^\n]*", "", f.read())
  body, = [body for kernel, _, body in _kernels(text) if kernel == "selective_scan_kernel"]
  assert re.search(r"atomicAdd\(p\.ticket, 1u\)", body)
  assert re.findall(r"[^\n]*blockIdx[^\n]*", body) == [
      "  for (int64_t item = p.chunks == 1 ? blockIdx.x : draw(); item < items;) {"]
  assert "gridDim" not in body


@pytest.mark.gpu
def test_chunks_where_only_a_part_of_the_grid_finds_a_place():
  """While a long call holds a part of the device, two calls in chunks start on it, the later one of higher priority:
  it takes the places that become free, so that the earlier one stays partly placed.  Every result is that of the
  call alone, and no wait ran out."""
  import recurrentgemma_b200 as rg
  from tests.test_state_space import scan_case
  long = scan_case(1, 1, 16, 5120, 16, torch.bfloat16, z=False)
  t = 20_000                                       # (one token's values over and over: strides of 0)
  long.update({k: long[k][:, :1].expand(1, t, *long[k].shape[2:]) for k in ("x", "dt", "b", "c")})
  cases = [scan_case(seed, 8, 520, 5120, 16, torch.bfloat16, doc=90) for seed in (2, 3)]
  want = [rg.selective_scan(**c) for c in cases]
  held = rg.selective_scan(**long)
  low, high = torch.cuda.Stream.priority_range()
  streams = [torch.cuda.Stream(priority=p) for p in (low, low, high)]
  torch.cuda.synchronize()
  for _ in range(6):
    got = []
    for c, stream in zip((long, *cases), streams):
      with torch.cuda.stream(stream):
        got.append(rg.selective_scan(**c))
    torch.cuda.synchronize()
    rg.check_status()
    for g, w in zip(got, (held, *want)):
      assert all(torch.equal(p, q) for p, q in zip(g, w))
