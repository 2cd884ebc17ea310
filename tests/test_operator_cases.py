"""The operator cases' inputs are made from their seed alone, as a comparison of two programs' outputs needs."""
import importlib.util
import os
import random

import pytest
import torch


def _cases():
  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
  spec = importlib.util.spec_from_file_location("operator_cases", path)
  module = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(module)
  return module


def _same(p, q):
  if isinstance(p, dict):
    return p.keys() == q.keys() and all(_same(p[k], q[k]) for k in p)
  return torch.equal(p, q) if torch.is_tensor(p) else p == q


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(256, 1000), (256, 3001), (33, 32_003), (4, 256_000)])
@pytest.mark.parametrize("mixed", [False, True])
def test_inputs_of_sampling_go_by_their_seed(rows, vocab, mixed):
  cases = _cases()
  case = dict(op="sample", dtype="float32", rows=rows, vocab=vocab, temperature=0.9, top_k=40, top_p=0.8,
              min_p=0.05, mixed=mixed)
  first = cases.prepare(case, 5)
  for _ in range(10):
    assert _same(first, cases.prepare(case, 5))
  assert not _same(first, cases.prepare(case, 6))


@pytest.mark.gpu
def test_inputs_of_sequences_go_by_their_seed():
  cases, rng, seen = _cases(), random.Random(3), set()
  while len(seen) < 6:
    case = cases.draw(rng)
    if case["op"] == "sample" or case["batch"] * case["seq"] * case["width"] > 1 << 24:
      continue
    seen.add(str(case))
    first = cases.prepare(case, 7)
    assert all(_same(first, cases.prepare(case, 7)) for _ in range(3))
