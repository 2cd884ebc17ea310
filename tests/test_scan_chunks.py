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


# More blocks of channels (128 a CTA at most, two CTAs an SM) than CTAs, and 512 steps or more: time is cut, whichever
# shape the number of states has.  Rows aligned to copies of 16 bytes, but for the last ones.
CHUNKED = [
    # b, t, e, n, groups, doc, options
    (8, 520, 5120, 16, 1, 90, {}),
    (8, 641, 5120, 16, 1, 0, dict(state=False, z=False)),
    (8, 520, 5120, 3, 1, 200, {}),
    (8, 520, 5120, 8, 2, 90, {}),
    (8, 520, 5120, 32, 1, 90, {}),
    (4, 530, 5120, 64, 1, 300, {}),
    (4, 520, 2560, 128, 1, 90, {}),
    (2, 513, 2560, 256, 1, 0, {}),
    (8, 515, 5130, 16, 2, 90, dict(part=True)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,e,n,groups,doc,options", CHUNKED)
def test_scan_in_chunks_of_time(b, t, e, n, groups, doc, options, dtype):
  """Against the definition, the state passed on beside the one that was given and over it."""
  import recurrentgemma_b200 as rg
  from tests.test_state_space import scan_case, scan_definition, within
  case = scan_case(t + n, b, t, e, n, dtype, groups, doc, **options)
  want, held, bound, bound_state = scan_definition(**case)
  y, state = rg.selective_scan(**case)
  within(y, want, bound, dtype)
  within(state, held, bound_state, torch.float32)
  given = torch.zeros(b, e, n, device="cuda") if case["state"] is None else case["state"].clone()
  again, back = rg.selective_scan(**{**case, "state": given}, inplace=True)
  assert back is given and torch.equal(back, state) and torch.equal(again, y)
  rg.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("taps,doc,half", [(4, 0, True), (4, 30, False), (3, 0, False), (2, 500, True)])
def test_convolution_of_a_prefill_batch(taps, doc, half, dtype):
  """Large enough for a thread's longest run of rows, in packs: 16 a thread, which 12 M elements and more take."""
  import recurrentgemma_b200 as rg
  from tests.test_state_space import conv_case, conv_definition, within
  b, t, e = 6, 803, 2560
  case = conv_case(taps + doc, b, t, e, taps, dtype, doc)
  if half:                                           # (one half of a projection's output)
    case["x"] = torch.cat([case["x"], case["x"]], -1)[..., :e]
  want, held, bound = conv_definition(**case)
  y, state = rg.causal_conv(**case)
  within(y, want, bound, dtype)
  assert torch.equal(state.double(), held)
  given = case["state"].clone()
  again, back = rg.causal_conv(**{**case, "state": given}, inplace=True)
  assert back is given and torch.equal(back, state) and torch.equal(again, y)


@pytest.mark.parametrize("name", ["causal_conv.cu", "selective_scan.cu", "sample.cu"])
def test_launchers_ask_for_the_number_of_sms(name):
  """No kernel is chosen by the number of SMs of one device."""
  with open(os.path.join(CSRC, name)) as f:
    text = re.sub(r"//[^\n]*", "", f.read())
  text = re.sub(r"constexpr Choice \w+\[\] = [^;]*;", "", text)          # (tables of times)
  assert not re.search(r"\b148\b", text)


def test_length_from_which_scratch_is_used():
  """The one of the header, on both sides."""
  from recurrentgemma_b200 import _lib
  root = os.path.dirname(os.path.dirname(os.path.dirname(CSRC + "/")))
  with open(os.path.join(root, "include", "rgk.h")) as f:
    assert int(re.search(r"RGK_SCAN_CHUNKS_FROM = (\d+)", f.read())[1]) == _lib.SCAN_CHUNKS_FROM


@pytest.mark.gpu
def test_short_scans_take_no_scratch():
  """In Python's form of the call, which strided states and the like take, as in the native one."""
  import recurrentgemma_b200 as rg
  from recurrentgemma_b200 import _lib
  from tests.test_state_space import scan_case
  for t in (1, 40):
    case = scan_case(t, 2, t, 64, 16, torch.bfloat16)
    want = rg.selective_scan(**case)
    wide = torch.empty((2, 64, 32), device="cuda")
    wide[..., :16] = case["state"]
    case["state"] = wide[..., :16]
    rg.selective_scan(**case)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = rg.selective_scan(**case)
    assert torch.cuda.max_memory_allocated() - held < _lib.load().rgk_selective_scan_workspace_bytes()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
def test_a_wait_for_a_chunk_expires_and_is_reported():
  """A call in chunks whose first chunk is never run: the wait for it gives up after 200 polls, the kernel returns, and
  check_status reports it once; the next call is right."""
  import recurrentgemma_b200 as rg
  from recurrentgemma_b200 import _lib
  from tests.test_state_space import scan_case
  dev = torch.device("cuda", torch.cuda.current_device())
  lib = _lib.load()
  case = scan_case(3, 8, 520, 5120, 16, torch.bfloat16)
  want = rg.selective_scan(**case)
  rg.check_status(dev)
  scratch = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
  _lib.check(lib.rgk_selftest_scan_wait_expiry(scratch.data_ptr(), scratch.numel(), _lib.status_ptr(dev),
                                               _lib.stream_ptr(dev)))
  torch.cuda.synchronize()                          # the kernel has returned by itself
  with pytest.raises(_lib.RgkError) as err:
    rg.check_status(dev)
  assert err.value.code == _lib.RGK_ETIMEOUT
  rg.check_status(dev)                              # reported once
  got = rg.selective_scan(**case)
  rg.check_status(dev)
  assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
def test_range_checked_build_runs_scans_clean():
  """librgk_checks.so checks the indices of states, outputs and chunk counters: a bad one would skip its access and show
  in the status word and the results of the tests that are run on it here."""
  import subprocess
  import sys
  root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
  lib_path = os.path.join(root, "recurrentgemma_b200", "librgk_checks.so")
  if not os.path.exists(lib_path):
    pytest.skip("librgk_checks.so not built (python -m recurrentgemma_b200.build --checks)")
  env = dict(os.environ, RGK_LIBRARY=lib_path)
  cmd = [sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", os.path.join(root, "tests", "test_scan_chunks.py"),
         os.path.join(root, "tests", "test_state_space.py"), "-k", "in_chunks or test_selective_scan or test_causal_conv",
         "-p", "no:cacheprovider"]
  r = subprocess.run(cmd, env=env, cwd=root, capture_output=True, text=True, timeout=600)
  assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
  assert " passed" in r.stdout


def test_refusals_of_the_self_test():
  from recurrentgemma_b200 import _lib, build
  build.build_library()
  lib = _lib.load()
  assert lib.rgk_selftest_scan_wait_expiry(None, 1 << 20, None, None) == _lib.RGK_EWORKSPACE
  assert lib.rgk_selftest_scan_wait_expiry(256, 1 << 18, None, None) == _lib.RGK_EWORKSPACE
  assert lib.rgk_selftest_scan_wait_expiry(128, 1 << 20, None, None) == _lib.RGK_EALIGN
  assert lib.rgk_selftest_scan_wait_expiry(256, 1 << 20, 18, None) == _lib.RGK_EALIGN


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,e,n,options", [
    (3, 70, 5120, 8, {}), (3, 70, 5120, 16, dict(part=True)), (1, 70, 2560, 64, {}), (1, 70, 2560, 128, {}),
    (2, 70, 1280, 32, {}), (1, 70, 1024, 128, dict(part=True))])
def test_shapes_between_one_round_of_sms_and_two(b, t, e, n, options, dtype):
  import recurrentgemma_b200 as rg
  from tests.test_state_space import scan_case, scan_definition, within
  case = scan_case(n, b, t, e, n, dtype, 1, 20, **options)
  y, state = rg.selective_scan(**case)
  want, held, bound, bound_state = scan_definition(**case)
  within(y, want, bound, dtype)
  within(state, held, bound_state, torch.float32)
