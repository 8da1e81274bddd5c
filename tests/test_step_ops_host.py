"""The self-attention step's operators without a GPU, continued: what a build depends on, and the bounds that the GPU tests use."""
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from matvec_bounds import fp32_rms_bound, rms_error


def cut(x, parts):
  """What `parts` bfloat16, each the leading 8 bits of what the ones before left, hold of fp32 numbers."""
  held, rest = torch.zeros_like(x), x.clone()
  for _ in range(parts):
    part = (rest.view(torch.int32) & -65536).view(torch.float32)
    held, rest = held + part, rest - part
  return held


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,vectors", [(80, 1558, 1), (300, 512, 16), (33, 127, 65)])
def test_the_bound_of_fp32_products_tells_lost_bits(group, zeros, n, k, vectors):
  """Products with plain fp32 sums keep the bound; vectors of two parts instead of three, of float16, and results of float16 do not."""
  g = torch.Generator().manual_seed(n + group)
  groups = -(-k // group)
  spread = lambda t: t.repeat_interleave(group, 1)[:, :k]  # noqa: E731
  c = torch.randint(0, 16, (n, k), generator=g).double()
  z = torch.randint(0, 16, (n, groups), generator=g).double() if zeros else torch.full((n, groups), 8.0).double()
  s = torch.rand(n, groups, generator=g) * 0.1 + 0.01
  w = (c - spread(z)) * spread(s.double())
  x = torch.randn(vectors, k, generator=g)
  want = x.double() @ w.t()
  bound = fp32_rms_bound(group, groups, zeros)
  sums = torch.zeros(vectors, n)
  for i in range(groups):
    at = slice(i * group, min(k, (i + 1) * group))
    sums += s[:, i] * (x[:, at] @ c[:, at].float().t() - z[:, i].float() * x[:, at].sum(1, keepdim=True))
  assert rms_error(sums, want) <= bound
  assert torch.equal(cut(x, 3), x)
  for wrong in (cut(x, 2).double() @ w.t(), x.half().double() @ w.t(), want.half()):
    assert rms_error(wrong, want) > 2 * bound


def test_objects_are_built_again_when_the_flags_change():
  """The flags stand in the makefiles (in the product's, the one that keeps packed fp32 arithmetic out)."""
  for folder, target in (("tacotron_amd/csrc", "taco_qmat.o"), ("tests/support", "libhold_cu.so"), ("tests/support", "libplace.so")):
    told = subprocess.check_output(["make", "-n", "-W", "Makefile", "-C", os.path.join(ROOT, folder), target], text=True)
    assert "-o " + target in told, (folder, told)


def test_a_build_compiles_whatever_is_there(monkeypatch):
  import __graft_entry__
  calls = []
  monkeypatch.setattr(__graft_entry__.subprocess, "check_call", lambda args, **kw: calls.append(args))
  __graft_entry__.build()
  assert len(calls) == 3 and all(args[0] == "make" and "-B" in args for args in calls)


def test_the_host_library_is_as_new_as_its_sources():
  """What test_step_ops.py loads has been compiled from the kernels' header as it is now."""
  age = lambda *path: os.path.getmtime(os.path.join(ROOT, *path))  # noqa: E731
  assert age("tests", "support", "libplace.so") >= max(age("tests", "support", "place.cpp"), age("tacotron_amd", "csrc", "taco_place.h"))
