"""The self-attention step's operators on the GPU, continued: every form of the kernels, the ends of the range of numbers, calls
that meet each other.  Tolerances as in test_gpu_step_ops.py."""
import ctypes as C
import math

import pytest
import torch

from matvec_bounds import fp32_rms_bound, rms_error
from test_gpu_step_ops import (BF16, DEV, E4M3, F16, F32, attend_case, check_attend, check_matvec, gen,
                               half_step, make_cache, make_codes)

pytestmark = pytest.mark.gpu


# ---- products -----------------------------------------------------------------------------------------------------------


def product_64(codes, scales, zeros, group, x):
  k = codes.shape[1]
  spread = lambda t: t.double().repeat_interleave(group, 1)[:, :k]  # noqa: E731
  return x.double() @ ((codes.double() - (8.0 if zeros is None else spread(zeros))) * spread(scales)).t()


# vectors, rows: up to a row block per CU, up to two, more; the same with more than a tile of vectors (256 CUs)
FORMS = [(1, 40), (3, 4200), (2, 8300), (20, 2100), (20, 4200), (33, 8300)]


@pytest.mark.parametrize("scale_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_every_form_of_the_product(dtype, group, scale_dtype):
  """Each way of dividing rows and vectors, with and without zero points, vectors at even and at odd addresses."""
  from tacotron_amd.w4 import W4Matrix
  k = 300
  for vectors, n in FORMS:
    for zeros in (False, True):
      g = gen(n + group)
      codes, packed, scales, z = make_codes(n, k, group, scale_dtype, zeros, g)
      W = W4Matrix.from_codes(packed, scales, zeros=z, in_features=k, group=group)
      x = torch.randn(vectors, k, generator=g, device=DEV).to(dtype)
      got = W.matvec(x)
      check_matvec(codes, scales, z, group, None, x, got)
      if dtype == F32:
        assert rms_error(got, product_64(codes, scales, z, group, x)) <= fp32_rms_bound(group, scales.shape[1], zeros), (vectors, n, zeros)
      wide = torch.full((vectors, k + 3), float("nan"), dtype=dtype, device=DEV)
      wide[:, 1:k + 1] = x
      assert torch.equal(W.matvec(wide[:, 1:k + 1]), got), (vectors, n, zeros)


@pytest.mark.parametrize("n,k,vectors,group,zeros", [
  (80, 1558, 1, 32, False), (4096, 1558, 16, 64, False), (8249, 9077, 1, 128, False), (33, 127, 65, 32, True), (4100, 257, 40, 128, True),
  (100, 20000, 3, 64, True)])
def test_fp32_products_keep_their_bits(n, k, vectors, group, zeros):
  from tacotron_amd.w4 import W4Matrix
  g = gen(n + k)
  codes, packed, scales, z = make_codes(n, k, group, F32, zeros, g)
  x = torch.randn(vectors, k, generator=g, device=DEV)
  got = W4Matrix.from_codes(packed, scales, zeros=z, in_features=k, group=group).matvec(x)
  assert rms_error(got, product_64(codes, scales, z, group, x)) <= fp32_rms_bound(group, scales.shape[1], zeros)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_largest_finite_vectors(dtype, group):
  """Vectors up to the largest finite number: the result is finite wherever the formula's is, whatever a group's sums before scaling are."""
  from tacotron_amd.w4 import W4Matrix
  most = torch.finfo(dtype).max
  for vectors, n, k in ((1, 40, 300), (17, 4200, 256), (2, 8300, 129)):
    for zeros in (False, True):
      g = gen(n + group)
      codes, packed, scales, z = make_codes(n, k, group, F32, zeros, g)
      scales *= 2.0 ** -20            # sums of |w x| stay below the largest number
      W = W4Matrix.from_codes(packed, scales, zeros=z, in_features=k, group=group)
      x = (1 - torch.rand(vectors, k, generator=g, device=DEV) / 4).to(dtype) * most
      for signed in (x, x * torch.where(torch.rand(x.shape, generator=g, device=DEV) < 0.5, -1, 1).to(dtype)):
        got = W.matvec(signed)
        assert torch.isfinite(got).all(), (vectors, n, zeros)
        check_matvec(codes, scales, z, group, None, signed, got)


@pytest.mark.parametrize("size", [1e-29, 1e-32])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_small_vectors_keep_their_bits(dtype, size):
  """Small vectors are as exact as any: the last bits of an fp32 number of 1e-32, 1e-39, times a code held as 2^-12 are subnormal numbers."""
  from tacotron_amd.w4 import W4Matrix
  g = gen(2)
  for zeros in (False, True):
    codes, packed, scales, z = make_codes(200, 512, 64, F32, zeros, g)
    W = W4Matrix.from_codes(packed, scales, zeros=z, in_features=512, group=64)
    x = (torch.randn(4, 512, generator=g, device=DEV) * size).to(dtype)
    error = rms_error(W.matvec(x), product_64(codes, scales, z, 64, x))
    assert error <= fp32_rms_bound(64, 8, zeros) + (half_step(BF16) if dtype == BF16 else 0), (zeros, error)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_as_many_vectors_as_there_may_be(dtype):
  """2^20 vectors of a small matrix: a launch's second dimension at its largest."""
  from tacotron_amd.w4 import W4Matrix
  g = gen(3)
  codes, packed, scales, z = make_codes(16, 32, 32, F32, True, g)
  W = W4Matrix.from_codes(packed, scales, zeros=z, group=32)
  x = torch.randn(1 << 20, 32, generator=g, device=DEV).to(dtype)
  got = W.matvec(x)
  for rows in (slice(0, 1 << 12), slice((1 << 19) - 100, (1 << 19) + 100), slice((1 << 20) - (1 << 12), 1 << 20)):
    check_matvec(codes, scales, z, 32, None, x[rows], got[rows])
  assert bool(torch.isfinite(got).all())


def test_quantize_weights_whose_scale_leaves_its_type():
  """Finite weights give finite matrices: a range beyond fp32, scales beyond float16."""
  from tacotron_amd import w4
  most = torch.finfo(F32).max
  w = torch.tensor([[most, -most, most / 2, 0.0], [most, -most / 3, 1.0, -1.0], [3.0, -4.0, 0.5, 0.0]], device=DEV)
  codes, scales, zeros = w4.quantize(w, 32, symmetric=False)
  s = torch.stack([(w.double().amax(1) - w.double().amin(1)) / 15], 1)
  assert ((scales.double() - s).abs() <= 3 * 2.0 ** -24 * s).all()
  unpacked = torch.stack([codes & 15, codes >> 4], -1).flatten(1).double()
  back = (unpacked - zeros.double()) * scales.double()
  assert ((back - w.double()).abs() <= s * (0.5 + 0.5 + 1e-5)).all()          # the zero point is rounded, and the code
  w = torch.tensor([[1e6, -2e6, 3e5, 0.0], [4e5, 1.0, -4e5, 65504.0]], device=DEV)
  for symmetric in (True, False):
    codes, scales, zeros = w4.quantize(w, 32, symmetric=symmetric, scale_dtype=F16)
    assert scales[0, 0].item() == 65504 and bool(torch.isfinite(scales).all())
    z = torch.full((2, 1), 8.0) if symmetric else zeros.cpu().float()
    want = ((w.cpu() / scales.cpu().float()).round() + z).clamp(0, 15)
    assert torch.equal(torch.stack([codes & 15, codes >> 4], -1).flatten(1).cpu().float(), want)
    W = w4.W4Matrix.from_codes(codes, scales, zeros=zeros, in_features=4, group=32)
    assert bool(torch.isfinite(W.matvec(torch.ones(1, 4, device=DEV))).all())


# ---- attend -------------------------------------------------------------------------------------------------------------

EDGES = [0, 1, 15, 16, 17, 33, 64, 65, 128, 129, 300]
INSTANCES = [
  # dtype, cache, heads, query heads, d, page, lens, window, order: types and head sizes with more than 16 query heads a cache head, and without
  (F16, F16, 2, 40, 64, 16, EDGES, 0, "own"),
  (F16, F16, 1, 5, 256, 32, EDGES, 40, "tokens"),
  (F16, F16, 2, 50, 256, 16, EDGES, 0, "heads"),
  (F16, F16, 1, 17, 144, 48, [700, 5], 0, "own"),
  (F16, F16, 2, 34, 128, 16, EDGES, 0, "wide"),
  (BF16, BF16, 2, 64, 128, 64, EDGES, 0, "own"),
  (BF16, BF16, 2, 48, 256, 16, EDGES, 0, "own"),
  (BF16, BF16, 1, 33, 208, 32, [1000, 0, 31], 130, "wide"),
  (BF16, BF16, 1, 71, 128, 16, [2000, 3], 0, "tokens"),
  (BF16, BF16, 3, 9, 64, 16, EDGES, 0, "own"),
  (F16, E4M3, 2, 66, 64, 32, EDGES, 0, "own"),
  (F16, E4M3, 3, 6, 128, 16, EDGES, 20, "tokens"),
  (F16, E4M3, 1, 4, 256, 16, EDGES, 0, "own"),
  (F16, E4M3, 1, 20, 112, 16, EDGES, 0, "own"),
  (BF16, E4M3, 4, 8, 64, 16, EDGES, 0, "heads"),
  (BF16, E4M3, 1, 24, 48, 16, EDGES, 0, "own"),
  (BF16, E4M3, 2, 40, 128, 32, EDGES, 65, "own"),
  (BF16, E4M3, 2, 36, 256, 48, EDGES, 0, "wide"),
  (F32, F32, 2, 34, 64, 16, EDGES, 0, "own"),
  (F32, F32, 1, 3, 160, 16, EDGES, 0, "tokens"),
]


@pytest.mark.parametrize("dtype,held,heads,hq,d,page,lens,window,order", INSTANCES)
def test_every_form_of_the_attention(dtype, held, heads, hq, d, page, lens, window, order):
  cache, q, table, lens_dev = attend_case(dtype, held, heads, hq, d, page, lens, window, order)
  got = cache.attend(q, table, lens_dev, window=window, return_lse=True)
  cache.check()
  check_attend(cache, q, table, lens, d ** -0.5, window, got)
  assert cache.attend(q, table, lens_dev, window=window, out=q) is q and torch.equal(q, got[0])


def captured_nodes(call):
  """How many nodes a call leaves in a graph."""
  graph = torch.cuda.CUDAGraph(keep_graph=True)
  with torch.cuda.graph(graph):
    keep = call()  # noqa: F841
  n = C.c_size_t()
  hip = C.CDLL("libamdhip64.so")
  assert hip.hipGraphGetNodes(C.c_void_p(graph.raw_cuda_graph()), None, C.byref(n)) == 0
  return n.value


def test_one_kernel_where_every_row_is_one_part():
  """A table with room for one part of a row (128 tokens, 64 in fp32) leaves nothing to join, however many rows there are."""
  for dtype, held, page, width, kernels in ((BF16, BF16, 64, 2, 1), (F32, F32, 16, 4, 1), (BF16, BF16, 64, 3, 2), (F32, F32, 16, 5, 2)):
    cache = make_cache(4, page, 8, 64, held, gen(1))
    table = torch.tensor([[0, 1, 2, 3, 0]], dtype=torch.int32, device=DEV)[:, :width].expand(600, width)
    lens = torch.full((600,), width * page - 5, dtype=torch.int32, device=DEV)
    q = torch.randn(600, 8, 64, generator=gen(2), device=DEV).to(dtype)
    got = cache.attend(q, table, lens, return_lse=True)
    for at in (slice(0, 3), slice(597, 600)):
      check_attend(cache, q[at], table[at], [width * page - 5] * 3, 0.125, 0, (got[0][at], got[1][at]))
    assert captured_nodes(lambda: cache.attend(q, table, lens)) == kernels, (dtype, width)


def test_window_of_a_length_beyond_the_table():
  """The window ends at the length that was given; of what it shows, the table's tokens are seen."""
  cache, q, table, _ = attend_case(BF16, BF16, 2, 4, 64, 16, [48, 48, 48, 48], 0)
  short = table[:, :3]
  ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
  o, lse = cache.attend(q, short, ints(100, 108, 40, 2 ** 31 - 1), window=60, return_lse=True)
  with pytest.raises(IndexError):
    cache.check()
  want, want_lse = cache.attend(q, short, ints(48, 0, 40, 0), window=8, return_lse=True)
  whole, whole_lse = cache.attend(q, short, ints(48, 48, 40, 0), return_lse=True)
  cache.check()
  assert torch.equal(o[:2], want[:2]) and torch.equal(lse[:2], want_lse[:2])       # tokens 40 .. 47, none
  assert torch.equal(o[2:], whole[2:]) and torch.equal(lse[2:], whole_lse[2:])
  assert not o[3].any() and bool((lse[3] == -math.inf).all())


def test_a_report_from_another_stream_is_not_lost():
  """What a call on another stream sets while a check reads and clears is reported by this check or the next."""
  cache = make_cache(4, 16, 2, 64, BF16, gen(1))
  k = torch.zeros(1, 2, 64, dtype=BF16, device=DEV)
  ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
  no_page, some_page, first, far = ints(-1)[None], ints(0)[None], ints(0), ints(1000)
  side = torch.cuda.Stream(device=DEV)
  torch.cuda.synchronize()
  for i in range(400):
    with torch.cuda.stream(side):
      torch.cuda._sleep(1 + 500 * i)
      cache.append(k, k, some_page, far)            # outside the table
    cache.append(k, k, no_page, first)              # no page
    said = ""
    for _ in range(2):
      try:
        cache.check()
      except IndexError as e:
        said += str(e)
      torch.cuda.synchronize()
    assert "page" in said and "outside" in said, (i, said)
    cache.check()
