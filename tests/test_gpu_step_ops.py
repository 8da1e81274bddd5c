"""The self-attention step's operators on the GPU against plain implementations in 64 bits.

Tolerances count roundings.  u(t) = torch.finfo(t).eps / 2 is half a step of type t; U = 2^-24 of fp32.
"""
import math
import random

import pytest
import torch

from tacotron_amd import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def gen(seed):
  return torch.Generator(device=DEV).manual_seed(seed)


def make_cache(n_pages, page, heads, d, dtype, g, order="own", scales=True):
  """A cache filled with random values: the framework's own order of pages, tokens and heads, or another one."""
  from tacotron_amd.paged import PagedCache
  kw = {}
  if dtype == E4M3 and scales:
    kw = {n: torch.rand(heads, generator=g, device=DEV) * 0.5 + 0.25 for n in ("k_scale", "v_scale")}

  def fill():
    if order == "own":
      t = torch.empty(n_pages, heads, page, d, device=DEV).transpose(1, 2)
    elif order == "tokens":
      t = torch.empty(n_pages, page, heads, d, device=DEV)
    elif order == "heads":              # heads outermost
      t = torch.empty(heads, n_pages, page, d, device=DEV).permute(1, 2, 0, 3)
    else:                               # rows with room behind them
      t = torch.empty(n_pages, page, heads, d + 32, device=DEV)
    base = torch.randn(t.shape, generator=g, device=DEV).to(dtype)
    out = torch.empty_strided(t.shape, t.stride(), dtype=dtype, device=DEV)
    out.copy_(base)
    return out[..., :d]
  return PagedCache.from_tensors(fill(), fill(), **kw)


def make_table(needs, n_pages, width, seed):
  """Different pages for every utterance; entries behind its need name no page at all."""
  order = list(range(n_pages))
  random.Random(seed).shuffle(order)
  rows = []
  for n in needs:
    rows.append([order.pop() for _ in range(n)] + [-1 - n if (width - n) % 2 else n_pages + 12345] * (width - n))
  return torch.tensor(rows, dtype=torch.int32, device=DEV).reshape(len(needs), width)


def values(cache):
  """Keys and values as float64, scales applied."""
  k, v = cache.k.double(), cache.v.double()
  if cache.k_scale is not None:
    k, v = k * cache.k_scale.double()[:, None], v * cache.v_scale.double()[:, None]
  return k, v


# ---- append -----------------------------------------------------------------------------------------------------------


def rotate(x, pos, inv_freq, interleaved):
  """x [tokens, heads, d] in 64 bits."""
  half = inv_freq.shape[0]
  out = x.clone()
  angle = pos.double()[:, None, None] * inv_freq
  c, s = angle.cos(), angle.sin()
  first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
  out[..., first] = x[..., first] * c - x[..., second] * s
  out[..., second] = x[..., second] * c + x[..., first] * s
  return out


def pair_size(x, half, interleaved):
  """|x| + |its partner|, what the rounding errors of a rotation go by."""
  out = x.abs().clone()
  if half:
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    both = out[..., first] + out[..., second]
    out[..., first] = both
    out[..., second] = both
  return out


def check_append(cache, k, v, q, table, past, new, inv_freq, interleaved, got_q, before, offset0=0):
  """Everything an append has to have done, and that it did nothing else.  A rotated element is x c - y s: the sine and
  cosine are off by at most 3 U (reduction's rounding to fp32 U/2, polynomial and its last rounding 2 U), the three operations
  by U of (|x| + |y|) each, so 6 U (|x| + |y|) in all, then half a step of the type (and 2 U more for the division by a scale)."""
  page, d = cache.page_size, cache.head_dim
  half = 0 if inv_freq is None else inv_freq.shape[0]
  k_want, v_want = before[0].clone(), before[1].clone()
  row = offset0
  touched = torch.zeros(cache.k.shape[:2], dtype=torch.bool, device=DEV)
  worst = []
  for b, n in enumerate(new):
    if n == 0:
      continue
    rows, pos = slice(row, row + n), torch.arange(past[b], past[b] + n, device=DEV)
    row += n
    pages, slots = table[b].long()[pos // page], pos % page
    touched[pages, slots] = True
    for x, got, stored, scale in ((k, cache.k, True, cache.k_scale), (q, got_q, False, None)):
      if x is None:
        continue
      x64 = x[rows].double()
      want = rotate(x64, pos, inv_freq, interleaved) if half else x64
      slack = (6 * U if half else 0) * pair_size(x64, half, interleaved)
      have = got[pages, slots] if stored else got[rows]
      if scale is not None:
        want, slack = want / scale.double()[:, None], (slack + 2 * U * want.abs()) / scale.double()[:, None]
        want = want.clamp(-448, 448)
      step = half_step(have.dtype) * (want.abs() + slack)
      if have.dtype == E4M3:
        step = torch.maximum(step, torch.full_like(step, 2.0 ** -10))       # half of the type's smallest value
      if have.dtype == F16:
        step = torch.maximum(step, torch.full_like(step, 2.0 ** -25))
      worst.append((((have.double() - want).abs() - slack - step).max().item(), stored))
    exact_v = v[rows].float()
    if cache.v_scale is not None:     # a division, a clamp and one rounding: nothing that may differ
      exact_v = (exact_v.cpu() / cache.v_scale.cpu()[:, None]).clamp(-448, 448).to(E4M3).to(DEV)
    assert torch.equal(cache.v[pages, slots].float(), exact_v.float())
  assert all(w <= 0 for w, _ in worst), worst
  for got, want in ((cache.k, before[0]), (cache.v, before[1])):
    keep = ~touched
    assert torch.equal(got.float()[keep], want.float()[keep])


APPENDS = [
  # dtype, cache, heads, query heads, d, page, new, past, rot, interleaved, order
  (F32, F32, 1, 1, 16, 16, [1], [0], 16, False, "own"),
  (F32, F32, 3, 6, 64, 48, [1, 1, 1], [47, 48, 0], 64, True, "tokens"),
  (F32, F32, 2, 2, 256, 16, [5, 0, 33], [11, 7, 190001], 128, False, "wide"),
  (F16, F16, 4, 4, 80, 32, [1] * 7, [31, 32, 33, 0, 5, 100, 63], 80, False, "heads"),
  (F16, F16, 2, 16, 96, 64, [70, 1], [1, 250000], 48, True, "own"),
  (BF16, BF16, 8, 32, 128, 64, [1] * 65, list(range(0, 130, 2)), 128, False, "own"),
  (BF16, BF16, 5, 35, 32, 16, [17, 16, 15, 1, 0, 100], [0, 1, 16, 15, 3, 77], 32, True, "tokens"),
  (BF16, BF16, 1, 0, 64, 256, [300], [255], 0, False, "own"),
  (BF16, E4M3, 8, 16, 128, 16, [1, 1], [0, 15], 64, False, "own"),
  (F16, E4M3, 2, 2, 48, 80, [81, 3], [79, 160], 48, True, "wide"),
  (BF16, E4M3, 3, 3, 192, 32, [40], [1000000], 192, False, "tokens"),
]


@pytest.mark.parametrize("dtype,held,heads,hq,d,page,new,past,rot,interleaved,order", APPENDS)
def test_append(dtype, held, heads, hq, d, page, new, past, rot, interleaved, order):
  g = gen(len(new) + d)
  first = [p // page for p in past]
  needs = [(p + n + page - 1) // page for p, n in zip(past, new)]
  n_pages = sum(n - f for n, f in zip(needs, first)) + 2
  cache = make_cache(n_pages, page, heads, d, held, g, order)
  table = torch.full((len(new), max(needs) + 1), n_pages, dtype=torch.int32, device=DEV)
  at = 1
  for b in range(len(new)):
    for p in range(first[b], needs[b]):
      table[b, p] = n_pages - at
      at += 1
  tokens = sum(new)
  # rows of one projection's output, as a layer has them: keys, values and queries side by side
  wide = torch.randn(tokens, 2 * heads + max(hq, 1), d, generator=g, device=DEV).to(dtype)
  k, v, q = wide[:, :heads], wide[:, heads:2 * heads], wide[:, 2 * heads:] if hq else None
  if held == E4M3 and tokens:
    k[0, 0, 0], k[0, 0, 1], v[0, 0, 0] = 1e4, -1e4, 1e4          # beyond the type's range
  inv_freq = None if not rot else 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device=DEV) * 2 / rot)
  before = cache.k.clone(), cache.v.clone()
  offsets = None
  if any(n != 1 for n in new):
    offsets = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
  got = cache.append(k, v, table, torch.tensor(past, dtype=torch.int32, device=DEV), q=q, offsets=offsets, inv_freq=inv_freq,
                     interleaved=interleaved)
  cache.check()
  check_append(cache, k, v, q, table, past, new, inv_freq, interleaved, got, before)


def test_append_in_place_and_rows_of_nobody():
  """Queries rotated in place; rows in front of the first utterance and behind the last stay as they were."""
  g = gen(3)
  cache = make_cache(6, 16, 2, 64, BF16, g)
  table = make_table([2, 2], 6, 3, 1)
  k, v, q = (torch.randn(30, 2, 64, generator=g, device=DEV).to(BF16) for _ in range(3))
  inv_freq = torch.rand(32, generator=g, device=DEV, dtype=torch.float64)
  before, q0 = (cache.k.clone(), cache.v.clone()), q.clone()
  offsets = torch.tensor([4, 9, 24], dtype=torch.int32, device=DEV)
  out = cache.append(k, v, table, torch.tensor([3, 12], dtype=torch.int32, device=DEV), q=q, offsets=offsets,
                     inv_freq=inv_freq, out=q)
  cache.check()
  assert out is q
  assert torch.equal(q[:4], q0[:4]) and torch.equal(q[24:], q0[24:])
  check_append(cache, k, v, q0, table, [3, 12], [5, 15], inv_freq, False, q, before, offset0=4)


def test_append_without_pages_sets_a_flag_and_writes_nothing():
  g = gen(4)
  cache = make_cache(4, 16, 2, 64, F32, g)
  table = torch.tensor([[0, -1], [4, 1], [2, 3]], dtype=torch.int32, device=DEV)
  k, v, q = (torch.randn(3, 2, 64, generator=g, device=DEV) for _ in range(3))
  before = cache.k.clone(), cache.v.clone()
  for past in ([16, 0, 32], [17, 15, -1], [31, 3, 2 ** 31 - 1]):      # bad entries, bad entry, place outside the table
    got = cache.append(k, v, table, torch.tensor(past, dtype=torch.int32, device=DEV), q=q)
    assert torch.equal(got, q)                                      # nothing to rotate: the queries come back whatever the places
    with pytest.raises(IndexError) as e:
      cache.check()
    assert "page" in str(e.value) and "outside" in str(e.value)
    cache.check()                                                   # cleared by the first
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])


# ---- attend -----------------------------------------------------------------------------------------------------------


def attend_64(cache, q, table, lens, scale, window):
  """(out, lse, sum of w |v|, largest |q||k| score bound) in 64 bits, utterance by utterance."""
  k, v = values(cache)
  n, hq, d = q.shape
  group = hq // cache.n_heads
  out, size = (torch.zeros(n, hq, d, dtype=torch.float64, device=DEV) for _ in range(2))
  lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=DEV)
  reach = torch.zeros(n, hq, dtype=torch.float64, device=DEV)
  for b, length in enumerate(lens):
    low = max(0, length - window) if window else 0
    if length == low:
      continue
    pos = torch.arange(low, length, device=DEV)
    pages, slots = table[b].long()[pos // cache.page_size], pos % cache.page_size
    kb, vb = (t[pages, slots].transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))     # [hq, tokens, d]
    qb = q[b].double()
    score = (kb @ qb[:, :, None])[..., 0] * scale
    reach[b] = ((kb.abs() @ qb.abs()[:, :, None])[..., 0] * abs(scale)).amax(1)
    lse[b] = torch.logsumexp(score, 1)
    w = torch.softmax(score, 1)
    out[b], size[b] = (w[:, None] @ vb)[:, 0], (w[:, None] @ vb.abs())[:, 0]
  return out, lse, size, reach


def check_attend(cache, q, table, lens, scale, window, got):
  """A score is off by at most (d + 6) U of scale * sum |q||k| (d products summed in fp32, the factors' roundings), a
  softmax weight by twice that (its own and its normaliser's) and 8 U of exp2's and its argument's; a weight is held as two values of the
  operand's type (2^-16 for two bfloat16, 2^-21 for two float16); sums of n terms in fp32 lose n U; then one rounding."""
  out, lse, size, reach = attend_64(cache, q, table, lens, scale, window)
  n = max([min(x, window) if window else x for x in lens] + [1])
  e_score = (cache.head_dim + 6) * U * reach
  split = {F32: 0.0, F16: 2.0 ** -21, BF16: 2.0 ** -16}[q.dtype]
  e_w = 2 * e_score + 16 * U + n * U + split
  tol = e_w[..., None] * size * 1.01 + 4 * U * out.abs()
  tol = tol + half_step(q.dtype) * (out.abs() + tol) + (2.0 ** -25 if q.dtype == F16 else 0)
  o, l = got
  assert torch.isfinite(o).all()
  excess = (o.double() - out).abs() - tol
  assert excess.max().item() <= 0, ("out", excess.max().item(), tol.flatten()[excess.argmax()].item())
  empty = lse == -math.inf
  assert torch.equal(l == -math.inf, empty)
  l_tol = e_score + n * U + 16 * U + 4 * U * lse.abs()
  bad = ((l.double() - lse).abs() - l_tol)[~empty]
  assert bad.numel() == 0 or bad.max().item() <= 0, ("lse", bad.max().item())


def attend_case(dtype, held, heads, hq, d, page, lens, window, order="own", seed=0, spread=1.0):
  g = gen(seed + d + len(lens))
  needs = [(n + page - 1) // page for n in lens]
  width = max(needs + [1]) + 1
  n_pages = sum(needs) + 2
  cache = make_cache(n_pages, page, heads, d, held, g, order)
  table = make_table(needs, n_pages, width, seed)
  used = torch.zeros(n_pages, page, dtype=torch.bool, device=DEV)
  for b, n in enumerate(lens):
    pos = torch.arange(n, device=DEV)
    used[table[b].long()[pos // page], pos % page] = True
    if window:                                       # what the window hides may be anything too
      pos = pos[:max(0, n - window)]
      used[table[b].long()[pos // page], pos % page] = False
  for t in (cache.k, cache.v):
    if held == E4M3:
      t.view(torch.uint8)[~used] = 0x7f             # a NaN
    else:
      t[~used] = float("nan")
  q = (torch.randn(len(lens), hq + 1, d, generator=g, device=DEV) * spread).to(dtype)[:, 1:]
  return cache, q, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 1, 0]
ATTENDS = [
  # dtype, cache, heads, query heads, d, page, lens, window, order
  (F32, F32, 1, 1, 16, 16, [1], 0, "own"),
  (F32, F32, 4, 4, 64, 16, EDGES, 0, "own"),
  (F32, F32, 2, 6, 128, 48, [777, 0, 100, 5], 0, "tokens"),
  (F32, F32, 2, 40, 256, 32, [70, 513], 33, "wide"),
  (F16, F16, 4, 4, 64, 16, EDGES, 17, "heads"),
  (F16, F16, 3, 15, 80, 80, [1000, 81, 80, 79], 0, "own"),
  (F16, F16, 1, 71, 96, 64, [300, 1], 0, "tokens"),
  (BF16, BF16, 8, 32, 128, 64, EDGES, 0, "own"),
  (BF16, BF16, 2, 2, 128, 16, [3000, 1, 2999], 1, "own"),
  (BF16, BF16, 1, 16, 256, 256, [511, 1025, 255], 300, "own"),
  (BF16, BF16, 3, 51, 32, 16, [100, 3, 33], 0, "wide"),
  (BF16, BF16, 2, 4, 192, 32, [400], 0, "heads"),
  (BF16, E4M3, 8, 64, 128, 32, EDGES, 0, "own"),
  (F16, E4M3, 2, 2, 64, 16, [1000, 17], 100, "tokens"),
  (BF16, E4M3, 1, 5, 208, 16, [333, 16], 0, "own"),
  (F16, E4M3, 2, 34, 256, 48, [49, 700], 0, "wide"),
  (BF16, BF16, 8, 32, 128, 64, [20000], 0, "own"),
  (BF16, BF16, 1, 8, 128, 64, [9000, 100, 0, 5000] + [40] * 300, 0, "own"),
  # tables with room for a part of a row only (128 tokens, 64 in fp32): nothing to join, unless there are more rows than workgroups
  (BF16, BF16, 4, 8, 64, 16, [112, 1, 0, 97, 64, 33], 0, "own"),
  (F32, F32, 3, 3, 128, 16, [48, 0, 17, 1], 0, "tokens"),
  (F16, E4M3, 1, 40, 128, 32, [96, 5], 20, "own"),
  (BF16, BF16, 8, 16, 128, 64, [64, 3, 50, 0, 33] * 60, 0, "own"),
]


@pytest.mark.parametrize("dtype,held,heads,hq,d,page,lens,window,order", ATTENDS)
def test_attend(dtype, held, heads, hq, d, page, lens, window, order):
  cache, q, table, lens_dev = attend_case(dtype, held, heads, hq, d, page, lens, window, order)
  scale = d ** -0.5
  got = cache.attend(q, table, lens_dev, window=window, return_lse=True)
  cache.check()
  check_attend(cache, q, table, lens, scale, window, got)
  again = cache.attend(q, table, lens_dev, scale=scale, window=window, return_lse=True)
  assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])       # no result depends on timing
  into = torch.full((len(lens), hq, d + 16), 7.0, dtype=dtype, device=DEV)
  assert cache.attend(q, table, lens_dev, window=window, out=into[..., :d]) is not None
  assert torch.equal(into[..., :d], got[0]) and bool((into[..., d:] == 7).all())
  assert cache.attend(q, table, lens_dev, window=window, out=q) is q and torch.equal(q, got[0])      # in place


def test_attend_peaked_scores():
  """Scores far apart, rising and falling along the cache: the running maximum is replaced many times."""
  for dtype, held in ((F32, F32), (BF16, BF16), (F16, E4M3)):
    cache, q, table, lens = attend_case(dtype, held, 2, 4, 64, 16, [500, 33, 1], 0, spread=1.0)
    for t in range(500):
      cache.k[table[0, t // 16].long(), t % 16] = (cache.k[table[0, t // 16].long(), t % 16].float() * (1 + t % 97) / 40).to(held)
    got = cache.attend(q, table, lens, scale=0.7, return_lse=True)
    check_attend(cache, q, table, [500, 33, 1], 0.7, 0, got)


@pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (F16, F16), (F16, E4M3)])
def test_attend_many_small_weights_beside_a_large_one(dtype, held):
  """One token's score is 15.72 above all others', whose weights are about 2^-22.7 each: what they sum to is seen where the
  first token's values are zero, and bounded there by its own size."""
  n, scale = 4000, 1.0
  cache, q, table, lens = attend_case(dtype, held, 2, 4, 64, 16, [n, 0, 77], 0)
  k, v = torch.zeros(2, 1, 64, device=DEV), torch.rand(2, 2, 64, generator=gen(5), device=DEV) + 0.5
  first = v[1].clone()
  first[:, ::2] = 0
  pages = table[0, :n // 16].long()
  cache.k[pages] = k[0].to(held)
  cache.v[pages] = v[0].to(held)
  cache.k[table[0, 33].long(), 5] = torch.nn.functional.pad(torch.tensor([7.5], device=DEV), (0, 63)).to(held)       # token 533
  cache.v[table[0, 33].long(), 5] = first.to(held)
  k_scale, v_scale = (torch.ones(2, device=DEV) if t is None else t for t in (cache.k_scale, cache.v_scale))
  q[0] = 0.0
  q[0, :, 0] = (2.096 / k_scale).repeat_interleave(2).to(dtype)
  got = cache.attend(q, table, lens, scale=scale, return_lse=True)
  check_attend(cache, q, table, [n, 0, 77], scale, 0, got)
  out = got[0][0].float() / v_scale.repeat_interleave(2)[:, None]
  assert bool((out[:, ::2] > 2.5e-4).all()) and bool((out[:, 1::2] > 0.4).all())


def test_attend_scale_and_window_are_taken_by_value():
  cache, q, table, lens = attend_case(F32, F32, 2, 4, 64, 16, [50, 20], 0)
  scale = torch.tensor(0.25)
  a = cache.attend(q, table, lens, scale=scale)
  assert torch.equal(a, cache.attend(q, table, lens, scale=0.25))
  scale.fill_(0.5)
  b = cache.attend(q, table, lens, scale=scale)
  assert torch.equal(b, cache.attend(q, table, lens, scale=0.5)) and not torch.equal(a, b)
  window = torch.tensor(7)
  c = cache.attend(q, table, lens, window=window)
  assert torch.equal(c, cache.attend(q, table, lens, window=7))
  for wide in (50, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40 + 3):      # wider than any length
    assert torch.equal(cache.attend(q, table, lens, window=wide), cache.attend(q, table, lens)), wide


def test_attend_bad_entries_and_lengths():
  """A block on a page that is none is not seen; a length beyond the table ends at it, a negative one is 0: all flagged."""
  cache, q, table, lens = attend_case(BF16, BF16, 2, 4, 64, 16, [100, 64, 20], 0)
  want = cache.attend(q, table, lens, return_lse=True)
  cache.check()
  bad = table.clone()
  bad[0, 2], bad[1, 3] = -5, cache.n_pages
  got = cache.attend(q, bad, lens, return_lse=True)
  with pytest.raises(IndexError):
    cache.check()
  assert torch.equal(got[0][2], want[0][2])
  k, v = values(cache)
  for b, keep in ((0, [t for t in range(100) if t // 16 != 2]), (1, list(range(48)))):
    pos = torch.tensor(keep, device=DEV)
    kb, vb = (t[table[b].long()[pos // 16], pos % 16].transpose(0, 1).repeat_interleave(2, 0) for t in (k, v))
    w = torch.softmax((kb @ q[b].double()[:, :, None])[..., 0] / 8, 1)
    out = (w[:, None] @ vb)[:, 0]
    # as in check_attend, with |score| sums below 64 * 4.5^2 / 8 = 162
    tol = (2 * 70 * U * 162 + 2.0 ** -16 + 120 * U) * (w[:, None] @ vb.abs())[:, 0]
    assert ((got[0][b].double() - out).abs() <= tol + half_step(BF16) * (out.abs() + tol)).all()
  all_bad = torch.full_like(table, -1)
  o, lse = cache.attend(q, all_bad, lens, return_lse=True)
  assert not o.any() and bool((lse == -math.inf).all())
  with pytest.raises(IndexError):
    cache.check()
  short = table[:, :3]
  o, lse = cache.attend(q, short, torch.tensor([100, -3, 20], dtype=torch.int32, device=DEV), return_lse=True)
  ref = cache.attend(q, short, torch.tensor([48, 0, 20], dtype=torch.int32, device=DEV), return_lse=True)
  assert torch.equal(o, ref[0]) and torch.equal(lse, ref[1])
  with pytest.raises(IndexError):
    cache.check()


def test_attend_non_finite_scores():
  """Scores of -inf count for nothing, a NaN that is seen shows, as in the formula."""
  cache, q, table, lens = attend_case(F32, F32, 1, 1, 16, 16, [20, 20, 20], 0)
  q[:] = 0.5
  row = lambda b, t: cache.k[table[b, t // 16].long(), t % 16, 0]  # noqa: E731
  want = cache.attend(q, table, lens, return_lse=True)
  for t in range(20):
    row(1, t)[:] = -math.inf
  row(2, 7)[3] = float("nan")
  o, lse = cache.attend(q, table, lens, return_lse=True)
  assert torch.equal(o[0], want[0][0])
  assert not o[1].any() and bool((lse[1] == -math.inf).all())
  assert bool(o[2].isnan().all())


def test_a_cache_beyond_32_bit_offsets():
  """Pages whose byte and element offsets pass 2^32: 70 000 pages of 16 tokens x 16 heads x 128 (4.6e9 bytes each)."""
  n_pages, page, heads, d = 70_000, 16, 16, 128
  from tacotron_amd.paged import PagedCache
  big = [torch.empty(n_pages, heads, page, d, dtype=BF16, device=DEV).transpose(1, 2) for _ in range(2)]
  cache = PagedCache.from_tensors(*big)
  g = gen(9)
  table = torch.tensor([[69_999, 3, 40_000], [69_998, 33_000, 65_536]], dtype=torch.int32, device=DEV)
  k, v = (torch.randn(80, heads, d, generator=g, device=DEV).to(BF16) for _ in range(2))
  offsets = torch.tensor([0, 40, 80], dtype=torch.int32, device=DEV)
  cache.append(k, v, table, torch.zeros(2, dtype=torch.int32, device=DEV), offsets=offsets)
  q = torch.randn(2, heads, d, generator=g, device=DEV).to(BF16)
  got = cache.attend(q, table, torch.tensor([40, 40], dtype=torch.int32, device=DEV), return_lse=True)
  cache.check()
  small = make_cache(6, page, heads, d, BF16, g)
  near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
  small.append(k, v, near, torch.zeros(2, dtype=torch.int32, device=DEV), offsets=offsets)
  for x, y in ((small.k, cache.k), (small.v, cache.v)):
    assert torch.equal(x[near.long()].flatten(1, 2)[:, :40], y[table.long()].flatten(1, 2)[:, :40])
  want = small.attend(q, near, torch.tensor([40, 40], dtype=torch.int32, device=DEV), return_lse=True)
  assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
  check_attend(small, q, near, [40, 40], d ** -0.5, 0, want)


def test_refused_tensors():
  from tacotron_amd.paged import PagedCache
  cache = PagedCache(4, 16, 2, 64, dtype=BF16, device=DEV)
  with pytest.raises(AttributeError):
    cache.k = cache.v
  assert (cache.n_pages, cache.page_size, cache.n_heads, cache.head_dim) == (4, 16, 2, 64)
  t = lambda *s, dtype=BF16, device=DEV: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
  i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
  k = t(3, 2, 64)
  for call in (
    lambda: PagedCache(4, 24, 2, 64, device=DEV), lambda: PagedCache(4, 16, 2, 60, device=DEV), lambda: PagedCache(0, 16, 2, 64, device=DEV),
    lambda: PagedCache(4, 16, 2, 64, dtype=torch.float64, device=DEV), lambda: PagedCache(4, 16, 2, 272, device=DEV),
    lambda: PagedCache(4, 16, 2, 64, device=DEV, k_scale=torch.ones(2, device=DEV)),
    lambda: PagedCache(4, 16, 2, 64, dtype=E4M3, device=DEV, k_scale=torch.ones(3, device=DEV)),
    lambda: PagedCache.from_tensors(t(4, 16, 2, 64), t(4, 16, 2, 64, dtype=F16)),
    lambda: PagedCache.from_tensors(t(4, 16, 2, 68)[..., 4:], t(4, 16, 2, 68)[..., 4:]),
    lambda: cache.append(k, t(2, 2, 64), i(3, 2), i(3)), lambda: cache.append(k, k, i(2, 2), i(2)),
    lambda: cache.append(k, k, i(3, 2), i(2)), lambda: cache.append(k, k, i(3, 2), i(3).long()),
    lambda: cache.append(k.float(), k.float(), i(3, 2), i(3)), lambda: cache.append(k, k, i(3, 2).long(), i(3)),
    lambda: cache.append(k, k, i(3, 2), i(3), inv_freq=t(32, dtype=F32)), lambda: cache.append(k, k, i(3, 2), i(3), inv_freq=t(40, dtype=torch.float64)),
    lambda: cache.append(k, k, i(3, 2), i(3), inv_freq=t(12, dtype=torch.float64)), lambda: cache.append(k, k, i(3, 2), i(3), out=k),
    lambda: cache.append(k, k, i(3, 2), i(3), q=k, out=t(3, 2, 32)), lambda: cache.append(k, k, i(3, 2), i(3), offsets=i(3)),
    lambda: cache.append(k, k, i(2, 3).t(), i(3)), lambda: cache.append(k.cpu(), k.cpu(), i(3, 2), i(3)),
    lambda: cache.attend(t(3, 3, 64), i(3, 2), i(3)), lambda: cache.attend(t(3, 4, 32), i(3, 2), i(3)), lambda: cache.attend(t(3, 4, 64), i(2, 2), i(2)),
    lambda: cache.attend(t(3, 4, 64), i(3, 2), i(3), window=-1), lambda: cache.attend(t(3, 4, 64, dtype=F16), i(3, 2), i(3)),
    lambda: cache.attend(t(3, 4, 64), i(3, 2), i(3), out=t(3, 4, 66)[..., 2:]),
    lambda: cache.attend(t(3, 4, 64), i(3, 2), i(3), out=t(3, 1, 64).expand(3, 4, 64)),
    lambda: cache.append(k, k, i(3, 2), i(3), q=k, out=t(1, 2, 64).expand(3, 2, 64)),
    lambda: PagedCache.from_tensors(t(1, 16, 2, 64).expand(4, 16, 2, 64), t(4, 16, 2, 64)), lambda: cache.attend(t(3, 4, 64), i(3, 2).cpu(), i(3)),
  ):
    with pytest.raises((ValueError, RuntimeError)):
      call()
  with pytest.raises(_lib.TacoError):
    cache.attend(t(3, 4, 64), i(3, 2), i(3), scale=float("nan"))


def test_rows_that_need_a_copy():
  """Keys, values and queries whose rows are not aligned, or whose heads lie outside the tokens."""
  g = gen(12)
  cache, other = (make_cache(4, 16, 2, 64, BF16, gen(1)) for _ in range(2))
  table = torch.tensor([[0], [1], [2]], dtype=torch.int32, device=DEV)
  past = torch.tensor([3, 0, 15], dtype=torch.int32, device=DEV)
  k, v, q = (torch.randn(2, 3, 65, generator=g, device=DEV).to(BF16).transpose(0, 1)[..., 1:] for _ in range(3))
  inv_freq = torch.rand(32, generator=g, device=DEV, dtype=torch.float64)
  a = cache.append(k, v, table, past, q=q, inv_freq=inv_freq)
  b = other.append(k.contiguous(), v.contiguous(), table, past, q=q.contiguous(), inv_freq=inv_freq)
  assert torch.equal(a, b) and torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)
  lens = past + 1
  assert torch.equal(cache.attend(q, table, lens), other.attend(q.contiguous(), table, lens))


def test_empty_calls():
  from tacotron_amd.paged import PagedCache
  cache = PagedCache(2, 16, 2, 64, device=DEV)
  none = torch.zeros(0, 2, 64, device=DEV)
  table = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
  zero = torch.zeros(0, dtype=torch.int32, device=DEV)
  assert cache.append(none, none, table, zero, q=none).shape == (0, 2, 64)
  out, lse = cache.attend(none, table, zero, return_lse=True)
  assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
  q = torch.randn(2, 2, 64, device=DEV)      # utterances without any table
  out = cache.attend(q, torch.zeros(2, 0, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV))
  cache.check()
  assert not out.any()
  # utterances without new tokens
  rows = torch.randn(0, 2, 64, device=DEV)
  cache.append(rows, rows, torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV),
               offsets=torch.zeros(3, dtype=torch.int32, device=DEV))


def test_graph_replays_with_new_lengths():
  """One captured step replayed as an utterance grows, eager work in between; two graphs over the same cache on two streams."""
  d, heads = 64, 4
  cache = make_cache(40, 16, heads, d, BF16, gen(5))
  plain = make_cache(40, 16, heads, d, BF16, gen(5))
  table = make_table([18, 18], 40, 18, 2)
  inv_freq = 1000.0 ** (-torch.arange(d // 2, dtype=torch.float64, device=DEV) / 32)
  past = torch.tensor([0, 100], dtype=torch.int32, device=DEV)
  lens = past + 1
  k, v, q = (torch.zeros(2, heads, d, dtype=BF16, device=DEV) for _ in range(3))
  outs = []
  graphs = []
  for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      turned = cache.append(k, v, table, past, q=q, inv_freq=inv_freq)
      out = cache.attend(turned, table, lens)
      torch.add(past, 0)                # work of the caller's own
    graphs.append(graph)
    outs.append(out)
  g = gen(6)
  side = [torch.cuda.Stream(device=DEV) for _ in range(2)]
  past_plain = past.clone()
  for step in range(12):
    for t in (k, v, q):
      t.copy_(torch.randn(2, heads, d, generator=g, device=DEV))
    torch.cuda.synchronize()
    if step % 3 == 2:                   # both graphs at once: the same tokens to the same places, outputs of their own
      for s, graph in zip(side, graphs):
        with torch.cuda.stream(s):
          graph.replay()
    else:
      graphs[step % 3].replay()
    torch.cuda.synchronize()
    want = plain.attend(plain.append(k, v, table, past_plain, q=q, inv_freq=inv_freq), table, past_plain + 1)
    for i, out in enumerate(outs):
      if step % 3 in (i, 2):
        assert torch.equal(out, want), (step, i)
    past += 1
    lens += 1
    past_plain += 1
  assert torch.equal(cache.k, plain.k) and torch.equal(cache.v, plain.v)
  cache.check()


def test_two_streams_at_once():
  """Calls of different utterances on two streams over one cache, each as on its own."""
  cache, q, table, lens = attend_case(BF16, BF16, 4, 16, 128, 64, [3000, 2999, 40, 1], 0)
  half = [(q[i:i + 2], table[i:i + 2], lens[i:i + 2]) for i in (0, 2)]
  want = [cache.attend(*h, return_lse=True) for h in half]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream(device=DEV) for _ in range(2)]
  got = []
  for _ in range(10):
    for s, h in zip(streams, half):
      with torch.cuda.stream(s):
        got.append(cache.attend(*h, return_lse=True))
  torch.cuda.synchronize()
  for i, (o, l) in enumerate(got):
    assert torch.equal(o, want[i % 2][0]) and torch.equal(l, want[i % 2][1])


# ---- 4-bit matrices ---------------------------------------------------------------------------------------------------


def make_codes(n, k, group, scale_dtype, zeros, g):
  groups = -(-k // group)
  codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
  flat = torch.nn.functional.pad(codes, (0, k % 2))
  packed = flat[:, 0::2] | (flat[:, 1::2] << 4)
  scales = (torch.rand(n, groups, generator=g, device=DEV) * 0.1 + 0.01).to(scale_dtype)
  z = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8) if zeros else None
  return codes, packed, scales, z


def check_matvec(codes, scales, zeros, group, bias, x, got):
  """A group's sum in fp32 is off by at most 3 (group + 8) U of the sum of |terms|; taking the offset off and
  scaling adds a few U more, the groups' and the waves' sums (groups + 16) U.  The terms are (16 + c) x and (16 + z) sum x, x in three parts for fp32 (whose sums of |terms| are together at most 1.01 times
  as large); then the bias and one rounding."""
  n, k = codes.shape
  s = scales.double().repeat_interleave(group, 1)[:, :k]
  z = torch.full_like(s, 8.0) if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :k]
  c, x64 = codes.double(), x.double()
  want = x64 @ ((c - z) * s).t()
  size = 1.01 * (32 + c + z) * s
  if bias is not None:
    want = want + bias.double()
  slack = (3 * (group + 8) + scales.shape[1] + 16 + 8) * U * (x64.abs() @ size.t()) + 2 * U * want.abs()
  tol = slack + half_step(x.dtype) * (want.abs() + slack) + (2.0 ** -25 if x.dtype == F16 else 0)
  excess = (got.double() - want).abs() - tol
  assert excess.max().item() <= 0, (excess.max().item(), want.flatten()[excess.argmax()].item())


MATVECS = [
  # x, scales, vectors, out, in, group, zeros, bias
  (F32, F32, 1, 1, 1, 32, False, False),
  (F32, F32, 1, 80, 1558, 32, False, True),
  (F32, F16, 16, 17, 129, 128, True, False),
  (F32, BF16, 17, 100, 333, 64, True, True),
  (F32, F32, 65, 33, 127, 32, True, False),
  (F16, F16, 1, 4096, 1024, 128, False, False),
  (F16, F32, 3, 15, 31, 32, True, True),
  (F16, F16, 33, 16, 128, 64, True, False),
  (F16, BF16, 5, 1000, 97, 128, False, True),
  (BF16, BF16, 1, 31, 4099, 128, True, False),
  (BF16, F32, 2, 48, 2048, 32, True, True),
  (BF16, F16, 16, 130, 1000, 64, False, False),
  (BF16, BF16, 130, 50, 65, 32, False, True),
  (BF16, BF16, 1, 3, 20000, 128, True, False),
  # every way of dividing the rows: up to a row block per CU, two, four
  (F32, F16, 2, 4100, 200, 32, True, True),
  (F16, F16, 16, 6000, 257, 64, False, False),
  (BF16, F32, 1, 9000, 300, 32, True, False),
  (BF16, BF16, 7, 8200, 2500, 128, True, True),
  (F32, F32, 16, 8209, 160, 64, False, True),
  (F16, F16, 20, 9001, 130, 32, False, False),
  # more than a tile of vectors, in each of them
  (F16, F16, 33, 2000, 129, 128, True, False),
  (BF16, F32, 30, 4000, 511, 32, True, True),
  (F16, F32, 64, 4100, 640, 64, False, True),
  (BF16, BF16, 45, 8200, 301, 64, True, False),
  (F16, F32, 17, 9001, 200, 32, True, False),
  (F32, F32, 33, 3000, 300, 64, True, True),
  (F32, F16, 40, 4100, 257, 128, False, False),
]


@pytest.mark.parametrize("dtype,scale_dtype,vectors,n,k,group,zeros,with_bias", MATVECS)
def test_matvec(dtype, scale_dtype, vectors, n, k, group, zeros, with_bias):
  from tacotron_amd.w4 import W4Matrix
  g = gen(n + k)
  codes, packed, scales, z = make_codes(n, k, group, scale_dtype, zeros, g)
  bias = torch.randn(n, generator=g, device=DEV).to(dtype) if with_bias else None
  W = W4Matrix.from_codes(packed, scales, zeros=z, bias=bias, in_features=k, group=group)
  assert (W.out_features, W.in_features, W.group) == (n, k, group)
  x = torch.randn(vectors, k, generator=g, device=DEV).to(dtype)
  got = W.matvec(x)
  check_matvec(codes, scales, z, group, bias, x, got)
  assert torch.equal(W.matvec(x), got)
  # every vector alone, rows of a wider tensor at odd addresses, and into a given output
  wide = torch.full((vectors, k + 3), float("nan"), dtype=dtype, device=DEV)
  wide[:, 1:k + 1] = x
  into = torch.full((vectors, n + 5), 7.0, dtype=dtype, device=DEV)
  W.matvec(wide[:, 1:k + 1], out=into[:, 2:n + 2])
  assert torch.equal(into[:, 2:n + 2], got) and bool((into[:, :2] == 7).all()) and bool((into[:, n + 2:] == 7).all())
  check_matvec(codes, scales, z, group, bias, x[-1:], W.matvec(x[-1])[None])
  assert W.matvec(x.reshape(1, vectors, k)).shape == (1, vectors, n)
  assert W.matvec(x[:0]).shape == (0, n)


def test_matvec_extreme_codes_and_values():
  """All codes at either end, inputs from the smallest subnormals to the largest finite ones."""
  from tacotron_amd.w4 import W4Matrix
  for dtype, values_ in ((F16, [6e-8, 6e-5, 1.0, 60000.0]), (BF16, [1e-38, 1e-30, 1.0, 1e30]), (F32, [1e-38, 1e-30, 1.0, 1e30])):
    for code, zero in ((0, 0), (0, 15), (15, 0), (15, 15), (7, 8)):
      z = torch.full((16, 1), zero, dtype=torch.uint8, device=DEV)
      scales = torch.full((16, 1), 1e-3, device=DEV)
      W = W4Matrix.from_codes(torch.full((16, 32), code * 17, dtype=torch.uint8, device=DEV), scales, zeros=z, group=64)
      for v in values_:
        x = torch.full((1, 64), v, dtype=dtype, device=DEV)
        x[0, ::3] *= -1
        got = W.matvec(x)
        size = 1.01 * (32 + code + zero) * 1e-3 * x.double().abs().sum().item()
        want = (code - zero) * scales[0].double() * x.double().sum()
        tol = 250 * U * size + half_step(dtype) * want.abs() + {F16: 2.0 ** -25, BF16: 2.0 ** -126, F32: 2.0 ** -126}[dtype]
        assert ((got.double() - want).abs() <= tol).all(), (dtype, code, zero, v)


@pytest.mark.parametrize("dtype,scale_dtype,n,k,group,symmetric", [
  (F32, None, 5, 97, 32, True), (F32, F16, 3, 128, 64, False), (BF16, None, 17, 1000, 128, True), (F16, F32, 1, 1, 32, False),
  (BF16, F32, 33, 65, 64, False)])
def test_quantize(dtype, scale_dtype, n, k, group, symmetric):
  from tacotron_amd import w4
  g = gen(k)
  w = torch.randn(n, k + 2, generator=g, device=DEV).to(dtype)[:, :k]
  w[0, :min(k, group)] = 0                              # a group of zeros
  codes, scales, zeros = w4.quantize(w, group, symmetric, scale_dtype)
  assert scales.dtype == (scale_dtype or dtype) and (zeros is None) == symmetric
  groups = -(-k // group)
  full = torch.nn.functional.pad(w.float().cpu(), (0, groups * group - k)).view(n, groups, group)
  lo, hi = full.amin(-1).clamp(max=0), full.amax(-1).clamp(min=0)
  s = ((torch.maximum(hi, -lo) / 7) if symmetric else (hi - lo) / 15).to(scales.dtype)
  assert torch.equal(scales.cpu(), s)
  s = s.float()[..., None]
  z = torch.full_like(s, 8.0) if symmetric else torch.where(s > 0, (-lo[..., None] / s).round().clamp(0, 15), 0.0)
  q = torch.where(s > 0, ((full / s).round() + z).clamp(0, 15), z).to(torch.uint8).flatten(1)[:, :k]
  unpacked = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, :k].cpu()
  assert torch.equal(unpacked, q)
  if zeros is not None:
    assert torch.equal(zeros.cpu().float(), z[..., 0])
  W = w4.W4Matrix.from_weights(w, group, symmetric, scale_dtype)
  x = torch.randn(2, k, generator=g, device=DEV)
  check_matvec(unpacked.to(DEV), scales, zeros, group, None, x, W.matvec(x))


def test_matrices_with_one_row_for_all():
  """Scales, zero points, codes and weights that are expanded over the rows."""
  from tacotron_amd.w4 import W4Matrix, quantize
  codes, packed, scales, z = make_codes(100, 300, 64, F16, True, gen(31))
  x = torch.randn(3, 300, generator=gen(32), device=DEV).to(F16)
  make = lambda c, s, zp: W4Matrix.from_codes(c, s, zeros=zp, in_features=300, group=64).matvec(x)  # noqa: E731
  one = lambda t: t[5:6].expand(t.shape)  # noqa: E731
  assert torch.equal(make(packed, one(scales), one(z)), make(packed, one(scales).contiguous(), one(z).contiguous()))
  assert torch.equal(make(one(packed), scales, z), make(one(packed).contiguous(), scales, z))
  assert torch.equal(make(packed, scales[:, :1].expand(100, 5), z), make(packed, scales[:, :1].repeat(1, 5), z))
  w = torch.randn(1, 300, generator=gen(33), device=DEV).expand(40, 300)
  for a, b in zip(quantize(w, 32, False), quantize(w.contiguous(), 32, False)):
    assert torch.equal(a, b)


def test_matvec_refusals():
  from tacotron_amd.w4 import W4Matrix, quantize
  codes, packed, scales, z = make_codes(8, 64, 32, F32, True, gen(1))
  W = W4Matrix.from_codes(packed, scales, zeros=z)
  x = torch.zeros(2, 64, device=DEV)
  for call in (
    lambda: W4Matrix.from_codes(packed, scales, in_features=65), lambda: W4Matrix.from_codes(packed, scales, in_features=0),
    lambda: W4Matrix.from_codes(packed, scales[:, :1], in_features=30), lambda: W4Matrix.from_codes(packed, scales, group=16),
    lambda: W4Matrix.from_codes(packed, scales[:4]), lambda: W4Matrix.from_codes(packed.int(), scales), lambda: W4Matrix.from_codes(packed, scales.double()),
    lambda: W4Matrix.from_codes(packed, scales, zeros=z[:, :1]), lambda: W4Matrix.from_codes(packed, scales, zeros=z.int()),
    lambda: W4Matrix.from_codes(packed, scales, bias=torch.zeros(7, device=DEV)), lambda: W4Matrix.from_codes(packed.cpu(), scales.cpu()),
    lambda: W4Matrix.from_weights(torch.ones(64, 64, device=DEV)).matvec(x, out=x), lambda: W.matvec(x[:, :63]), lambda: W.matvec(x.double()), lambda: W.matvec(x.cpu()), lambda: W.matvec(x, out=torch.zeros(2, 9, device=DEV)),
    lambda: W.matvec(x, out=torch.zeros(8, 2, device=DEV).t()), lambda: W.matvec(x, out=torch.zeros(1, 8, device=DEV).expand(2, 8)),
    lambda: quantize(torch.zeros(3, 0, device=DEV)), lambda: quantize(torch.zeros(3, 8, device=DEV), group=48), lambda: quantize(torch.zeros(3, 8)),
  ):
    with pytest.raises((ValueError, RuntimeError)):
      call()


# ---- a run of them together ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (F16, E4M3)])
def test_layers_of_a_decoder_step(dtype, held):
  """Prompts of several utterances, then single frames, through two layers: projection, append, attend, projection.  Every
  operator is checked against 64 bits on what the one before it gave."""
  from tacotron_amd.w4 import W4Matrix
  g = gen(21)
  width, hq, hkv, d, page, layers = 256, 4, 2, 64, 16, 2
  qkv = hq + 2 * hkv
  weights = []
  for _ in range(layers):
    for n, k in ((qkv * d, width), (width, hq * d)):
      codes, packed, scales, z = make_codes(n, k, 64, F32 if dtype == F32 else dtype, True, g)
      weights.append((codes, scales, z, W4Matrix.from_codes(packed, scales, zeros=z, group=64)))
  caches = [make_cache(24, page, hkv, d, held, g) for _ in range(layers)]
  table = make_table([5, 4, 6], 24, 6, 3)
  inv_freq = 10000.0 ** (-torch.arange(d // 2, dtype=torch.float64, device=DEV) / (d // 2))
  past = [0, 0, 0]
  for new in ([15, 33, 60], [1, 1, 1], [1, 1, 1], [2, 0, 1], [1, 1, 1]):
    x = (torch.randn(sum(new), width, generator=g, device=DEV) * 0.1).to(dtype)
    offsets = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    single = all(n == 1 for n in new)
    past_dev = torch.tensor(past, dtype=torch.int32, device=DEV)
    lens = [p + n for p, n in zip(past, new)]
    for layer in range(layers):
      codes, scales, z, W = weights[2 * layer]
      h = W.matvec(x)
      check_matvec(codes, scales, z, 64, None, x, h)
      h = (h / h.float().abs().mean()).to(dtype).view(-1, qkv, d)
      q, k, v = h[:, :hq], h[:, hq:hq + hkv], h[:, hq + hkv:]
      cache = caches[layer]
      before = cache.k.clone(), cache.v.clone()
      turned = cache.append(k, v, table, past_dev, q=q, offsets=None if single else offsets, inv_freq=inv_freq)
      check_append(cache, k, v, q, table, past, new, inv_freq, False, turned, before)
      # the last token of every utterance that has one attends
      rows = [b for b, n in enumerate(new) if n]
      last = torch.tensor([int(offsets[b + 1]) - 1 for b in rows], device=DEV)
      got = cache.attend(turned[last], table[rows], torch.tensor([lens[b] for b in rows], dtype=torch.int32, device=DEV), return_lse=True)
      check_attend(cache, turned[last], table[rows], [lens[b] for b in rows], d ** -0.5, 0, got)
      cache.check()
      codes, scales, z, W = weights[2 * layer + 1]
      y = W.matvec(got[0].flatten(1))
      check_matvec(codes, scales, z, 64, None, got[0].flatten(1), y)
      x = x.clone()
      x[last] += (y / y.float().abs().mean() * 0.1).to(dtype)
    past = lens


def test_matrix_and_step_in_a_graph():
  """A captured step of one layer (projection, append, attend, projection), replayed with new inputs; every replay equals the
  eager calls on the same inputs, which run in between."""
  from tacotron_amd.w4 import W4Matrix
  g = gen(31)
  width, hq, hkv, d = 192, 4, 2, 48
  qkv = hq + 2 * hkv
  W = [W4Matrix.from_weights(torch.randn(n, k, generator=g, device=DEV).to(BF16), group=64, symmetric=False)
       for n, k in ((qkv * d, width), (width, hq * d))]
  caches = [make_cache(12, 32, hkv, d, BF16, gen(8)) for _ in range(2)]
  table = make_table([4, 4, 3], 12, 4, 5)
  past = torch.tensor([0, 31, 64], dtype=torch.int32, device=DEV)
  inv_freq = torch.rand(8, generator=g, device=DEV, dtype=torch.float64)
  x = torch.zeros(3, width, dtype=BF16, device=DEV)

  def step(cache):
    h = W[0].matvec(x).view(3, qkv, d)
    q = cache.append(h[:, hq:hq + hkv], h[:, hq + hkv:], table, past, q=h[:, :hq], inv_freq=inv_freq, interleaved=True)
    return W[1].matvec(cache.attend(q, table, past + 1).flatten(1))
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step(caches[0])
  for _ in range(8):
    x.copy_(torch.randn(3, width, generator=g, device=DEV))
    graph.replay()
    want = step(caches[1])
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    past += 1
  for c in caches:
    c.check()
  assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)


def test_matvec_on_two_streams():
  """One matrix, two streams at once, each as alone."""
  from tacotron_amd.w4 import W4Matrix
  g = gen(33)
  W = W4Matrix.from_weights(torch.randn(5000, 700, generator=g, device=DEV).to(F16), group=32)
  xs = [torch.randn(n, 700, generator=g, device=DEV).to(F16) for n in (1, 16)]
  want = [W.matvec(x) for x in xs]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream(device=DEV) for _ in range(2)]
  got = []
  for _ in range(10):
    for s, x in zip(streams, xs):
      with torch.cuda.stream(s):
        got.append(W.matvec(x))
  torch.cuda.synchronize()
  for i, y in enumerate(got):
    assert torch.equal(y, want[i % 2])
