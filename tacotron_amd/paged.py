"""A paged cache of keys and values for a decoder with self-attention, on the HIP library's ``taco_kv_*`` entry points
(include/taco.h): ``PagedCache.append`` stores the keys and values of new frames with the position rotation applied on the
way, ``PagedCache.attend`` is the attention of one new frame per utterance over them.  The reference has no counterpart (its
decoder step is src/tacotron/model.py:454-491).

Everything is enqueued on the device's current stream and nothing waits, so calls can be captured into a graph; what only
the device can see - a table entry that is no page, a length beyond the table - is reported by ``PagedCache.check()``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch

from tacotron_amd import _lib, abi


def _device(device: Union[torch.device, str, int]) -> torch.device:
  device = torch.device(device)
  if device.type != "cuda":
    raise RuntimeError(f"the cache lives on an AMD GPU only (got device '{device}'); there is no CPU path")
  return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


def _check_vector(t: torch.Tensor, name: str, dtype: torch.dtype, size: int, device: torch.device) -> None:
  if t.dtype != dtype or t.dim() != 1 or t.shape[0] != size or t.device != device or not t.is_contiguous():
    raise ValueError(f"{name} must be a contiguous {dtype} [{size}] tensor on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _rows_ok(t: torch.Tensor) -> bool:
  """Whether the kernels can read ``t`` as it is: unit stride in the last dimension, rows at multiples of 16 bytes."""
  size = t.element_size()
  return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * size % 16 == 0 for s in t.stride()[:-1])


class PagedCache:
  """``n_pages`` pages of ``page_size`` tokens of ``n_heads`` heads of ``head_dim`` elements, keys and values.

  ``k`` and ``v`` are tensors [n_pages, page_size, n_heads, head_dim] (a view: a page's tokens of one head lie side by
  side in memory).  ``page_size`` and ``head_dim`` are multiples of 16, ``head_dim`` at most 256.  Which pages belong to an
  utterance says a table, int32 [utterances, pages], that the caller keeps: token t is in slot ``t % page_size`` of page
  ``table[b, t // page_size]``.  ``dtype`` is float32, float16, bfloat16 or float8_e4m3fn; the last holds x / scale with
  one scale per head (``k_scale`` / ``v_scale``, float32 [n_heads], 1 when not given).

  Pages and tables are the caller's to hand out; calls on different streams may overlap as long as they touch different
  pages."""

  def __init__(self, n_pages: int, page_size: int, n_heads: int, head_dim: int, dtype: torch.dtype = torch.float32,
               device: Union[torch.device, str, int] = "cuda", k_scale: Optional[torch.Tensor] = None,
               v_scale: Optional[torch.Tensor] = None):
    device = _device(device)
    if min(n_pages, page_size, n_heads, head_dim) < 1:
      raise ValueError(f"a cache of {n_pages} pages of {page_size} tokens of {n_heads} heads of {head_dim} elements")
    shape = (n_pages, n_heads, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
    self._init(k, v, k_scale, v_scale)

  @classmethod
  def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None) -> "PagedCache":
    """A cache over tensors [n_pages, page_size, n_heads, head_dim] that the caller has allocated, in any order of pages,
    tokens and heads (unit stride in head_dim, rows at multiples of 16 bytes)."""
    self = cls.__new__(cls)
    self._init(k, v, k_scale, v_scale)
    return self

  def _init(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor]) -> None:
    if k.dtype not in abi.DTYPES or v.dtype != k.dtype:
      raise ValueError(f"a cache holds one of {', '.join(str(d) for d in abi.DTYPES)}, not {k.dtype} / {v.dtype}")
    if k.dim() != 4 or v.shape != k.shape or v.device != k.device:
      raise ValueError(f"k and v must be [n_pages, page_size, n_heads, head_dim] on one device, got {tuple(k.shape)} / {tuple(v.shape)}")
    n_pages, page_size, n_heads, head_dim = k.shape
    if page_size < 16 or page_size % 16 or head_dim < 16 or head_dim % 16 or head_dim > 256 or min(n_pages, n_heads) < 1:
      raise ValueError(f"page_size {page_size} and head_dim {head_dim} must be multiples of 16, head_dim at most 256, and "
                       f"neither pages ({n_pages}) nor heads ({n_heads}) may be missing")
    self.device = _device(k.device)
    if not (_rows_ok(k) and _rows_ok(v)):
      raise ValueError("rows of the cache must have unit stride and start at multiples of 16 bytes")
    if k.dtype == torch.float8_e4m3fn:
      k_scale, v_scale = (torch.ones(n_heads, device=self.device) if s is None else s for s in (k_scale, v_scale))
      _check_vector(k_scale, "k_scale", torch.float32, n_heads, self.device)
      _check_vector(v_scale, "v_scale", torch.float32, n_heads, self.device)
    elif k_scale is not None or v_scale is not None:
      raise ValueError(f"scales belong to an 8-bit cache, not to {k.dtype}")
    self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
    self._flags = torch.zeros(1, dtype=torch.int32, device=self.device)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    self._c = abi.TacoKvCache(
      k=p(k), v=p(v), k_stride=tuple(k.stride()[:3]), v_stride=tuple(v.stride()[:3]), k_scale=p(k_scale), v_scale=p(v_scale),
      flags=p(self._flags), n_pages=n_pages, page_size=page_size, n_heads=n_heads, head_dim=head_dim,
      dtype=abi.DTYPES[k.dtype], device=self.device.index)
    self._ref = C.byref(self._c)
    self._takes = (torch.float16, torch.bfloat16) if k.dtype == torch.float8_e4m3fn else (k.dtype,)
    self._lib = _lib.lib()

  @property
  def n_pages(self) -> int:
    return self.k.shape[0]

  @property
  def page_size(self) -> int:
    return self.k.shape[1]

  @property
  def n_heads(self) -> int:
    return self.k.shape[2]

  @property
  def head_dim(self) -> int:
    return self.k.shape[3]

  def _stream(self) -> int:
    return torch.cuda.current_stream(self.device).cuda_stream

  def _rows(self, t: torch.Tensor, name: str, tokens: int, heads: Optional[int]) -> torch.Tensor:
    """``t`` [tokens, heads, head_dim] checked, as the kernels can read it (a copy where its rows are not aligned)."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != self.head_dim or (shape[1] != heads if heads else shape[1] < 1):
      raise ValueError(f"{name} must be [{tokens}, {heads or 'heads'}, {self.head_dim}], got {tuple(shape)}")
    if t.dtype not in self._takes or t.device != self.device:
      raise ValueError(f"{name} must be {' or '.join(str(d) for d in self._takes)} on {self.device}, got {t.dtype} on {t.device}")
    return t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format)

  def _out(self, out: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    if out is None:
      return torch.empty(like.shape, dtype=like.dtype, device=self.device)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != self.device or not _rows_ok(out):
      raise ValueError(f"out must be {like.dtype} {tuple(like.shape)} on {self.device} with unit stride and rows at multiples of "
                       f"16 bytes, got {out.dtype} {tuple(out.shape)} on {out.device}")
    return out

  def _index(self, t: torch.Tensor, name: str, size: int) -> int:
    if t.dtype != torch.int32 or t.shape != (size,) or t.device != self.device or not t.is_contiguous():
      raise ValueError(f"{name} must be a contiguous int32 [{size}] tensor on {self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()

  def _table(self, table: torch.Tensor) -> Tuple[int, int]:
    if table.dtype != torch.int32 or table.dim() != 2 or table.device != self.device:
      raise ValueError(f"table must be int32 [utterances, pages] on {self.device}, got {table.dtype} {tuple(table.shape)} on {table.device}")
    if table.shape[1] > 1 and table.stride(1) != 1:
      raise ValueError("the pages of an utterance must lie side by side in the table")
    return table.shape

  def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, past: torch.Tensor,
             q: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
             inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
             out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Stores new tokens: ``k``, ``v`` [tokens, n_heads, head_dim]; ``past`` int32 [utterances] is how many tokens of each
    utterance the cache holds already.  Without ``offsets`` there is one new token per utterance; with ``offsets`` (int32
    [utterances + 1], rising) rows ``offsets[b]:offsets[b + 1]`` are utterance b's.  ``inv_freq`` (float64 [R / 2], R a
    multiple of 16 up to head_dim) rotates the first R elements of every key head by ``position * inv_freq``: the pairs
    (i, i + R/2), or (2i, 2i + 1) with ``interleaved``.  ``q`` [tokens, query heads, head_dim] are queries of the same
    tokens, rotated likewise: returned, or written to ``out`` (which may be ``q``).  Rows that belong to no utterance are
    left as they were in ``out``.  No two tokens of a call may go to the same place, and ``out`` may overlap no other
    input."""
    n, width = self._table(table)
    k, v = self._rows(k, "k", k.shape[0], self.n_heads), self._rows(v, "v", k.shape[0], self.n_heads)
    tokens = k.shape[0]
    if offsets is None and tokens != n:
      raise ValueError(f"{tokens} tokens for {n} utterances need offsets")
    a = abi.TacoKvAppendArgs(
      k=k.data_ptr(), v=v.data_ptr(), table=table.data_ptr(), past=self._index(past, "past", n),
      k_stride=k.stride()[:2], v_stride=v.stride()[:2], table_stride=table.stride(0), n_tokens=tokens, n_seqs=n,
      table_width=width, interleaved=bool(interleaved), dtype=abi.DTYPES[k.dtype])
    if offsets is not None:
      a.offsets = self._index(offsets, "offsets", n + 1)
    if v.dtype != k.dtype:
      raise ValueError(f"k and v differ in type: {k.dtype}, {v.dtype}")
    if inv_freq is not None:
      if inv_freq.dim() != 1 or inv_freq.shape[0] % 8 or 2 * inv_freq.shape[0] > self.head_dim:
        raise ValueError(f"inv_freq must have a multiple of 8 frequencies, at most head_dim / 2 = {self.head_dim // 2}, got {tuple(inv_freq.shape)}")
      _check_vector(inv_freq, "inv_freq", torch.float64, inv_freq.shape[0], self.device)
      a.inv_freq, a.rot_dim = inv_freq.data_ptr(), 2 * inv_freq.shape[0]
    if q is not None:
      rows = self._rows(q, "q", tokens, None)
      if q.dtype != k.dtype:
        raise ValueError(f"q and k differ in type: {q.dtype}, {k.dtype}")
      out = self._out(out, q)
      a.q, a.q_out, a.n_q_heads = rows.data_ptr(), out.data_ptr(), q.shape[1]
      a.q_stride, a.q_out_stride = rows.stride()[:2], out.stride()[:2]
    elif out is not None:
      raise ValueError("out without q")
    if tokens:
      _lib.check(self._lib.taco_kv_append(self._ref, C.byref(a), self._stream()))
    return out

  def attend(self, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, scale: Optional[float] = None, window: int = 0,
             return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of one new token per utterance: ``q`` [utterances, query heads, head_dim] over the first ``lens`` (int32
    [utterances]) tokens of each, or the last ``window`` of those; ``scale`` defaults to head_dim ** -0.5.  Query head h
    reads cache head ``h // (query heads / n_heads)``.  Returns the output like ``q`` (or in ``out``) and, with
    ``return_lse``, the logarithm of the softmax's sum, float32 [utterances, query heads].  An utterance that sees nothing
    (length 0, or no score above -inf) gets zeros and -inf.  What lies in slots at and behind ``lens`` does not matter; an
    infinite value that is seen gives NaN."""
    n, width = self._table(table)
    rows = self._rows(q, "q", n, None)
    heads = q.shape[1]
    if heads % self.n_heads:
      raise ValueError(f"{heads} query heads cannot share {self.n_heads} cache heads evenly")
    if window < 0:
      raise ValueError(f"window must not be negative, got {window}")
    out = self._out(out, q)
    lse = torch.empty(n, heads, dtype=torch.float32, device=self.device) if return_lse else None
    a = abi.TacoKvAttendArgs(
      q=rows.data_ptr(), out=out.data_ptr(), table=table.data_ptr(), lens=self._index(lens, "lens", n),
      q_stride=rows.stride()[:2], out_stride=out.stride()[:2], table_stride=table.stride(0),
      scale=self.head_dim ** -0.5 if scale is None else scale, window=window, n_seqs=n, table_width=width, n_q_heads=heads,
      dtype=abi.DTYPES[q.dtype])
    if return_lse:
      a.lse = lse.data_ptr()
    if n:
      need = self._lib.taco_kv_attend_workspace(self._ref, C.byref(a))
      if need < 0:
        _lib.check(int(need))
      if need:      # allocated per call: the allocator orders its reuse by stream, and a captured graph gets one of its own
        work = torch.empty(need, dtype=torch.uint8, device=self.device)
        a.workspace, a.workspace_bytes = work.data_ptr(), need
      _lib.check(self._lib.taco_kv_attend(self._ref, C.byref(a), self._stream()))
    return (out, lse) if return_lse else out

  def check(self) -> None:
    """Waits for the current stream and raises an IndexError if a call since the last check has met a table entry that is
    no page of the cache, or a position or length outside its table (such tokens are neither stored nor seen)."""
    _lib.check(self._lib.taco_kv_status(self._ref, self._stream()))
