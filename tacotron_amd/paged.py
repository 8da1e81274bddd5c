"""A paged cache of keys and values for a decoder with self-attention, on the HIP library's ``taco_kv_*`` entry points
(include/taco.h): ``PagedCache.append`` stores the keys and values of new frames with the position rotation applied on the
way, ``PagedCache.attend`` is the attention of one new frame per utterance over them.  The reference has no counterpart (its
decoder step is src/tacotron/model.py:454-491).

Everything is enqueued on the device's current stream and nothing waits, so calls can be captured into a graph; what only
the device can see - a table entry that is no page, a length beyond the table - is reported by ``PagedCache.check()``.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Dict, Optional, Tuple, Union

import torch

from tacotron_amd import _lib, abi


# A call's argument block is its addresses, packed here, followed by what its tensors' forms say, kept per form.
_APPEND_POINTERS = struct.Struct("8Q")      # k, v, q, q_out, table, past, offsets, inv_freq
_ATTEND_POINTERS = struct.Struct("6Q")      # q, out, lse, table, lens, workspace
_MOST_FORMS = 256


def _form(t: torch.Tensor) -> Tuple:
  return t.shape, t.stride(), t.dtype, t.get_device()


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


def _apart(t: torch.Tensor) -> bool:
  """Whether no two elements of ``t`` share an address."""
  extent = 1
  for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
    if stride < extent:
      return False
    extent = stride * (size - 1) + extent
  return True


class PagedCache:
  """``n_pages`` pages of ``page_size`` tokens of ``n_heads`` heads of ``head_dim`` elements, keys and values.

  ``k`` and ``v`` are tensors [n_pages, page_size, n_heads, head_dim] (a view: a page's tokens of one head lie side by
  side in memory).  ``page_size`` and ``head_dim`` are multiples of 16, ``head_dim`` at most 256.  Which pages belong to an
  utterance says a table, int32 [utterances, pages], that the caller keeps: token t is in slot ``t % page_size`` of page
  ``table[b, t // page_size]``.  ``dtype`` is float32, float16, bfloat16 or float8_e4m3fn; the last holds x / scale with
  one scale per head (``k_scale`` / ``v_scale``, float32 [n_heads], 1 when not given).

  ``append`` takes any number of new tokens of an utterance, ``attend`` the queries of one, its last: the attention among a
  prompt's own tokens is not offered here.  Pages and tables are the caller's to hand out; calls on different streams may
  overlap as long as none writes a page that another reads or writes.  Inference only: results carry no gradients."""

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
    if not (_rows_ok(k) and _rows_ok(v) and _apart(k) and _apart(v)):
      raise ValueError("rows of the cache must have unit stride, start at multiples of 16 bytes and not overlap")
    if k.dtype == torch.float8_e4m3fn:
      k_scale, v_scale = (torch.ones(n_heads, device=self.device) if s is None else s for s in (k_scale, v_scale))
      _check_vector(k_scale, "k_scale", torch.float32, n_heads, self.device)
      _check_vector(v_scale, "v_scale", torch.float32, n_heads, self.device)
    elif k_scale is not None or v_scale is not None:
      raise ValueError(f"scales belong to an 8-bit cache, not to {k.dtype}")
    self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
    self._flags = torch.zeros(1, dtype=torch.int32, device=self.device)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    self._c = abi.TacoKvCache(
      k=p(k), v=p(v), k_stride=tuple(k.stride()[:3]), v_stride=tuple(v.stride()[:3]), k_scale=p(k_scale), v_scale=p(v_scale),
      flags=p(self._flags), n_pages=n_pages, page_size=page_size, n_heads=n_heads, head_dim=head_dim,
      dtype=abi.DTYPES[k.dtype], device=self.device.index)
    self._ref = C.byref(self._c)
    self._takes = (torch.float16, torch.bfloat16) if k.dtype == torch.float8_e4m3fn else (k.dtype,)
    self._lib = _lib.lib()
    # what a call's checks have found, by the shapes, strides, types and devices of its tensors (never by their addresses)
    self._append_forms: Dict[Tuple, bytes] = {}
    self._attend_forms: Dict[Tuple, Tuple[bytes, int, torch.Tensor]] = {}

  @property
  def k(self) -> torch.Tensor:
    return self._k

  @property
  def v(self) -> torch.Tensor:
    return self._v

  @property
  def k_scale(self) -> Optional[torch.Tensor]:
    return self._k_scale

  @property
  def v_scale(self) -> Optional[torch.Tensor]:
    return self._v_scale

  @property
  def n_pages(self) -> int:
    return self._k.shape[0]

  @property
  def page_size(self) -> int:
    return self._k.shape[1]

  @property
  def n_heads(self) -> int:
    return self._k.shape[2]

  @property
  def head_dim(self) -> int:
    return self._k.shape[3]

  def _rows(self, t: torch.Tensor, name: str, tokens: int, heads: Optional[int]) -> None:
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != self.head_dim or (shape[1] != heads if heads else shape[1] < 1):
      raise ValueError(f"{name} must be [{tokens}, {heads or 'heads'}, {self.head_dim}], got {tuple(shape)}")
    if t.dtype not in self._takes or t.device != self.device:
      raise ValueError(f"{name} must be {' or '.join(str(d) for d in self._takes)} on {self.device}, got {t.dtype} on {t.device}")

  def _out(self, out: torch.Tensor, like: torch.Tensor) -> None:
    if out.shape != like.shape or out.dtype != like.dtype or out.device != self.device or not _rows_ok(out) or not _apart(out):
      raise ValueError(f"out must be {like.dtype} {tuple(like.shape)} on {self.device} with unit stride and separate rows at "
                       f"multiples of 16 bytes, got {out.dtype} {tuple(out.shape)} on {out.device}")

  def _index(self, t: torch.Tensor, name: str, size: int) -> None:
    if t.dtype != torch.int32 or t.shape != (size,) or t.device != self.device or not t.is_contiguous():
      raise ValueError(f"{name} must be a contiguous int32 [{size}] tensor on {self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")

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
    left as they were in ``out``.  No two tokens of a call may go to the same place, keys and values of the cache may not share
    memory, and ``out`` may be ``q`` but else overlap no input."""
    interleaved = bool(interleaved)
    key = (_form(k), _form(v), _form(table), _form(past), None if q is None else _form(q), None if offsets is None else _form(offsets),
           None if inv_freq is None else _form(inv_freq), interleaved, None if out is None else _form(out))
    tail = self._append_forms.get(key)
    kp, vp, qp = k.data_ptr(), v.data_ptr(), 0 if q is None else q.data_ptr()
    op = 0 if out is None else out.data_ptr()
    if tail is None or (kp | vp | qp | op) % 16:
      rows = [None if t is None else t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format) for t in (k, v, q)]
      tail = self._append_tail(rows[0], rows[1], table, past, rows[2], offsets, inv_freq, interleaved, out)
      if rows[0] is k and rows[1] is v and rows[2] is q:
        if len(self._append_forms) >= _MOST_FORMS:
          self._append_forms.clear()
        self._append_forms[key] = tail
      k, v = rows[0], rows[1]      # kept until the call is enqueued
      kp, vp, qp = k.data_ptr(), v.data_ptr(), 0 if q is None else rows[2].data_ptr()
    if q is not None and out is None:
      out = _lib.new(q)
      op = out.data_ptr()
    if kp:      # no tokens have no address
      head = _APPEND_POINTERS.pack(kp, vp, qp, op, table.data_ptr(), past.data_ptr(), 0 if offsets is None else offsets.data_ptr(),
                                   0 if inv_freq is None else inv_freq.data_ptr())
      rc = self._lib.taco_kv_append(self._ref, head + tail, _lib.raw_stream(self._c.device))
      if rc:
        _lib.check(rc)
    return out

  def _append_tail(self, k, v, table, past, q, offsets, inv_freq, interleaved, out) -> bytes:
    """Checks an append's tensors and returns the part of its argument block that their forms decide."""
    n, width = self._table(table)
    self._rows(k, "k", k.shape[0] if k.dim() else -1, self.n_heads)
    self._rows(v, "v", k.shape[0], self.n_heads)
    tokens = k.shape[0]
    if offsets is None and tokens != n:
      raise ValueError(f"{tokens} tokens for {n} utterances need offsets")
    if v.dtype != k.dtype:
      raise ValueError(f"k and v differ in type: {k.dtype}, {v.dtype}")
    self._index(past, "past", n)
    if offsets is not None:
      self._index(offsets, "offsets", n + 1)
    a = abi.TacoKvAppendArgs(
      k_stride=k.stride()[:2], v_stride=v.stride()[:2], table_stride=table.stride(0), n_tokens=tokens, n_seqs=n,
      table_width=width, interleaved=interleaved, dtype=abi.DTYPES[k.dtype])
    if inv_freq is not None:
      if inv_freq.dim() != 1 or inv_freq.shape[0] % 8 or 2 * inv_freq.shape[0] > self.head_dim:
        raise ValueError(f"inv_freq must have a multiple of 8 frequencies, at most head_dim / 2 = {self.head_dim // 2}, got {tuple(inv_freq.shape)}")
      _check_vector(inv_freq, "inv_freq", torch.float64, inv_freq.shape[0], self.device)
      a.rot_dim = 2 * inv_freq.shape[0]
    if q is not None:
      self._rows(q, "q", tokens, None)
      if q.dtype != k.dtype:
        raise ValueError(f"q and k differ in type: {q.dtype}, {k.dtype}")
      if out is not None:
        self._out(out, q)
      a.n_q_heads, a.q_stride = q.shape[1], q.stride()[:2]
      a.q_out_stride = (q.shape[1] * q.shape[2], q.shape[2]) if out is None else out.stride()[:2]
    elif out is not None:
      raise ValueError("out without q")
    return bytes(a)[_APPEND_POINTERS.size:]

  def attend(self, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, scale: Optional[float] = None, window: int = 0,
             return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of one new token per utterance: ``q`` [utterances, query heads, head_dim] over the first ``lens`` (int32
    [utterances]) tokens of each, or the last ``window`` of those; ``scale`` defaults to head_dim ** -0.5.  Query head h
    reads cache head ``h // (query heads / n_heads)``.  Returns the output like ``q`` (or in ``out``, which may be ``q``
    and else overlaps no input) and, with ``return_lse``, the logarithm of the softmax's sum, float32 [utterances, query
    heads].  An utterance that sees nothing (length 0, or no score above -inf) gets zeros and -inf.  What lies in slots at
    and behind ``lens`` does not matter; an infinite value that is seen gives NaN."""
    scale, window = None if scale is None else float(scale), int(window)      # numbers: a tensor would stand for itself in the key
    key = (_form(q), _form(table), _form(lens), scale, window, None if out is None else _form(out))
    found = self._attend_forms.get(key)
    qp, op = q.data_ptr(), 0 if out is None else out.data_ptr()
    if found is None or (qp | op) % 16:
      rows = q if _rows_ok(q) else q.clone(memory_format=torch.contiguous_format)
      found = self._attend_tail(rows, table, lens, scale, window, out)
      if rows is q:
        if len(self._attend_forms) >= _MOST_FORMS:
          self._attend_forms.clear()
        self._attend_forms[key] = found
      q = rows      # kept until the call is enqueued
      qp = q.data_ptr()
    tail, need, lse_form = found
    if out is None:
      out = _lib.new(q)
      op = out.data_ptr()
    lse = _lib.new(lse_form) if return_lse else None
    if op:        # no utterances have no address
      # allocated per call: the allocator orders its reuse by stream, and a captured graph gets one of its own
      work = torch.empty(need, dtype=torch.uint8, device=self.device)
      head = _ATTEND_POINTERS.pack(qp, op, 0 if lse is None else lse.data_ptr(), table.data_ptr(), lens.data_ptr(), work.data_ptr())
      rc = self._lib.taco_kv_attend(self._ref, head + tail, _lib.raw_stream(self._c.device))
      if rc:
        _lib.check(rc)
    return (out, lse) if return_lse else out

  def _attend_tail(self, q, table, lens, scale, window, out) -> Tuple[bytes, int, torch.Tensor]:
    """Checks an attend's tensors; the part of its argument block that their forms decide, the size of its workspace, the form
    of its logarithms."""
    n, width = self._table(table)
    self._rows(q, "q", n, None)
    heads = q.shape[1]
    if heads % self.n_heads:
      raise ValueError(f"{heads} query heads cannot share {self.n_heads} cache heads evenly")
    if window < 0:
      raise ValueError(f"window must not be negative, got {window}")
    self._index(lens, "lens", n)
    if out is not None:
      self._out(out, q)
    a = abi.TacoKvAttendArgs(
      q_stride=q.stride()[:2], out_stride=(heads * self.head_dim, self.head_dim) if out is None else out.stride()[:2],
      table_stride=table.stride(0), scale=self.head_dim ** -0.5 if scale is None else scale,
      window=min(window, 2 ** 31 - 1), n_seqs=n,
      table_width=width, n_q_heads=heads, dtype=abi.DTYPES[q.dtype])
    need = self._lib.taco_kv_attend_workspace(self._ref, C.byref(a))
    if need < 0:
      _lib.check(int(need))
    a.workspace_bytes = need
    return bytes(a)[_ATTEND_POINTERS.size:], need, _lib.shape_of((n, heads), torch.float32, self.device)

  def check(self) -> None:
    """Waits for the current stream and raises an IndexError if a call since the last check has met a table entry that is
    no page of the cache, or a position or length outside its table (such tokens are neither stored nor seen).  What calls on
    other streams find after that is raised by the next check."""
    _lib.check(self._lib.taco_kv_status(self._ref, _lib.raw_stream(self._c.device)))
