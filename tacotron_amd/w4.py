"""Matrices of 4-bit weights with group scales and their products with a few vectors, on the HIP library's ``taco_qmat_*``
entry points (include/taco.h).  The reference has no counterpart: it computes with fp32 weights only."""
from __future__ import annotations

import ctypes as C
from typing import Dict, Optional, Tuple

import torch

from tacotron_amd import _lib, abi

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _on_gpu(t: torch.Tensor, name: str) -> torch.device:
  if t.device.type != "cuda":
    raise RuntimeError(f"{name} must be on an AMD GPU (got device '{t.device}'); there is no CPU path")
  return t.device


def _check(t: torch.Tensor, name: str, shape: Tuple[int, ...], dtypes, device: torch.device) -> None:
  if tuple(t.shape) != shape or t.dtype not in dtypes or t.device != device:
    raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)} {list(shape)} on {device}, got {t.dtype} "
                     f"{tuple(t.shape)} on {t.device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
  """``t`` if its rows lie apart and their elements side by side, or a copy (of a matrix with one row for all, say)."""
  apart = t.shape[0] == 1 or t.stride(0) >= t.shape[1]
  return t if apart and (t.shape[1] == 1 or t.stride(1) == 1) else t.clone(memory_format=torch.contiguous_format)


def _pitch(t: torch.Tensor) -> int:
  """Elements from row to row (a single row may have any stride)."""
  return t.shape[1] if t.shape[0] == 1 else t.stride(0)


def quantize(weight: torch.Tensor, group: int = 128, symmetric: bool = True,
             scale_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
  """Codes, scales and zero points (None if ``symmetric``) of ``weight`` [out, in], which must be finite, as
  ``W4Matrix.from_codes`` takes them: the scale of a group is max|w| / 7, or (max - min) / 15 with zero points, and a code the
  nearest to its weight.  ``scale_dtype`` defaults to the weight's type; a scale beyond its range becomes its largest number."""
  device = _on_gpu(weight, "weight")
  if weight.dim() != 2 or weight.dtype not in _FLOATS or weight.numel() == 0:
    raise ValueError(f"weight must be a float matrix, got {weight.dtype} {tuple(weight.shape)}")
  scale_dtype = scale_dtype or weight.dtype
  if group not in (32, 64, 128) or scale_dtype not in _FLOATS:
    raise ValueError(f"groups are 32, 64 or 128 columns (got {group}), scales float32, float16 or bfloat16 (got {scale_dtype})")
  n, k = weight.shape
  groups = -(-k // group)
  weight = _rows(weight)
  codes = torch.empty(n, -(-k // 2), dtype=torch.uint8, device=device)
  scales = torch.empty(n, groups, dtype=scale_dtype, device=device)
  zeros = None if symmetric else torch.empty(n, groups, dtype=torch.uint8, device=device)
  m = abi.TacoQmat(n_rows=n, n_cols=k, group=group, scale_dtype=abi.DTYPES[scale_dtype], has_zeros=not symmetric, device=device.index)
  _lib.check(_lib.lib().taco_qmat_quantize(
    C.byref(m), weight.data_ptr(), _pitch(weight), abi.DTYPES[weight.dtype], codes.data_ptr(), codes.shape[1], scales.data_ptr(),
    groups, None if zeros is None else zeros.data_ptr(), groups, torch.cuda.current_stream(device).cuda_stream))
  return codes, scales, zeros


class W4Matrix:
  """A matrix [out_features, in_features] of 4-bit codes: W[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group]),
  zero = 8 without zero points.  It owns a copy of them in the order the kernel reads, made once."""

  def __init__(self, packed: torch.Tensor, bias: Optional[torch.Tensor], c: abi.TacoQmat):
    self._packed, self._bias, self._c = packed, bias, c
    self._ref = C.byref(c)
    self.device, self.in_features, self.out_features, self.group = packed.device, c.n_cols, c.n_rows, c.group
    self._lib = _lib.lib()
    # vectors, row strides and result of a call, by the shapes, strides, types and devices of its tensors
    self._forms: Dict[Tuple, Tuple] = {}

  @classmethod
  def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, in_features: Optional[int] = None, group: Optional[int] = None) -> "W4Matrix":
    """``codes`` uint8 [out, >= ceil(in / 2)], two columns in a byte, the even one in its low half; ``scales`` [out, groups]
    float32, float16 or bfloat16; ``zeros`` uint8 [out, groups], 0 .. 15; ``bias`` [out].  ``in_features`` defaults to all the
    codes there are; ``group`` (32, 64 or 128) to the one that the number of scales leaves."""
    device = _on_gpu(codes, "codes")
    if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.numel() == 0:
      raise ValueError(f"codes must be uint8 [out, in / 2], got {codes.dtype} {tuple(codes.shape)}")
    n, k = codes.shape[0], 2 * codes.shape[1] if in_features is None else int(in_features)
    if not 1 <= k <= 2 * codes.shape[1]:
      raise ValueError(f"codes of {2 * codes.shape[1]} columns cannot have {k} in_features")
    if scales.dim() != 2:
      raise ValueError(f"scales must be [out, groups], got {tuple(scales.shape)}")
    fits = [g for g in ((32, 64, 128) if group is None else (group,)) if g in (32, 64, 128) and -(-k // g) == scales.shape[1]]
    if len(fits) != 1:
      raise ValueError(f"{scales.shape[1]} scales a row for {k} columns fit groups of {fits or 'no allowed size'}"
                       f"{'' if group is None else f' ({group} given)'}: groups are 32, 64 or 128 columns")
    _check(scales, "scales", (n, scales.shape[1]), _FLOATS, device)
    if zeros is not None:
      _check(zeros, "zeros", tuple(scales.shape), (torch.uint8,), device)
      zeros = _rows(zeros)
    if bias is not None:
      _check(bias, "bias", (n,), _FLOATS, device)
      bias = bias.detach().to(torch.float32, copy=True).contiguous()
    codes, scales = _rows(codes), _rows(scales)
    m = abi.TacoQmat(n_rows=n, n_cols=k, group=fits[0], scale_dtype=abi.DTYPES[scales.dtype], has_zeros=zeros is not None,
                     device=device.index)
    L = _lib.lib()
    size = L.taco_qmat_bytes(C.byref(m))
    if size < 0:
      _lib.check(int(size))
    packed = torch.empty(size, dtype=torch.uint8, device=device)
    _lib.check(L.taco_qmat_pack(
      C.byref(m), codes.data_ptr(), _pitch(codes), scales.data_ptr(), _pitch(scales), None if zeros is None else zeros.data_ptr(),
      0 if zeros is None else _pitch(zeros), packed.data_ptr(), torch.cuda.current_stream(device).cuda_stream))
    m.packed, m.bias = packed.data_ptr(), None if bias is None else bias.data_ptr()
    return cls(packed, bias, m)

  @classmethod
  def from_weights(cls, weight: torch.Tensor, group: int = 128, symmetric: bool = True, scale_dtype: Optional[torch.dtype] = None,
                   bias: Optional[torch.Tensor] = None) -> "W4Matrix":
    """The nearest 4-bit matrix to ``weight`` [out, in] (see ``quantize``)."""
    codes, scales, zeros = quantize(weight, group, symmetric, scale_dtype)
    return cls.from_codes(codes, scales, zeros=zeros, bias=bias, in_features=weight.shape[1], group=group)

  @property
  def nbytes(self) -> int:
    """Bytes that a product reads of the matrix."""
    return self._packed.numel()

  def matvec(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x W^T + bias for vectors ``x`` [..., in_features] in float32, float16 or bfloat16; the result [..., out_features] has
    x's type, its sums are fp32 and rounded once (an infinite element gives NaN).  ``out`` may not overlap ``x``.  Meant for a few vectors: the matrix is read
    again for every 32 (every 16 in float32).  Inference only: results carry no gradients."""
    key = (x.shape, x.stride(), x.dtype, x.get_device()) if out is None else \
          (x.shape, x.stride(), x.dtype, x.get_device(), out.shape, out.stride(), out.dtype, out.get_device())
    form = self._forms.get(key)
    if form is None:
      form = self._form(x, out)
      if len(self._forms) >= 256:
        self._forms.clear()
      self._forms[key] = form
    n, x_pitch, y_pitch, code, want, copies = form
    if copies:        # columns apart, expanded or overlapping vectors
      x = x.contiguous()
    if out is None:
      out = _lib.new(want)
    if n:
      xp, op = x.data_ptr(), out.data_ptr()
      if xp == op:
        raise ValueError("out may not be x: every result needs all of its vector")
      rc = self._lib.taco_qmat_multiply(self._ref, xp, x_pitch, op, y_pitch, n, code, _lib.raw_stream(self._c.device))
      if rc:
        _lib.check(rc)
    return out

  def _form(self, x: torch.Tensor, out: Optional[torch.Tensor]) -> Tuple:
    """Checks a product's tensors: vectors, elements from vector to vector and from result to result, type, the result's
    form, whether the vectors have to be copied."""
    shape, k, n = x.shape, self.in_features, self.out_features
    if x.dtype not in _FLOATS or x.device != self.device or len(shape) < 1 or shape[-1] != k:
      raise ValueError(f"x must be a float [..., {k}] tensor on {self.device}, got {x.dtype} {tuple(shape)} on {x.device}")
    vectors = x.numel() // k
    side_by_side = k == 1 or x.stride(-1) == 1
    as_rows = side_by_side and (vectors == 1 or (x.dim() == 2 and x.stride(0) >= k))
    want = (*shape[:-1], n)
    pitch = n
    if out is not None:
      if out.dim() == 2 and out.shape == want and (n == 1 or out.stride(1) == 1) and (vectors <= 1 or out.stride(0) >= n):
        pitch = out.stride(0)
      elif out.shape != want or not out.is_contiguous():
        raise ValueError(f"out must be {want} with its rows side by side, got {tuple(out.shape)} {out.stride()}")
      if out.dtype != x.dtype or out.device != self.device:
        raise ValueError(f"out must be {x.dtype} on {self.device}, got {out.dtype} on {out.device}")
    return (vectors, x.stride(0) if as_rows and vectors > 1 else k, pitch, abi.DTYPES[x.dtype],
            _lib.shape_of(want, x.dtype, self.device), not (as_rows or x.is_contiguous()))
