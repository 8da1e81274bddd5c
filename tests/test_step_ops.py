"""The self-attention step's operators without a GPU: the paged cache's address arithmetic (compiled for the host from the
kernels' header) and what the C entry points refuse before they touch a device."""
import ctypes as C
import os
import random
import subprocess

import pytest

from tacotron_amd import _lib, abi
from conftest import ROOT

SUPPORT = os.path.join(ROOT, "tests", "support")


@pytest.fixture(scope="module")
def place():
  path = os.path.join(SUPPORT, "libplace.so")
  if not os.path.exists(path):
    subprocess.check_call(["make", "-C", SUPPORT, "libplace.so"], stdout=subprocess.DEVNULL)
  return C.CDLL(path)


def test_division_by_a_page_size(place):
  r = random.Random(1)
  for d in [1, 2, 3, 4, 5, 6, 7, 9, 16, 31, 48, 64, 100, 255, 4096, 65535, 65536] + [r.randint(1, 65536) for _ in range(200)]:
    at = {0, 1, d - 1, d, d + 1, 2 ** 30 - 1, (2 ** 30 - 1) // d * d, (2 ** 30 - 1) // d * d - 1}
    for n in at | {r.randrange(2 ** 30) for _ in range(200)}:
      if n >= 0:
        assert place.place_divide(n, d) == n // d, (n, d)


def test_places_in_and_out_of_the_table(place):
  row = (C.c_int32 * 4)(5, 0, -1, 7)
  out = (C.c_int32 * 3)()

  def find(at, width=4, n_pages=7):
    place.place_find(row, width, n_pages, C.c_int64(at), 48, out)
    return tuple(out)
  assert find(0) == (5, 0, 0) and find(47) == (5, 47, 0) and find(48) == (0, 0, 0) and find(95) == (0, 47, 0)
  assert find(96)[0] == -1 and find(96)[2] == 1                       # entry -1
  assert find(150)[0] == -1 and find(150)[2] == 1                     # entry 7 of 7 pages
  assert find(150, n_pages=8) == (7, 6, 0)
  for at in (192, -1, 2 ** 30, 2 ** 31, 2 ** 32 + 5, -2 ** 40):       # behind the table, in front of it, beyond 32 bits
    assert find(at)[0] == -1 and find(at)[2] == 2, at
  assert find(48, width=1)[2] == 2 and find(0, width=0)[2] == 2


def _cache(**change):
  base = dict(k=4096, v=4096, k_stride=(4096, 64, 1024), v_stride=(4096, 64, 1024), flags=64, n_pages=3, page_size=16,
              n_heads=4, head_dim=64, dtype=abi.TACO_BF16, device=0)
  return abi.TacoKvCache(**{**base, **change})


def _append(**change):
  base = dict(k=4096, v=4096, table=64, past=64, k_stride=(256, 64), v_stride=(256, 64), table_stride=3, n_tokens=2, n_seqs=2,
              table_width=3, dtype=abi.TACO_BF16)
  return abi.TacoKvAppendArgs(**{**base, **change})


def _attend(**change):
  base = dict(q=4096, out=4096, table=64, lens=64, q_stride=(512, 64), out_stride=(512, 64), table_stride=3, scale=0.125,
              n_seqs=2, table_width=3, n_q_heads=8, dtype=abi.TACO_BF16)
  return abi.TacoKvAttendArgs(**{**base, **change})


BAD_CACHES = [
  (dict(dtype=4), "dtype"), (dict(dtype=-1), "dtype"), (dict(dtype=abi.TACO_F16), "dtype"), (dict(n_pages=0), "pages"),
  (dict(n_heads=0), "heads"), (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=0), "page_size"),
  (dict(head_dim=72), "head_dim"), (dict(head_dim=272), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(flags=None), "flags"),
  (dict(k_scale=64, v_scale=64), "scales"), (dict(k_scale=64), "scales"), (dict(dtype=abi.TACO_E4M3), "scales"),
  (dict(k=4100), "16 bytes"), (dict(v=None), "16 bytes"), (dict(k_stride=(4096, 60, 1024)), "16 bytes"),
  (dict(v_stride=(4095, 64, 1024)), "16 bytes"),
]


@pytest.mark.parametrize("change,word", BAD_CACHES)
def test_bad_caches_are_refused(change, word):
  L, cache = _lib.lib(), _cache(**change)
  for call in (lambda: L.taco_kv_append(C.byref(cache), C.byref(_append()), None),
               lambda: L.taco_kv_attend(C.byref(cache), C.byref(_attend()), None)):
    with pytest.raises(_lib.TacoError) as e:
      _lib.check(call())
    assert e.value.code == abi.TACO_EINVAL and word in str(e.value)


@pytest.mark.parametrize("change,word", [
  (dict(n_tokens=-1), "tokens"), (dict(n_tokens=1 << 24, offsets=64), "tokens at once"), (dict(n_seqs=-1), "utterances"), (dict(n_tokens=3), "offsets"), (dict(table_width=-1), "table"),
  (dict(rot_dim=8, inv_freq=64), "rot_dim"), (dict(rot_dim=80, inv_freq=64), "rot_dim"), (dict(rot_dim=-16, inv_freq=64), "rot_dim"),
  (dict(rot_dim=32), "frequencies"), (dict(q=4096, n_q_heads=4), "queries"), (dict(q_out=4096, n_q_heads=4), "queries"),
  (dict(q=4096, q_out=4096), "queries"), (dict(table=None), "table"), (dict(past=None), "past"), (dict(k=4098), "16 bytes"),
  (dict(v_stride=(255, 64)), "16 bytes"), (dict(q=4096, q_out=4104, n_q_heads=4, q_stride=(256, 64), q_out_stride=(256, 64)), "16 bytes"),
  (dict(dtype=abi.TACO_F32), "dtype"),
])
def test_bad_appends_are_refused(change, word):
  with pytest.raises(_lib.TacoError) as e:
    _lib.check(_lib.lib().taco_kv_append(C.byref(_cache()), C.byref(_append(**change)), None))
  assert e.value.code == abi.TACO_EINVAL and word in str(e.value)


@pytest.mark.parametrize("change,word", [
  (dict(n_seqs=-1), "utterances"), (dict(n_q_heads=6), "query heads"), (dict(n_q_heads=0), "query heads"), (dict(window=-1), "window"),
  (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(table_width=1 << 27), "pages"),
  (dict(table=None), "table"), (dict(lens=None), "lens"), (dict(q=4100), "16 bytes"), (dict(out=None), "16 bytes"),
  (dict(out_stride=(512, 63)), "16 bytes"), (dict(n_seqs=1 << 29), "utterances of"),
  (dict(n_seqs=1 << 21), "utterances of"), (dict(n_seqs=1 << 10, table_width=(1 << 26) - 1), "utterances of"),
])
def test_bad_attends_are_refused(change, word):
  with pytest.raises(_lib.TacoError) as e:
    _lib.check(_lib.lib().taco_kv_attend(C.byref(_cache()), C.byref(_attend(**change)), None))
  assert e.value.code == abi.TACO_EINVAL and word in str(e.value)


def test_nothing_to_do_and_null_arguments():
  L = _lib.lib()
  assert L.taco_kv_append(C.byref(_cache()), C.byref(_append(n_tokens=0, n_seqs=0)), None) == 0
  assert L.taco_kv_attend(C.byref(_cache()), C.byref(_attend(n_seqs=0)), None) == 0
  for rc in (L.taco_kv_append(None, C.byref(_append()), None), L.taco_kv_append(C.byref(_cache()), None, None),
             L.taco_kv_attend(None, C.byref(_attend()), None), L.taco_kv_attend(C.byref(_cache()), None, None),
             L.taco_kv_attend_workspace(C.byref(_cache()), None), L.taco_kv_status(None, None)):
    assert rc == abi.TACO_EINVAL


def test_struct_layouts_match_the_header(tmp_path):
  names = ["taco_kv_cache", "taco_kv_append_args", "taco_kv_attend_args", "taco_qmat"]
  src = tmp_path / "s.c"
  src.write_text('#include <stdio.h>\n#include "taco.h"\nint main(void) { printf("' + "%zu " * len(names) + '\\n", ' +
                 ", ".join(f"sizeof({n})" for n in names) + "); return 0; }\n")
  subprocess.check_call(["cc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
  sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
  assert sizes == [C.sizeof(t) for t in (abi.TacoKvCache, abi.TacoKvAppendArgs, abi.TacoKvAttendArgs, abi.TacoQmat)]


def test_the_cache_has_no_cpu_path():
  from tacotron_amd.paged import PagedCache
  with pytest.raises(RuntimeError):
    PagedCache(2, 16, 1, 64, device="cpu")


def _qmat(**change):
  return abi.TacoQmat(**{**dict(packed=4096, n_rows=32, n_cols=100, group=64, scale_dtype=abi.TACO_F16), **change})


def test_size_of_a_packed_matrix():
  """Blocks of 16 x 128 codes (1 KiB) for whole multiples of 64 rows, then 64 scales, then 64 zero points per 64 rows and group."""
  L = _lib.lib()
  for n, k, group, dtype, zeros, want in (
    (32, 100, 64, abi.TACO_F16, 0, 4 * 1024 + 2 * 2 * 64), (32, 100, 64, abi.TACO_F16, 1, 4 * 1024 + 2 * 2 * 64 + 2 * 64),
    (1, 1, 32, abi.TACO_F32, 0, 4 * 1024 + 4 * 4 * 64), (65, 129, 128, abi.TACO_BF16, 1, 16 * 1024 + 2 * 4 * 64 + 4 * 64),
    (28672, 8192, 128, abi.TACO_BF16, 0, 28672 * 4096 + 28672 * 64 * 2),
    (1 << 20, 1 << 20, 128, abi.TACO_F32, 0, (1 << 39) + (1 << 35))):
    assert L.taco_qmat_bytes(C.byref(_qmat(n_rows=n, n_cols=k, group=group, scale_dtype=dtype, has_zeros=zeros))) == want


@pytest.mark.parametrize("change,word", [
  (dict(n_rows=0), "rows"), (dict(n_cols=0), "columns"), (dict(n_rows=1 << 29), "rows"), (dict(n_rows=1 << 26), "rows"), (dict(group=16), "group"), (dict(group=0), "group"),
  (dict(scale_dtype=3), "scale_dtype"), (dict(scale_dtype=-1), "scale_dtype")])
def test_bad_matrices_are_refused(change, word):
  L, m = _lib.lib(), _qmat(**change)
  calls = (lambda: L.taco_qmat_pack(C.byref(m), 64, 50, 64, 2, None, 0, 64, None),
           lambda: L.taco_qmat_quantize(C.byref(m), 64, 100, 0, 64, 50, 64, 2, None, 0, None),
           lambda: L.taco_qmat_multiply(C.byref(m), 64, 100, 64, 32, 1, 0, None))
  for call in calls:
    with pytest.raises(_lib.TacoError) as e:
      _lib.check(call())
    assert e.value.code == abi.TACO_EINVAL and word in str(e.value)
  assert L.taco_qmat_bytes(C.byref(m)) == abi.TACO_EINVAL


def test_bad_matrix_calls_are_refused():
  L, m, mz = _lib.lib(), C.byref(_qmat()), C.byref(_qmat(has_zeros=1))
  for rc in (
    L.taco_qmat_bytes(None), L.taco_qmat_pack(None, 64, 50, 64, 2, None, 0, 64, None), L.taco_qmat_pack(m, None, 50, 64, 2, None, 0, 64, None),
    L.taco_qmat_pack(m, 64, 49, 64, 2, None, 0, 64, None), L.taco_qmat_pack(m, 64, 50, 64, 1, None, 0, 64, None),
    L.taco_qmat_pack(m, 64, 50, 64, 2, 64, 2, 64, None), L.taco_qmat_pack(mz, 64, 50, 64, 2, None, 0, 64, None),
    L.taco_qmat_pack(mz, 64, 50, 64, 2, 64, 1, 64, None), L.taco_qmat_pack(m, 64, 50, 64, 2, None, 0, 72, None),
    L.taco_qmat_quantize(m, 64, 99, 0, 64, 50, 64, 2, None, 0, None), L.taco_qmat_quantize(m, 64, 100, 3, 64, 50, 64, 2, None, 0, None),
    L.taco_qmat_quantize(m, None, 100, 0, 64, 50, 64, 2, None, 0, None), L.taco_qmat_quantize(mz, 64, 100, 0, 64, 50, 64, 2, None, 0, None),
    L.taco_qmat_multiply(m, 64, 100, 64, 32, -1, 0, None), L.taco_qmat_multiply(m, 64, 100, 64, 32, 1, 3, None),
    L.taco_qmat_multiply(m, None, 100, 64, 32, 1, 0, None), L.taco_qmat_multiply(m, 64, 100, None, 32, 1, 0, None),
    L.taco_qmat_multiply(m, 66, 100, 64, 32, 1, 0, None), L.taco_qmat_multiply(m, 64, 99, 64, 32, 2, 0, None),
    L.taco_qmat_multiply(m, 64, 100, 64, 31, 2, 0, None), L.taco_qmat_multiply(C.byref(_qmat(packed=None)), 64, 100, 64, 32, 1, 0, None),
    L.taco_qmat_multiply(C.byref(_qmat(packed=4104)), 64, 100, 64, 32, 1, 0, None)):
    assert rc == abi.TACO_EINVAL
  assert L.taco_qmat_multiply(m, 64, 100, 64, 32, 0, 0, None) == 0


def test_matrices_have_no_cpu_path():
  import torch
  from tacotron_amd import w4
  with pytest.raises(RuntimeError):
    w4.quantize(torch.zeros(4, 64))
  with pytest.raises(RuntimeError):
    w4.W4Matrix.from_codes(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2))


def test_rows_of_a_matrix():
  """Rows are read with a stride of a row at least; one row that stands for all is copied."""
  import torch
  from tacotron_amd.w4 import _pitch, _rows
  base = torch.arange(24).view(4, 6)
  for t in (base, base[:, :5], base[::2], base[:1], base[:, :1], base[:1].expand(4, 6), base[:, :1].expand(4, 6), base.t(), base[:, ::2],
            base[0, :1].expand(3, 1), base.as_strided((4, 6), (2, 1)), base[:1].expand(1, 6)):
    rows = _rows(t)
    assert _pitch(rows) >= rows.shape[1]
    assert torch.equal(rows.as_strided(rows.shape, (_pitch(rows), 1)), t)
    assert (rows.shape[0] - 1) * _pitch(rows) + rows.shape[1] <= rows.untyped_storage().nbytes() // 8 - rows.storage_offset()
  assert _rows(base[:, :5]).data_ptr() == base.data_ptr()
