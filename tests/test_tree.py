"""What the repository holds."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT


def test_no_compiled_code_is_under_version_control():
  if not os.path.exists(os.path.join(ROOT, ".git")) or not shutil.which("git"):
    pytest.skip("not a checkout")
  built = []
  for name in subprocess.check_output(["git", "-c", "safe.directory=*", "-C", ROOT, "ls-files", "-z"], text=True).split("\0"):
    path = os.path.join(ROOT, name)
    if name and os.path.isfile(path):
      with open(path, "rb") as f:
        head = f.read(24)
      if head[:4] == b"\x7fELF" or head == b"__CLANG_OFFLOAD_BUNDLE__" or head[:8] == b"!<arch>\n" or ".o." in name or name.endswith((".o", ".so", ".a")):
        built.append(name)
  assert not built
