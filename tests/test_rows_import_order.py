"""torch ships a HIP runtime of its own: an order of imports that loads two of them is refused, whichever way it came about."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytest.importorskip("torch")


def _run(code):
  return subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("code", [
    "from cuhnsw_amd import CuHNSW\nfrom cuhnsw_amd import rows",
    "from cuhnsw_amd import CuHNSW\nimport torch\nfrom cuhnsw_amd import rows",
    "from cuhnsw_amd import CuHNSW\nh = CuHNSW({'py_log_level': 1})\nimport torch\nh.pack_rows()",
    "from cuhnsw_amd import capi\ncapi.load()\nfrom cuhnsw_amd import rows",
    "from cuhnsw_amd import capi\ncapi.load()\nimport torch\nfrom cuhnsw_amd import rows",
])
def test_torch_after_the_native_library_is_refused(code):
  r = _run(code)
  assert r.returncode != 0 and "ImportError" in r.stderr and "import torch before cuhnsw_amd" in r.stderr


@pytest.mark.parametrize("code", [
    "import torch\nfrom cuhnsw_amd import CuHNSW, rows",
    "from cuhnsw_amd import rows\nfrom cuhnsw_amd import CuHNSW",
    "from cuhnsw_amd import datasets\nimport torch\nfrom cuhnsw_amd import capi, rows\ncapi.load()",
])
def test_torch_first_is_not(code):
  r = _run(code + "\nassert rows._one_hip_runtime()")
  assert r.returncode == 0, r.stderr
