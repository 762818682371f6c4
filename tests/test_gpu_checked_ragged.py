"""The tests of masked attention and of the 8-bit cache once more against the checked build of the library: their stores'
indices too are tested there against their tensors' extents."""

import os
import subprocess
import sys

import pytest

from tests.test_gpu_checked_build import CHECKED, ROOT

pytestmark = pytest.mark.gpu

FILES = ["tests/test_gpu_masked_attention.py", "tests/test_gpu_kv_cache.py", "tests/test_gpu_ragged_edges.py"]


def test_ragged_operators_with_index_checks():
    if not os.path.exists(CHECKED):
        pytest.skip("checked library not built (python -m nano_omni_b200.build --checked)")
    if os.environ.get("NOB200_LIBRARY"):
        pytest.skip("already running against another build of the library")
    run = subprocess.run(
        [sys.executable, "-m", "pytest", *FILES, "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider"],
        cwd=ROOT, env=dict(os.environ, NOB200_LIBRARY=CHECKED), capture_output=True, text=True, timeout=1500,
    )  # fmt: skip
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]
