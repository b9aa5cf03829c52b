"""Vectors that are not finite, many vectors, rows at any address and states beside one another, once more under the checked build
(tests/test_gpu_checked_decoding.py has the other suites of these operators)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHECKED = os.environ.get("VSK_CHECKED", "0") not in ("", "0")
SUITES = ["tests/test_gpu_int4_vectors.py", "tests/test_gpu_beam_rows.py",
          "tests/test_gpu_beam_states.py", "tests/test_gpu_int4_sizes.py"]


@pytest.mark.skipif(CHECKED, reason="this is the child process")
def test_suites_under_the_checked_build():
    assert os.path.exists(os.path.join(ROOT, "vectorstorekit_b200", "libvsk_cuda_checked.so")), "python -m vectorstorekit_b200.build --checked"
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider"] + SUITES, cwd=ROOT,
                       env=dict(os.environ, VSK_CHECKED="1"), capture_output=True, text=True, timeout=1200)
    assert r.returncode == 0 and " passed" in r.stdout, "\n".join(r.stdout.strip().splitlines()[-25:]) + r.stderr[-2000:]
