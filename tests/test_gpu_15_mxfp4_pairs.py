"""The tests of the MXFP4 products again, with every product of K up to 1536 on CTA pairs.

By default only large products run there; the kernel has to be right for any."""
import os
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = pathlib.Path(__file__).resolve().parent


@pytest.mark.parametrize("name,which", [
    ("test_gpu_11_mxfp4.py", "grouped_linear or nan_stays or rows_past or offsets or drops"),
    ("test_gpu_12_mxfp4_experts.py", ""),
    ("test_gpu_13_mxfp4_products.py", ""),
    ("test_gpu_14_mxfp4_edges.py", "not 32_bits"),
])
def test_on_cta_pairs(name, which):
    # HMOE_GEMM_KERNEL is read once per process
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-k", which, str(HERE / name)],
                       env=dict(os.environ, HMOE_GEMM_KERNEL="pair"), cwd=HERE.parent, timeout=600,
                       capture_output=True, text=True)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]
