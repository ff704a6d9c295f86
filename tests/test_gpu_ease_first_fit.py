"""The first EASE fit of a process, at a size whose last inverse panel is short: the diagonal-block chains of the panels before it are still running
when its own begins (kernels of a first call are loaded as they are launched, which makes that certain)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import numpy as np
from recpack_amd import _lib, get_context
from recpack_amd.synth import powerlaw_csr

n = int(__import__("sys").argv[1])
X = powerlaw_csr(40000, n, 0.004, seed=7).to_scipy()
ctx = get_context(0)
dX = _lib.DeviceCSR.from_host(ctx, X.indptr, X.indices, X.shape)
B = _lib.ease_fit(ctx, dX, 50.0, 0.0).dense_download()
# A (I - B) is diagonal, A = X^T X + 50 I: both probes give its diagonal (1e-4 relative: the bar of the full-size probes)
v = []
for seed in (1, 2):
    z = np.random.default_rng(seed).choice([-1.0, 1.0], n) * np.random.default_rng(seed + 9).uniform(0.5, 1.5, n)
    y = z - B.astype(np.float64) @ z
    v.append((X.T @ (X @ y) + 50.0 * y) / z)
print("error", float(np.abs(v[0] / v[1] - 1).max()))
"""


@pytest.mark.parametrize("n", [8960, 9000, 8300])
def test_first_fit_of_a_process(n):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", CHILD, str(n)], cwd=root, capture_output=True, text=True, timeout=110)
    assert out.returncode == 0, out.stderr[-2000:]
    assert float(out.stdout.split()[-1]) <= 1e-4
