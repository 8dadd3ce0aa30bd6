"""Distillation's temperature: refused (CPU) where its square or its inverse leaves the
floats, and the formula (GPU) at extremes that do not."""
import subprocess
import sys

import numpy as np
import pytest

from test_gpu_distill import check, inputs, reference, run
from test_head_refusals import HEAD, ROOT


@pytest.mark.parametrize("T", ["1e-39", "1e-30", "1e-19", "1e19", "1e20", "3e38"])
def test_refused(T):
    r = subprocess.run([sys.executable, "-c", HEAD + f"M.distill(f(4, 8), i(4, 2), f(4, 2), {T})\nprint('not refused')"],
                       cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode != 0 and "not refused" not in r.stdout
    assert "malus: " in r.stderr and "between 2^-60 and 2^60" in r.stderr, r.stderr[-500:]


@pytest.mark.gpu
@pytest.mark.parametrize("V", [100, 3001])
@pytest.mark.parametrize("T", [2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60])
def test_extremes(M, T, V):
    s, ids, te = inputs(5, V, 6, V)
    got = run(M, s, ids, te, T)
    assert all(np.isfinite(a).all() for a in got)
    check(got, *reference(s, ids, te, T))
