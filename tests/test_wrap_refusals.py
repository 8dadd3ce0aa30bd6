"""CPU: memory that cannot be a tensor's is refused when it is wrapped, before a kernel
could read it.  Nothing reads the addresses; a refusal prints "malus: ..." and aborts
the process."""
import subprocess
import sys

import pytest

from test_head_refusals import HEAD, ROOT

CASES = [
    ("M.Tensor.wrap((1 << 20) + 2, (4,), np.float32)", "not aligned"),
    ("M.Tensor.wrap((1 << 20) + 1, (4,), np.int32)", "not aligned"),
    ("M.Tensor.wrap((1 << 20) + 4, (4,), np.int64)", "not aligned"),
    ("M.Tensor.wrap(1 << 20, (1,) * 9)", "rank 9 exceeds"),
    ("M.Tensor.wrap(1 << 20, (1,) * 70)", "rank 70 exceeds"),
    ("lib.malus_tensor_wrap(1, 1 << 20, (M.C.c_size_t * 1)(4), 1)", "unsupported dtype"),
    ("lib.malus_tensor_wrap_shared(0, (1 << 20) + 3, (M.C.c_size_t * 1)(4), 1)", "not aligned"),
]


@pytest.mark.parametrize("call,says", CASES)
def test_refused(call, says):
    r = subprocess.run([sys.executable, "-c", HEAD + call + "\nprint('not refused')"], cwd=ROOT, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode != 0 and "not refused" not in r.stdout
    assert "malus: " in r.stderr and says in r.stderr, r.stderr[-500:]


def test_taken():
    r = subprocess.run([sys.executable, "-c", HEAD + "M.Tensor.wrap((1 << 20) + 4, (2, 0, 1, 1, 1, 1, 1, 1)); "
                        "M.Tensor.wrap(0, (0,), np.int64); M.Tensor.wrap((1 << 20) + 8, (), np.int64); print('ok')"],
                       cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-500:]
