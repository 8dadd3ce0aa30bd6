"""CPU: what the tape's records of a model's last part refuse.  The handles wrap
addresses that nothing reads; a refusal prints "malus: ..." and aborts the process."""
import subprocess
import sys

import pytest

from test_head_refusals import HEAD, ROOT

CASES = [
    ("x, y = f(4, 8), f(4, 8); lib.tape_record_layernorm_affine(x.h, 0, 0, y.h, 0)", "needs the forward pass's stats"),
    ("x, y, s = f(4, 8), f(8, 4), f(4, 2); lib.tape_record_layernorm_affine(x.h, 0, 0, y.h, s.h)", "not x's shape"),
]


@pytest.mark.parametrize("call,says", CASES)
def test_refused(call, says):
    r = subprocess.run([sys.executable, "-c", HEAD + call + "\nprint('not refused')"], cwd=ROOT, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode != 0 and "not refused" not in r.stdout
    assert "malus: " in r.stderr and says in r.stderr, r.stderr[-500:]


def test_a_paused_tape_takes_no_stats():
    r = subprocess.run([sys.executable, "-c", HEAD + "x, y = f(4, 8), f(4, 8); lib.tape_pause()\n"
                        "lib.tape_record_layernorm_affine(x.h, 0, 0, y.h, 0); print('ok')"], cwd=ROOT, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-500:]
