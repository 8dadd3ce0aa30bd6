"""CPU: what the affine layer norm, the head's cross entropy and distillation
refuse.  Every check comes before any device work, so the handles wrap addresses
that nothing reads; a refusal prints "malus: ..." and aborts the process."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
HEAD = """
import numpy as np, malus_b200 as M
lib = M.load()
f = lambda *s: M.Tensor.wrap(1 << 20, s, np.float32)
i = lambda *s: M.Tensor.wrap(1 << 20, s, np.int32)
"""
CASES = [
    ("M.layernorm_affine(i(4, 8))", "expects an f32 tensor"),
    ("M.layernorm_affine(f(4, 0))", "empty last axis"),
    ("M.layernorm_affine(f(4, 8), f(9))", "weight must have shape [8]"),
    ("M.layernorm_affine(f(4, 8), f(8), f(1, 8))", "bias must have shape [8]"),
    ("M.layernorm_affine(f(4, 8), i(8))", "weight must be f32"),
    ("M.layernorm_affine(f(4, 8), eps=-1.0)", "eps must not be negative"),
    ("M.layernorm_affine(f(4, 8), eps=float('nan'))", "eps must not be negative"),
    ("M.layernorm_affine_bwd(f(4, 8), None, f(3, 2), f(4, 8))", "stats must be the [4, 2]"),
    ("M.layernorm_affine_bwd(f(4, 8), None, f(4, 2), f(8, 4))", "x's shape"),
    ("M.distill(f(4, 8), f(4, 2), f(4, 2))", "ids must be Tensor<i32>"),
    ("M.distill(f(4, 8), i(4, 2), i(4, 2))", "must be f32"),
    ("M.distill(f(4, 8, 1), i(4, 2), f(4, 2))", "rank-2 [N, V]"),
    ("M.distill(f(4, 8), i(3, 2), f(3, 2))", "ids must be rank-2 [4, K]"),
    ("M.distill(f(4, 8), i(4, 2), f(4, 3))", "the same shape"),
    ("M.distill(f(4, 8), i(4, 0), f(4, 0))", "1 to 1024 teacher entries"),
    ("M.distill(f(4, 8), i(4, 1025), f(4, 1025))", "1 to 1024 teacher entries"),
    ("M.distill(f(4, 0), i(4, 2), f(4, 2))", "empty vocabulary"),
    ("M.distill(f(1, (1 << 24) + 1), i(1, 2), f(1, 2))", "limited to 16777216"),
    ("M.distill(f(4, 8), i(4, 2), f(4, 2), 0.0)", "temperature must be positive"),
    ("M.distill(f(4, 8), i(4, 2), f(4, 2), float('inf'))", "temperature must be positive"),
    ("M.linear_xent(f(4, 8), f(9, 8), f(4))", "targets must be Tensor<i32>"),
    ("M.linear_xent(f(4, 8), f(9, 7), i(4))", "does not match x's last axis 8"),
    ("M.linear_xent(f(4, 8), f(9, 8), i(4), tied=False)", "does not match x's last axis 8"),
    ("M.linear_xent(f(4, 8), f(9, 8, 1), i(4))", "weight must be rank-2"),
    ("M.linear_xent(f(4, 8), f(9, 8), i(5))", "4 rows but targets has 5"),
    ("M.linear_xent(f(4, 8), f(0, 8), i(4))", "empty axis"),
    ("M.linear_xent(f(4, 0), f(9, 0), i(4))", "empty axis"),
    ("M.linear_xent(f(4, 8), f((1 << 24) + 1, 8), i(4))", "limited to 16777216"),
    ("M.linear_xent(i(4, 8), f(9, 8), i(4))", "expects f32"),
    ("a, b, c = f(4), f(5), f(1); lib.tape_record_loss((M.C.c_int64 * 1)(a.h), (M.C.c_int64 * 1)(b.h), 1, c.h)",
     "its input's shape"),
    ("a, b, c = f(4), f(4), f(2); lib.tape_record_loss((M.C.c_int64 * 1)(a.h), (M.C.c_int64 * 1)(b.h), 1, c.h)",
     "not 1"),
]


@pytest.mark.parametrize("call,says", CASES)
def test_refused(call, says):
    r = subprocess.run([sys.executable, "-c", HEAD + call + "\nprint('not refused')"], cwd=ROOT, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode != 0 and "not refused" not in r.stdout
    assert "malus: " in r.stderr and says in r.stderr, r.stderr[-500:]
    assert "CUDA" not in r.stderr
