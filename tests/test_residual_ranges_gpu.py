"""The residual path's kernels where the choice of a launch, a sum or an
address depends on the size: the first call of a process, rows far from zero,
rows too wide for the rings, strided batches of many rows, and tensors of
different types.  The operators in 64 bits and most bounds are
residual_reference.py's; a tighter one of the norms' backward is derived here."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import mhc_proj
import residual_reference as ref
from test_residual_gpu import DTYPES, EPS, affine_of, gen, leaf, mixing, normal, offset_copy, rows, same_bits, streams

pytestmark = pytest.mark.gpu
f = mhc_proj.torch
HERE = os.path.dirname(os.path.abspath(__file__))


# ---- the first call of a process -----------------------------------------------------

# (type, width, offset of X): rows of single elements whose stages need between 28
# and 32 KB of dynamic shared memory beside the four streams' 20 KB of static
FIRST = [("float32", C, 0) for C in (41, 42, 43)] + [("float32", 44, 1)] \
    + [("bfloat16", C, 0) for C in range(81, 88)] + [("bfloat16", 88, 1), ("float16", 81, 0), ("float16", 88, 1)]

FIRST_CALL = """
import sys
import torch, mhc_proj
import residual_reference as ref
from test_residual_gpu import gen, normal, offset_copy, streams
dtype, C, offset = getattr(torch, sys.argv[1]), int(sys.argv[2]), int(sys.argv[3])
g = gen(C)
X, G, h = streams(9, C, g, dtype), normal(g, 9, C).to(dtype), torch.sigmoid(normal(g, 9, 4))
w, b = 1 + 0.3 * normal(g, C), 0.3 * normal(g, C)
mean, rstd = normal(g, 9), 0.5 + torch.rand(9, device="cuda", generator=g)
X = offset_copy(X, offset, 0)
out = mhc_proj.torch.stream_norm_n4_backward(G, X, h, mean, rstd, w, b)
ref.check(out, ref.stream_norm_backward(G, X, h, mean, rstd, w, b))
print("ok")
"""


def first_call(case):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([HERE, os.path.join(os.path.dirname(HERE), "mhc-proj_b200")]))
    run = subprocess.run([sys.executable, "-c", FIRST_CALL, *map(str, case)], env=env, cwd=HERE, capture_output=True,
                         text=True, timeout=300)
    return run.stdout.strip() if run.returncode == 0 else run.stderr[-600:]


def test_a_process_may_begin_with_any_width():
    """A kernel's limit of dynamic shared memory, once raised, stays for the
    process, so a call that forgets to raise it fails only where no wider one
    came before it: each case is a process's first call."""
    with ThreadPoolExecutor(4) as pool:
        got = dict(zip(FIRST, pool.map(first_call, FIRST)))
    assert {k: v for k, v in got.items() if v != "ok"} == {}
