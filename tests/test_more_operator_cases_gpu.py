"""The timed cases of perf/more_operators.py on the framework's buffers: what torch does with a pass's outputs comes after
the pass, without a wait of the caller's. In a process of its own, where torch brings its HIP runtime first."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PASSES = """
import torch
from perf import more_operators as op

op.own = True
for kind in ("draft", "fork", "compact", "attention", "adapters"):
    case = next(c for c in op.listed() if c["kind"] == kind)
    s = op.prepare(case, 3)
    assert torch.cuda.current_stream().cuda_stream == op._compute.stream, "torch works on another stream"
    out = op.run(s)
    leaves = [t for v in out.values() for t in (v if isinstance(v, list) else [v])]
    taken = [t.clone() for t in leaves]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(taken, leaves)), kind
    print(kind, "ok", flush=True)
"""


def test_outputs_are_ordered_with_torch():
    r = subprocess.run([sys.executable, "-u", "-c", PASSES], cwd=ROOT, capture_output=True, text=True, timeout=170)
    assert r.returncode == 0 and r.stdout.count("ok") == 5, (r.returncode, r.stdout, r.stderr[-3000:])
