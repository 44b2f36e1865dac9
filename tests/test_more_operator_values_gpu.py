"""The timed cases of perf/more_operators.py, every listed one and some drawn ones: what the framework's operators write, held to the
plain forms (whole numbers, pools of pages: equal) and to float64 (attention, adapters). In a process of its own, where torch brings
its HIP runtime first.

Tolerances, e = 2^-24: attention (2 (hd + 4 + 4) e S + 2 (n + 8 + 4) e + n 2^-36) max|v| with S = scale max|q| max|k| for n keys, as in
tests/test_attention_pages_gpu.py and with room for operands in two f16 (4 e each, and 2^-36 of the largest weight); adapters (cols +
rank + 12) e of the sum of magnitudes and e of the result, as in tests/test_adapters_gpu.py. The 2-norms of the differences are held to 16 e
sqrt(hd + n) max(1, sqrt(S)) and 16 e sqrt(cols + rank) of those of the results (adapters: of the magnitudes' root sums of squares).
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PASSES = """
import math, random, sys
import torch
from perf import more_operators as op

E = 2.0 ** -24
kind, draws = sys.argv[1], int(sys.argv[2])
cases = [c for c in op.listed() if c["kind"] == kind]
rng = random.Random(kind)
while draws:
    c = op.draw(rng)
    if c["kind"] == kind:
        cases.append(dict(c, name="drawn"))
        draws -= 1


def flat(out):
    return {n + str(i): t for n, v in out.items() for i, t in enumerate(v if isinstance(v, list) else [v])}


def attention(case, s, got, want):
    n, hd = int(s["lengths"].max()), case["head_dim"]
    S = op._full(case)["scale"] * float((s["q"].double() ** 2).sum(-1).max() * (s["k"].double() ** 2).sum(-1).max()) ** 0.5
    bound = (2 * (hd + 8) * E * S + 2 * (n + 12) * E + n * 2.0 ** -36) * float(s["v"].abs().max())
    off = got.double() - want
    assert float(off.abs().max()) <= bound, (float(off.abs().max()), bound)
    assert float(off.norm()) <= 16 * E * math.sqrt(hd + n) * max(1, math.sqrt(S)) * float(want.norm()), (float(off.norm()), float(want.norm()))


def adapters(case, s, got, want):
    size, root = torch.zeros_like(want), 0.0
    for w in range(case["adapters"]):
        at = torch.nonzero(s["which"] == w)[:, 0]
        x, a, b, f = s["x"][at].double(), s["a"][w].double(), s["b"][w].double(), float(s["scales"][w])
        size[at] = f * ((x.abs() @ a.abs().t()) @ b.abs().t())
        root += float((f * f * ((x ** 2 @ a.t() ** 2) @ b.t() ** 2)).sum())
    n, off, on = case["cols"] + case["rank"], (got.double() - want).abs(), s["which"] >= 0
    assert bool((off <= (n + 12) * E * size + E * want.abs()).all())
    assert float(off[on].norm()) <= 16 * E * math.sqrt(n) * (math.sqrt(root) + float(want[on].norm()))
    assert torch.equal(got[~on], s["y"][~on])


for seed, case in enumerate(cases):
    print(case, flush=True)
    op.own = False
    given = op._INPUTS[kind](case, seed)
    plain = op.prepare(case, seed)
    op.run(plain)
    want = flat(op.run(plain))
    op.own = True
    own = op.prepare(case, seed)
    op.run(own)
    got = flat(op.run(own))  # a second pass: from the state that the first left, as the plain form's
    torch.cuda.synchronize()
    assert got.keys() == want.keys()
    if kind in ("attention", "adapters"):
        assert got.keys() == {"y0"}
        if kind == "adapters":
            own = op.prepare(case, seed)
            got = flat(op.run(own))
        torch.cuda.synchronize()
        op.own = False
        exact = op.exact(case, seed)["y"]
        globals()[kind](case, given, got["y0"], exact)
    else:
        for name in want:
            assert got[name].dtype == want[name].dtype and torch.equal(got[name], want[name]), name
    del plain, own, got, want, given
    print("ok", flush=True)
print("all", len(cases), flush=True)
"""


@pytest.mark.parametrize("kind,listed,draws", [("draft", 2, 6), ("fork", 2, 6), ("compact", 2, 6), ("attention", 3, 8), ("adapters", 3, 6)])
def test_timed_cases_hold(kind, listed, draws):
    r = subprocess.run([sys.executable, "-u", "-c", PASSES, kind, str(draws)], cwd=ROOT, capture_output=True, text=True, timeout=170)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("all %d" % (listed + draws)), (r.returncode, r.stdout[-2000:], r.stderr[-3000:])
