"""Tree attention where its launches differ: what lies behind the partial outputs of splits, and the kernel that
stages keys in LDS (k_attn_tree_staged) with two and four row groups in a workgroup, windows that hide cached
keys, and rings that wrap. Bounds are those of tests/tree_dense.py.
"""
import math

import numpy as np
import pytest

from tests import tree_dense
from tests.test_tree_gpu import Held, assert_near, random_tree, run_tree, tree_case, up  # noqa: F401
from tests.tree_dense import NO_WINDOW, STAGED
from webgpu_amd.gpu import Compute

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("heads,hd,nodes,start,splits", [(1, 17, 9, 150, 3), (3, 5, 7, 300, 5), (1, 511, 1, 18, 5), (2, 17, 9, 150, 3)])
def test_pairs_behind_an_odd_count_of_partial_outputs(heads, hd, nodes, start, splits, kv):
    """The (max, sum) pairs of the splits are 8-byte values: behind splits * rows * head_dim floats, an odd count in
    all but the last of these, they start one float later, and the scratch has room for it."""
    gpu = Compute().init()  # a context of its own: its scratch is this call's alone
    up = Held(gpu)
    try:
        rng = np.random.default_rng(hd)
        q, k, v, _ = tree_case(rng, heads, 1, hd, nodes, start, NO_WINDOW, 0, kv)
        parents = random_tree(rng, nodes)
        before = gpu.allocated
        got = run_tree(gpu, up, q, k, v, parents, start, 1 / math.sqrt(hd), NO_WINDOW)
        scratch = gpu.allocated - before - sum(b.size for b in up.held)
        rows = nodes * heads
        assert scratch == 4 * ((splits * rows * hd + 1) // 2 * 2 + 2 * splits * rows)
        assert_near(got, q, k, v, parents, start, 1 / math.sqrt(hd), NO_WINDOW)
    finally:
        up.free()
        gpu.dispose()


@pytest.mark.parametrize("case", STAGED, ids=lambda c: "-".join("w" if v == NO_WINDOW else str(v) for v in c))
def test_staged_keys(gpu, up, case):  # noqa: F811
    start, window = case[4:6]
    q, k, v, parents, sees, first, scale = tree_dense.inputs(case, case[3] // 8)
    want, S = tree_dense.attention(q, k, v, sees, first, scale)
    got = run_tree(gpu, up, q, k, v, parents, start, scale, window, tail=5)
    keys, most = sees.shape[1], float(np.abs(v).max())
    assert tree_dense.within(got, want, S, keys, most), (np.abs(got - want).max(), np.linalg.norm(got - want), tree_dense.bounds(want, S, keys, most))
    assert np.all(got[~sees.any(1)] == 0)


# heads, kv_heads, head_dim, nodes, start, window, slots to spare: staged with two row groups, with four, in a window
REDONE = [(7, 1, 128, 64, 3000, NO_WINDOW, 4), (16, 1, 64, 70, 2000, NO_WINDOW, 4), (8, 1, 256, 33, 2500, NO_WINDOW, 4),
          (8, 1, 128, 64, 9001, 2500, 27), (4, 1, 128, 64, 20011, 8200, 3), (4, 1, 256, 32, 6000, 2100, 27)]


@pytest.mark.parametrize("case", REDONE, ids=lambda c: "-".join("w" if v == NO_WINDOW else str(v) for v in c))
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_formed_again_hold_the_formula(gpu, up, case, bad):  # noqa: F811
    """A node's K and V that are not finite: the nodes that do not see it keep the values that the formula gives
    (tests/test_tree_dense.py shows what the bounds tell apart)."""
    start, window, nodes = case[4], case[5], case[3]
    q, k, v, parents, sees, first, scale = tree_dense.inputs(case, 0)
    want, S = tree_dense.attention(q, k, v, sees, first, scale)
    most, keys, hit = float(np.abs(v).max()), sees.shape[1], nodes // 2
    hits = [(start + hit, sees[:, hit - nodes])]
    if window != NO_WINDOW:
        hits.append((first, sees[:, 0]))  # the cached key that only nodes of depth 0 see
    for t, seen in hits:
        free = np.flatnonzero(~seen)
        assert 0 < len(free) < nodes
        k1, v1 = k.copy(), v.copy()
        k1[t % len(k)], v1[t % len(k)] = bad, bad
        unused = [(start + nodes + e) % len(k) for e in range(case[6])]
        k1[unused], v1[unused] = bad, bad
        got = run_tree(gpu, up, q, k1, v1, parents, start, scale, window)
        assert tree_dense.within(got[free], want[free], S, keys, most), (np.abs(got - want)[free].max(), tree_dense.bounds(want[free], S, keys, most))
        assert not np.isfinite(got[seen]).any()


# ------------------------------------------------------------------------------- what f16 rings round
#
# Over f16 rings, head dims that are multiples of 8 up to 256, a query is held as two f16: off by 2^-22 of itself and 2^-39
# of the row's largest |q|, Q. So are the weights, by 2^-22 of themselves and 2^-36 of the largest; their sum has them
# in f32. With e = 2^-24 a score (2 hd products of f16 added in f32) is off by
#   d = scale ((2^-22 + (2 hd + 8) e) sum|q k| + 2^-39 Q sum|k|) + e (|s| + 32),
# a weight by r = 2 d + 2^-21 of itself, sums of n terms by n e, and an output by
#   (sum w |v| (r + n e) + 2^-36 sum|v|) / sum w + |y| (r + n e).
# f32 rings: without the terms of 2^-39 and 2^-36.

def rounding(q, k, v, scale, half):
    """Exact outputs of one query and their bounds: q [hd], k and v [n][hd]."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    n, hd, e = len(k), len(q), 2.0 ** -24
    s = k @ q * scale
    w = np.exp(s - s.max())
    d = scale * ((2.0 ** -22 + (2 * hd + 8) * e) * (np.abs(k) @ np.abs(q)).max() + (2.0 ** -39 * np.abs(q).max() * np.abs(k).sum(1).max() if half else 0))
    r = 2 * (d + e * (np.abs(s).max() + 32)) + 2.0 ** -21
    y = w @ v / w.sum()
    grid = 2.0 ** -36 * np.abs(v).sum(0) if half else 0
    return y, (w @ np.abs(v) * (r + n * e) + grid) / w.sum() + np.abs(y) * (r + n * e)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd,heads,start", [(64, 1, 900), (128, 1, 900), (256, 1, 900), (72, 1, 900), (64, 64, 8500), (128, 64, 8500), (256, 64, 8500)])
@pytest.mark.parametrize("faint", [-12.0, -18.3, -25.4, -31.7, -40.2])
def test_faint_weights(gpu, up, hd, heads, start, faint, kv):  # noqa: F811
    """A first key that takes nearly all the weight and whose value is 0, beside keys of weight 2^faint."""
    half = kv == "f16"
    q = np.zeros((1, heads, hd), np.float32)
    q[..., 0] = 1
    k, v = np.zeros((start + 1, 1, hd), np.float32), np.ones((start + 1, 1, hd), np.float32)
    k[0, 0, 0], v[0] = 16, 0
    v[1:] += 0.25 * (np.arange(hd) % 3)
    dtype = np.float16 if half else np.float32
    k, v, scale = k.astype(dtype), v.astype(dtype), -faint * math.log(2) / 16
    want, bound = rounding(q[0, 0], k[:, 0], v[:, 0], scale, half)
    got = run_tree(gpu, up, q, k, v, np.array([-1], np.int32), start, scale, NO_WINDOW)
    assert np.all(np.abs(got[0] - want) <= bound), (np.abs(got[0] - want).max() / want.max(), (bound / want).max())


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd,heads,start", [(64, 1, 900), (128, 1, 900), (256, 1, 900), (72, 1, 900), (64, 64, 8500), (128, 64, 8500), (256, 64, 8500)])
@pytest.mark.parametrize("largest", [2.0 ** 12, 2.0 ** 18, 2.0 ** 24])
def test_queries_with_one_large_entry(gpu, up, hd, heads, start, largest, kv):  # noqa: F811
    """Where the keys are 0: the scores come from the small entries."""
    half = kv == "f16"
    rng = np.random.default_rng(hd)
    q = rng.standard_normal((1, heads, hd)).astype(np.float32)
    q[..., 3] = largest
    k, v = (rng.standard_normal((start + 1, 1, hd)).astype(np.float16 if half else np.float32) for _ in range(2))
    k[..., 3] = 0
    got = run_tree(gpu, up, q, k, v, np.array([-1], np.int32), start, 1 / math.sqrt(hd), NO_WINDOW)
    for h in range(heads):
        want, bound = rounding(q[0, h], k[:, 0], v[:, 0], 1 / math.sqrt(hd), half)
        assert np.all(np.abs(got[0, h] - want) <= bound), (h, np.abs(got[0, h] - want).max(), bound.max())
