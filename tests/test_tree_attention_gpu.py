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
