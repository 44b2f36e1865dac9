"""Tree attention where its launches differ: what lies behind the partial outputs of splits."""
import math

import numpy as np
import pytest

from tests.test_tree_gpu import NO_WINDOW, Held, assert_near, random_tree, run_tree, tree_case
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
