"""Tree attention whose keys are cut into splits: values that are not finite reach the rows that see them, also from a split
whose scores all lie far below the best."""
import math

import numpy as np
import pytest

from tests import tree_ref
from tests.test_tree_gpu import run_tree, up  # noqa: F401

pytestmark = pytest.mark.gpu
NO_WINDOW = 1 << 30


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 48, 20])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_far_values_that_are_not_finite_reach_the_rows(gpu, up, hd, kv, bad):  # noqa: F811
    """Keys of scores of -200 and -inf below others of 0: 0 times what is not finite is NaN. Node 2 does not see nodes 0 and 1, whose
    values are; the first of the far keys, seen by all, and finite ones leave nothing."""
    rng = np.random.default_rng(hd)
    start, far, nodes, scale = 6000, 3000, 3, 1 / math.sqrt(hd)
    kind = np.float16 if kv == "f16" else np.float32
    q = np.repeat(np.abs(rng.standard_normal((1, 1, hd))) + 0.5, nodes, 0).astype(np.float32)
    v = rng.standard_normal((start + nodes, 1, hd)).astype(kind)
    x = q[0, 0].astype(np.float64)
    for below in (-200 / (scale * (x ** 2).sum()) * x, -np.inf):
        k = np.zeros((start + nodes, 1, hd), kind)
        k[:far, 0] = np.asarray(below).astype(kind)
        parents = np.array([-1, 0, -1], np.int32)
        clean = run_tree(gpu, up, q, k, v, parents, start, scale, NO_WINDOW)
        # equal weights of 3001 or 3002 keys: tests/test_tree_gpu.py's bound with scores of 0, and of at most 200 that add nothing
        room = 2 * (far + nodes + 8) * 2.0 ** -24 * float(np.abs(v).max())
        assert np.abs(clean - tree_ref.attention(q, k, v, parents, start, scale, NO_WINDOW)).max() <= room
        kept, v[20, 0, 3] = v[20, 0, 3], bad
        v[start + 1, 0, 5] = bad  # a node's own
        got, want = (f(*a, parents, start, scale, NO_WINDOW) for f, a in ((lambda *b: run_tree(gpu, up, *b), (q, k, v)), (tree_ref.attention, (q, k, v))))
        fine = np.isfinite(want)
        assert np.flatnonzero(~fine[0, 0]).tolist() == [3] and np.flatnonzero(~fine[1, 0]).tolist() == [3, 5] and np.flatnonzero(~fine[2, 0]).tolist() == [3]
        assert np.array_equal(np.isfinite(got), fine)
        assert np.abs(got[fine] - want[fine]).max() <= room
        v[20, 0, 3], v[start + 1, 0, 5] = kept, 0
