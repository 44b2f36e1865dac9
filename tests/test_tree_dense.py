"""The dense float64 form of tree attention against the one that goes node by node, and what its bounds tell
apart: mistakes are planted in the mask of the float64 form."""
import numpy as np
import pytest

from tests import tree_dense, tree_ref
from tests.tree_dense import NO_WINDOW, STAGED


@pytest.mark.parametrize("window", [NO_WINDOW, 9, 1])
def test_the_dense_form_is_the_reference(window):
    q, k, v, parents, sees, first, scale = tree_dense.inputs((6, 2, 8, 20, 31, window, 3), 3)
    want = tree_ref.attention(q, k, v, parents, 31, scale, window)
    assert np.abs(tree_dense.attention(q, k, v, sees, first, scale)[0] - want).max() < 1e-13
    assert sum(p is None for p in tree_ref.paths(parents)) == (~sees.any(1)).sum() >= 3


def mistakes(sees, nodes, window):
    """Masks that are wrong in one way each."""
    base = sees.shape[1] - nodes
    own, real = np.eye(nodes, dtype=bool), sees.any(1)
    if window != NO_WINDOW:
        wrong = sees.copy()
        wrong[np.arange(nodes), np.maximum(sees.argmax(1) - 1, 0)] |= real
        yield "a key too many at the window's end", wrong
    for name, tree in (("nodes do not see themselves", sees[:, base:] & ~own), ("no node but itself", own & real[:, None]),
                       ("all nodes see each other", np.repeat(real[:, None], nodes, 1) & real), ("causal among the nodes", np.tril(np.ones_like(own)) & real[:, None])):
        yield name, np.concatenate([sees[:, :base], tree], 1)
    wrong = sees.copy()
    wrong[:, 32:64] = False
    yield "a block of keys lost", wrong


@pytest.mark.parametrize("case", [c for c in STAGED if c[1] == 1] + [(7, 1, 128, 64, 3000, NO_WINDOW, 4), (8, 1, 256, 33, 2500, NO_WINDOW, 4)], ids=lambda c: "-".join("w" if v == NO_WINDOW else str(v) for v in c))
def test_the_bounds_tell_wrong_masks_apart(case):
    q, k, v, parents, sees, first, scale = tree_dense.inputs(case, case[3] // 8)
    want, S = tree_dense.attention(q, k, v, sees, first, scale)
    most = float(np.abs(v).max())
    assert tree_dense.within(want.astype(np.float32), want, S, sees.shape[1], most)
    for name, wrong in mistakes(sees, case[3], case[5]):
        assert not tree_dense.within(tree_dense.attention(q, k, v, wrong, first, scale)[0], want, S, sees.shape[1], most), name
