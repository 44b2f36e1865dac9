"""Attention over pages where a row's keys are cut into parts: values that are not finite reach every row that sees them,
however far their scores lie below the best and whatever part they fall into. Finite results are held to the bound of
tests/test_attention_pages_gpu.py (Batch.bound)."""
import math

import numpy as np
import pytest

from tests.test_attention_pages_gpu import Batch, NO_WINDOW
from tests.test_pages_gpu import up  # noqa: F401

pytestmark = pytest.mark.gpu


def far_keys(b, r, n, below, scale):
    """Sets the first n keys of request r, whole pages of them, against its query, their scores at -below, and all others to zero (scores of 0)."""
    q = b.q[r, 0, 0].astype(np.float64)
    b.k[...] = 0
    b.k[b.table[r, :n // b.page]] = (-below / (scale * (q ** 2).sum()) * q).astype(b.k.dtype)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 48, 20])
@pytest.mark.parametrize("below", [20.0, 200.0])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_far_values_that_are_not_finite_reach_the_row(gpu, up, hd, kv, below, bad):  # noqa: F811
    """exp(-200) is 0 in f32: 0 times what is not finite is NaN, in a part of such keys alone as beside the best score. In float64 it is not 0."""
    rng = np.random.default_rng(hd)
    scale = 1 / math.sqrt(hd)
    for n, shared in ((900, 0), (324, 0), (900, 512)):
        sharers = (0, 1) if shared else ()
        b = Batch(rng, 1, 1, hd, 16, [n, n - 1], shared=shared, sharers=sharers, kv=kv)
        far_keys(b, 0, 320, below, scale)
        b.v[b.table[0, 1], 4, 0, 3] = bad
        got, want = b.run(gpu, up, scale), b.want(scale)
        fine = np.isfinite(want)
        assert not fine[0, 0, 0, 3] and fine[0, 0, 0, :3].all() and fine[0, 0, 0, 4:].all() and fine[1].all() == (not shared)
        assert np.array_equal(np.isfinite(got), fine), n
        assert np.abs(got[fine] - want[fine]).max() <= b.bound(scale)[2]


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 40])
def test_parts_without_a_finite_score(gpu, up, hd, kv):  # noqa: F811
    """Scores of -inf weigh their values with 0, which is nothing for finite ones and NaN for others; where a row sees no other
    scores, 0 / 0 is NaN."""
    rng = np.random.default_rng(hd + 1)
    b = Batch(rng, 1, 1, hd, 16, [900], kv=kv)
    b.q[...] = np.abs(b.q) + 0.5
    b.k[b.table[0, :20]] = -np.inf  # the first 320 keys: whole parts of them
    got, want = b.run(gpu, up, 0.1), b.want(0.1)
    assert np.isfinite(want).all() and np.abs(got - want).max() <= b.bound(0.1)[2]
    b.v[b.table[0, 3], 7, 0, 2] = np.inf
    got, want = b.run(gpu, up, 0.1), b.want(0.1)
    fine = np.isfinite(want)
    assert np.flatnonzero(~fine).tolist() == [2]
    assert np.array_equal(np.isfinite(got), fine)
    assert np.abs(got[fine] - want[fine]).max() <= b.bound(0.1)[2]
    b.k[...] = -np.inf
    assert np.isnan(b.want(0.1)).all() and np.isnan(b.run(gpu, up, 0.1)).all()
    b.k[b.table[0, 0], 0] = 0  # the first key alone
    b.v[...] = 1
    assert np.array_equal(b.run(gpu, up, 0.1), np.ones((1, 1, 1, hd), np.float32))
    assert np.isnan(b.run(gpu, up, 0.1, 800)).all()  # a window that hides it
    assert np.array_equal(b.run(gpu, up, 0.1, NO_WINDOW), np.ones((1, 1, 1, hd), np.float32))
