"""Host parts of the drafted-tree operators: the frequency factors, and the plain float64 forms that
the GPU tests compare with, checked against independent formulations."""
import math

import numpy as np
import pytest

from tests import tree_ref
from webgpu_amd.rope import llama3_factors, yarn_factors


def test_llama3_factors_keep_fast_pairs_and_slow_the_others():
    theta, rot, original = 5e5, 128, 8192
    f = llama3_factors(rot, theta, 8.0, 1.0, 4.0, original)
    assert f.dtype == np.float32 and f.shape == (64,)
    for j in range(64):
        wave = 2 * math.pi * theta ** (2 * j / rot)
        if wave < original / 4:
            want = 1.0
        elif wave > original:
            want = 8.0
        else:
            s = (original / wave - 1) / 3
            want = 1 / ((1 - s) / 8 + s)
        assert abs(f[j] - want) <= 2 ** -23 * want, j
    assert f[0] == 1 and f[-1] == 8


def test_yarn_factors_ramp_between_the_two_pairs():
    f, m = yarn_factors(128, 1e4, 4.0, 4096)
    assert m == 0.1 * math.log(4) + 1
    assert f[0] == 1 and f[-1] == 4 and np.all(np.diff(f) >= 0)
    # the pair that turns 32 times in the original context is still whole, the one that turns once is not
    turns = 4096 / (2 * math.pi * 1e4 ** (np.arange(64) / 64))
    assert f[np.searchsorted(-turns, -32) - 1] == 1 and f[np.searchsorted(-turns, -1) + 1] == 4
    ones, m = yarn_factors(64, 1e6, 1.0, 8192)
    assert m == 1 and np.all(ones == 1)


@pytest.mark.parametrize("call", [lambda: llama3_factors(127, 1e4, 8, 1, 4, 8192), lambda: llama3_factors(128, 1e4, 8, 4, 1, 8192),
                                  lambda: llama3_factors(128, 1e4, 0, 1, 4, 8192), lambda: yarn_factors(128, 1e4, 0.5, 4096),
                                  lambda: yarn_factors(0, 1e4, 2, 4096), lambda: yarn_factors(128, 1e4, 2, 0)])
def test_factors_refuse_what_has_no_meaning(call):
    with pytest.raises(ValueError):
        call()


def test_reference_tree_attention_of_a_chain_is_causal_attention():
    from oracle import orc
    rng = np.random.default_rng(3)
    n, heads, kvh, hd, start, window, cap = 5, 4, 2, 8, 11, 7, 12
    q, k, v = (rng.standard_normal(s) for s in ((n, heads, hd), (cap, kvh, hd), (cap, kvh, hd)))
    got = tree_ref.attention(q, k, v, list(range(-1, n - 1)), start, 0.3, window)
    want = orc.attention(q.astype(np.float32).ravel(), k.astype(np.float32).ravel(), v.astype(np.float32).ravel(), heads, kvh, hd,
                         start, 0.3, window, cap, n)
    assert np.abs(got.ravel() - want).max() < 1e-5


def test_reference_draws_follow_the_oracle_of_the_single_row():
    from oracle import orc
    rng = np.random.default_rng(4)
    for i in range(60):
        l = np.round(rng.standard_normal(80) * 3, 1).astype(np.float32)
        l[rng.integers(0, 80, 5)] = rng.choice([np.nan, np.inf, -np.inf])
        t, k, p = float(rng.uniform(0.1, 2)), int(rng.integers(1, 60)), float(rng.uniform(0.05, 1))
        u = float(rng.random())
        assert orc.sample(l, t, k, p, u) in tree_ref.draw(l, u, t, k, p, 0.0)


def test_reference_min_p_and_whole_row():
    l = np.log(np.array([0.1, 0.4, 0.2, 0.3])).astype(np.float32)
    order = [1, 3, 2, 0]
    cum = np.cumsum([0.4, 0.3, 0.2, 0.1])
    for u in np.linspace(0.01, 0.99, 25):
        if np.abs(cum - u).min() > 1e-6:
            assert tree_ref.draw(l, u, 1.0, 0, 1.0, 0.0) == {order[int(np.sum(cum < u))]}
    assert tree_ref.draw(l, 0.99, 1.0, 0, 1.0, 0.6) == {3}      # 0.3 / 0.4 stays, 0.2 / 0.4 does not
    assert tree_ref.draw(l, 0.99, 1.0, 0, 0.6, 0.0) == {3}
    assert tree_ref.draw(l, 0.5, 0.0, 0, 1.0, 0.0) == {1}
    assert tree_ref.draw(np.full(3, np.nan, np.float32), 0.5, 1.0, 0, 1.0, 0.0) == {-1}


def test_reference_walk():
    parents, drafted = [-1, 0, 0, 1, 2, 2, -2, 4], [9, 5, 6, 7, 8, 8, 8, 3]
    assert tree_ref.accept(parents, drafted, [6, 0, 8, 0, 3, 0, 0, 4]) == (4, 4, [0, 2, 4, 7])
    assert tree_ref.accept(parents, drafted, [1, 0, 8, 0, 3, 0, 0, 4]) == (1, 1, [0])
    assert tree_ref.accept([-2], [3], [4]) == (0, -1, [])
    assert tree_ref.accept(parents, drafted, [-1] * 8) == (1, -1, [0])
