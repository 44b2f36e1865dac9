"""Draws of whole rows whose logits lie close together for the temperature: a bin of (best - l) / T then holds thousands
of tokens. Draws are checked as in tests/test_tree_gpu.py (tree_ref.draw)."""
import time

import numpy as np
import pytest

from tests import tree_ref
from tests.test_tree_gpu import draw_rows, up  # noqa: F401

pytestmark = pytest.mark.gpu
N = 262144


def in_bin_of_cut(logits, best, t, top):
    """The tokens in the bin in which the running weight reaches `top` of it all."""
    x = (best - np.sort(logits.astype(np.float64))[::-1]) / t
    w = np.cumsum(np.exp(-x))
    at = int(np.searchsorted(w, top * w[-1]))
    bins = np.floor(x * 2048 / 48).astype(np.int64)
    return int((bins == bins[at]).sum())


# standard deviation, temperature, top-k, top-p, and whether the bin of top-p holds more than 2048 tokens (without top-k)
FLAT = [(1.0, 1.5, 0, 0.95, True), (1.5, 2.0, 0, 0.95, True), (2.0, 2.0, 0, 0.9, True), (1.0, 1.0, 0, 0.9, True), (2.5, 1.0, 0, 0.95, False),
        (1.0, 1.2, 100000, 0.9, True), (1.0, 1.2, 100000, 1.0, True), (0.6, 2.0, 0, 0.9, True), (0.6, 2.0, 130000, 0.8, True), (0.3, 1.0, 90000, 1.0, True),
        (0.02, 1.0, 0, 0.5, True), (0.02, 1.0, 70000, 0.9, True)]


@pytest.mark.parametrize("std,t,k,p,full", FLAT)
def test_draws_of_rows_close_together(gpu, up, std, t, k, p, full):  # noqa: F811
    rng = np.random.default_rng(int(1000 * std) + k)
    logits = (rng.standard_normal((4, N)) * std).astype(np.float32)
    logits[3, ::3] = -np.inf
    for l in logits[:3]:
        assert k or (in_bin_of_cut(l, np.float64(l.max()), t, p) > 2048) == full
    for us in (rng.random(4), np.array([1e-9, 0.5, 1 - 1e-9, 0.97])):
        got = draw_rows(gpu, up, logits, us, t, k, p, 0.0)
        for g, l, u in zip(got, logits, us):
            assert g in tree_ref.draw(l, u, t, k, p, 0.0), (g, u)


@pytest.mark.parametrize("rows", [1, 16])
def test_a_higher_temperature_takes_the_same_launches(gpu, up, rows):  # noqa: F811
    """At temperature 2 the bin of top-p holds 2356 of 262144 logits of deviation 2, 694 at temperature 1 and 2.5. Its list has
    room for either: a row that does without its list takes 12 to 16 times as long, four are allowed."""
    rng = np.random.default_rng(rows)
    base = rng.standard_normal((rows, N))
    uniforms, tokens = up(np.full(rows, 0.5)), up(np.zeros(rows, np.int32))

    def took(std, t, p):
        logits, best = up((base * std).astype(np.float32)), []
        for _ in range(5):
            gpu.done()
            begin = time.perf_counter()
            for _ in range(10):
                gpu.sample_rows(logits, N, rows, uniforms, tokens, t, 0, p)
            gpu.done()
            best.append(time.perf_counter() - begin)
        return min(best)

    assert took(2.0, 2.0, 0.9) < 4 * took(2.5, 1.0, 0.95)
