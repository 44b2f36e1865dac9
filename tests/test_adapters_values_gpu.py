"""Adapters with weights, inputs and scales far from 1 on the MI355X against float64, and rows with one entry far above the others.

Tolerance: that of tests/test_adapters_gpu.py, (cols + rank + 4) e of the sum of magnitudes and e of the result, with e = 2^-24. With
f16 weights 8 e more (both splits leave 2^-22 = 4 e of an entry), and beside that 2^-39 of the largest entry of a row: of x in every
product of the first sum, where |x| becomes |x| + 2^-39 max|x|, and of h in the second. f32's least step, 2^-149, bounds what a
sum, a product or a split of it can hold: cols + rank + 8 times that of h through |B| s, and of y.
"""
import math

import numpy as np
import pytest

from tests.test_adapters_gpu import case, run
from tests.test_pages_gpu import up  # noqa: F401

pytestmark = pytest.mark.gpu
EPS, LEAST = 2.0 ** -24, 2.0 ** -149


def bounds(y, x, a, b, which, scales):
    """(want, tolerance) of every element, in float64."""
    half, (cols, rank) = a.dtype == np.float16, (a.shape[2], a.shape[1])
    want, room = y.astype(np.float64), np.zeros(y.shape)
    for t, w in enumerate(which):
        if not 0 <= w < len(scales):
            continue
        A, B, xs, s = a[w].astype(np.float64), b[w].astype(np.float64), x[t].astype(np.float64), abs(float(scales[w]))
        h = A @ xs
        want[t] += float(scales[w]) * (B @ h)
        size = np.abs(A) @ np.abs(xs)
        off = (cols + 2 + (4 if half else 0)) * EPS * size + (cols + 4) * LEAST
        if half:
            off += 2.0 ** -39 * np.abs(xs).max() * np.abs(A).sum(1)
        near = np.abs(h) + off
        if half:
            for k in range(0, rank, 64):
                off[k:k + 64] += 2.0 ** -39 * near[k:k + 64].max()
        sums = np.abs(B) @ near
        room[t] = s * (np.abs(B) @ off + (rank + 2 + (4 if half else 0)) * EPS * sums + (rank + 4) * LEAST) + EPS * np.abs(want[t]) + LEAST
    return want, room


def held(gpu, up, a, b, x, y, which, scales):  # noqa: F811
    got = run(gpu, up, a, b, x, y, which, scales)
    want, room = bounds(y, x, a, b, which, scales)
    assert np.isfinite(got).all()
    over = np.abs(got - want) - room
    assert over.max() <= 0, (over.max(), np.unravel_index(over.argmax(), over.shape))
    assert np.linalg.norm(got - want) <= np.linalg.norm(room)
    return got


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("x_size,scale", [(1e30, 1.0), (1e30, 1e5), (1e-30, 1.0), (1e-34, 1e-3), (1e-34, 0.3), (1e-25, 1e-12), (1e-34, 1e6), (1.0, 1e-30), (1.0, 1e30),
                                          (1e-20, -1e20), (1e-20, 1e-18), (1e-20, -1e-20)])
@pytest.mark.parametrize("batch,rank,cols,rows", [(5, 8, 300, 64), (70, 20, 256, 33), (3, 130, 1024, 16)])
def test_adapters_of_large_and_small_inputs(gpu, up, batch, rank, cols, rows, x_size, scale, half):  # noqa: F811
    rng = np.random.default_rng(rank)
    a, b, x, _ = case(rng, batch, 3, rank, cols, rows, half)
    scales = (rng.uniform(0.5, 1, 3) * scale).astype(np.float32)
    held(gpu, up, a, b, (x * x_size).astype(np.float32), np.zeros((batch, rows), np.float32), rng.integers(0, 3, batch), scales)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("batch,rank", [(40, 65), (25, 128), (3, 300), (40, 1024)])
def test_adapters_of_many_ranks_round_y_once(gpu, up, batch, rank, half):  # noqa: F811
    """What is added is far smaller than y: the one rounding of the sum into y is nearly all of the error."""
    rng = np.random.default_rng(rank)
    a, b, x, scales = case(rng, batch, 2, rank, 24, 257, half)
    held(gpu, up, a, b, (x * 1e-5).astype(np.float32), rng.uniform(1, 2, (batch, 257)).astype(np.float32), rng.integers(0, 2, batch), scales)


@pytest.mark.parametrize("half", [False, True])
def test_adapters_whose_scale_and_inner_sums_are_large(gpu, up, half):  # noqa: F811
    """The scale times an inner sum passes f32's range, the scale times B's products with them does not."""
    rng = np.random.default_rng(8)
    a, b, x, scales = case(rng, 30, 2, 12, 200, 64, False)
    kind = np.float16 if half else np.float32
    held(gpu, up, a.astype(kind), (b * 1e-6).astype(kind), (x * 1e30).astype(np.float32), np.zeros((30, 64), np.float32), rng.integers(-1, 2, 30),
         (scales * 1e13).astype(np.float32))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("weight", [1e-6, 3e-8, 2e3])
def test_adapters_of_large_and_small_weights(gpu, up, weight, half):  # noqa: F811
    """1e-6 and 3e-8 are below f16's least normal number, 2^-14, and about a half of its least one, 2^-24."""
    rng = np.random.default_rng(7)
    a, b, x, scales = case(rng, 40, 3, 24, 520, 80, False)
    kind = np.float16 if half else np.float32
    y = rng.standard_normal((40, 80)).astype(np.float32) * np.float32(weight)
    for wa, wb in ((weight, 1.0), (1.0, weight), (weight, weight)):
        held(gpu, up, (a * 20 * wa).astype(kind), (b * wb).astype(kind), x, y, rng.integers(-1, 3, 40), scales)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("far", [1e3, 1e6, 1e10, 1e20, 1e30])
def test_adapters_of_rows_with_one_large_entry(gpu, up, far, half):  # noqa: F811
    """One column of x, wherever it lies among the column ranges, and one row of A; what the largest entry meets may be a weight of zero."""
    rng = np.random.default_rng(9)
    batch, rank, cols, rows = 24, 70, 1300, 36
    a, b, x, scales = case(rng, batch, 2, rank, cols, rows, half)
    at = rng.integers(0, cols, batch)
    at[:4] = 0, cols - 1, 31, 640
    x[np.arange(batch), at] *= np.float32(far)
    which = np.arange(batch) % 2
    held(gpu, up, a, b, x, np.zeros((batch, rows), np.float32), which, scales)
    a[:, :, at] = 0
    held(gpu, up, a, b, x, np.zeros((batch, rows), np.float32), which, scales)
    x[np.arange(batch), at] /= np.float32(far)
    a, b, x, scales = case(rng, batch, 2, rank, cols, rows, half)
    a[:, 5] *= 60000 if half else np.float32(min(far, 1e10))
    held(gpu, up, a, b, x, np.zeros((batch, rows), np.float32), which, scales)
