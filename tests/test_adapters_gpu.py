"""Low-rank adapters of many rows on the MI355X against float64.

Tolerance, with e = 2^-24 (half a step of f32): weights are exact in f32; h is a sum of `cols` products, off by at most cols e of
the sum of its magnitudes; the second sum adds (rank + 2) e, the scale and the sum into y two more roundings, the last of them of
y itself: |y - want| <= (cols + rank + 4) e s sum_k |B| (sum_c |A| |x|) + e |want|. With f16 weights x and h enter the products as two
f16 each: f16 has 11 bits, so the first leaves 2^-11 of an entry at most and the second 2^-11 of that, 2^-22 = 4 e of each: 8 e more (the grid that the
row's largest entry sets, 2^-39 of it, adds less than e: the weighted mean of the magnitudes lies far above 2^-15 of the largest).
The bound is for the worst signs: roundings are independent, so the 2-norm of the difference is held to 16 e sqrt(cols + rank) times
that of the magnitudes' root sums of squares as well.
"""
import ctypes
import math

import numpy as np
import pytest

from tests import pages_ref as ref
from tests.test_pages_gpu import Held, Hip, read, up  # noqa: F401
from webgpu_amd.gpu import Compute, WgdError, WGD_E_INVALID, WGD_E_STATE

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def case(rng, batch, n, rank, cols, rows, half):
    kind = np.float16 if half else np.float32
    a = (rng.standard_normal((n, rank, cols)) / math.sqrt(cols)).astype(kind)
    b = (rng.standard_normal((n, rows, rank)) / math.sqrt(rank)).astype(kind)
    return a, b, rng.standard_normal((batch, cols)).astype(np.float32), rng.uniform(0.1, 2, n).astype(np.float32)


def run(gpu, up, a, b, x, y, which, scales, base=0, type_=None):  # noqa: F811
    n, rank, cols = a.shape
    yb = up(y)
    gpu.adapters((1 if a.dtype == np.float16 else 0) if type_ is None else type_, up(a), up(b), up(np.asarray(which, np.int32)), up(scales), up(x), yb,
                 cols, b.shape[1], rank, n, y.shape[1], base, len(which))
    return read(gpu, yb, y.shape, np.float32)


def assert_near(got, y, x, a, b, which, scales):
    want = ref.adapters(y, x, a, b, which, scales)
    size = ref.adapters(np.zeros_like(y), np.abs(x), np.abs(a), np.abs(b), which, scales)
    cols, rank = a.shape[2], a.shape[1]
    split = 8 if a.dtype == np.float16 else 0
    assert np.all(np.abs(got - want) <= (cols + rank + 4 + split) * EPS * size + EPS * np.abs(want))
    on = (np.asarray(which) >= 0) & (np.asarray(which) < len(scales))
    assert np.array_equal(got[~on], y[~on])
    root = np.zeros(len(which))
    for t in np.flatnonzero(on):  # the norm of independent roundings: of h's products through B, and of the sums
        w = which[t]
        h = np.sqrt((a[w].astype(np.float64) ** 2) @ (x[t].astype(np.float64) ** 2))
        root[t] = scales[w] * np.sqrt(((b[w].astype(np.float64) ** 2) @ h ** 2).sum())
    assert np.linalg.norm(got - want) <= 16 * EPS * math.sqrt(cols + rank) * (np.linalg.norm(root) + np.linalg.norm(want[on]))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("batch,n,rank,cols,rows,extra", [
    (1, 1, 1, 1, 1, 0), (1, 3, 8, 1024, 2048, 0), (4, 3, 8, 1024, 2048, 0), (64, 24, 16, 512, 1000, 0), (65, 2, 16, 256, 64, 7), (3, 2, 5, 33, 17, 2),
    (16, 16, 4, 128, 48, 0), (130, 7, 64, 320, 200, 1), (200, 1, 33, 96, 130, 0), (7, 5, 128, 260, 68, 0), (2, 2, 1024, 64, 20, 0), (300, 64, 2, 36, 36, 0),
    (5, 3, 17, 4096, 30, 0), (1, 2, 16, 14336, 256, 0), (70, 9, 16, 31, 1, 0), (129, 3, 24, 4104, 66, 4)])
def test_adapters(gpu, up, batch, n, rank, cols, rows, extra, half):  # noqa: F811
    rng = np.random.default_rng(batch * 7 + rank)
    a, b, x, scales = case(rng, batch, n, rank, cols, rows, half)
    which = rng.integers(-1, n + 1, batch)
    which[:1] = n - 1
    base = extra // 2
    y = rng.standard_normal((batch, rows + extra)).astype(np.float32)
    got = run(gpu, up, a, b, x, y, which, scales, base)
    inside = slice(base, base + rows)
    assert_near(got[:, inside], y[:, inside], x, a, b, which, scales)
    keep = np.ones(rows + extra, bool)
    keep[inside] = False
    assert np.array_equal(got[:, keep], y[:, keep])
    assert np.array_equal(got, run(gpu, up, a, b, x, y, which, scales, base))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("order", ["runs", "mixed", "one", "none"])
def test_adapters_of_a_prompt(gpu, up, order, half):  # noqa: F811
    rng = np.random.default_rng(4)
    batch, n, rank, cols, rows = 700, 5, 16, 200, 96
    a, b, x, scales = case(rng, batch, n, rank, cols, rows, half)
    which = {"runs": np.arange(batch) // 150 - 1, "mixed": rng.integers(-1, n, batch), "one": np.full(batch, 3), "none": np.full(batch, -7)}[order]
    y = rng.standard_normal((batch, rows)).astype(np.float32)
    assert_near(run(gpu, up, a, b, x, y, which, scales), y, x, a, b, which, scales)


@pytest.mark.parametrize("half", [False, True])
def test_adapters_values_that_are_not_finite_stay_with_their_rows(gpu, up, half):  # noqa: F811
    rng = np.random.default_rng(5)
    batch, n, rank, cols, rows = 40, 4, 12, 100, 52
    a, b, x, scales = case(rng, batch, n, rank, cols, rows, half)
    which = rng.integers(0, n - 1, batch)
    which[::5] = -1
    y = rng.standard_normal((batch, rows)).astype(np.float32)
    clean = run(gpu, up, a, b, x, y, which, scales)
    a[n - 1], b[n - 1], x[3], x[0] = np.nan, np.inf, np.inf, np.nan  # an adapter that no row has; a row; a row without an adapter
    a[1, 2, 7] = np.inf
    scales[n - 1] = np.nan
    got = run(gpu, up, a, b, x, y, which, scales)
    spoilt = (which == 1) | (np.arange(batch) == 3)
    assert which[0] == -1 and which[3] >= 0 and np.array_equal(got[~spoilt], clean[~spoilt])
    assert not np.isfinite(got[spoilt]).all(1).any()


def test_adapters_offsets_pass_32_bits(gpu, up):  # noqa: F811
    """Weights and rows of y behind 2^32 bytes."""
    rng = np.random.default_rng(6)
    rank, cols, rows, n = 16, 4096, 8, 16500 * 2
    big = gpu.buffer(n * rank * cols * 2, "many adapters")
    out = gpu.buffer(3 * (1 << 30) * 4 + 4096, "far rows")
    try:
        a, b, x, scales = case(rng, 3, 1, rank, cols, rows, True)
        gpu.write(big, a[0], (n - 1) * rank * cols * 2)
        bb = gpu.buffer(n * rows * rank * 2, "many adapters")
        gpu.write(bb, b[0], (n - 1) * rows * rank * 2)
        sc = np.ones(n, np.float32)
        sc[-1] = scales[0]
        gpu.adapters(1, big, bb, up(np.array([n - 1, -1, n - 1], np.int32)), up(sc), up(x), out, cols, rows, rank, n, 1 << 30, 5, 3)
        got = np.stack([np.frombuffer(gpu.read(out, rows * 4, (t * (1 << 30) + 5) * 4), np.float32) for t in range(3)])
        assert_near(got, np.zeros((3, rows), np.float32), x, a, b, np.array([0, -1, 0]), scales)
        gpu.destroy(bb)
    finally:
        gpu.destroy(big)
        gpu.destroy(out)


def test_adapters_replay_in_a_graph():
    gpu = Compute().init()
    up = Held(gpu)  # noqa: F811
    hip, stream = Hip(), ctypes.c_void_p(gpu.stream)
    try:
        rng = np.random.default_rng(7)
        batch, n, rank, cols, rows = 70, 6, 16, 320, 96
        a, b, x, scales = case(rng, batch, n, rank, cols, rows, True)
        y = rng.standard_normal((batch, rows)).astype(np.float32)
        bufs = [up(v) for v in (a, b, np.zeros(batch, np.int32), scales, x, y)]
        call = lambda: gpu.adapters(1, *bufs, cols, rows, rank, n, rows, 0, batch)  # noqa: E731
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        gpu.done()
        hip("hipStreamBeginCapture", stream, 2)
        with pytest.raises(WgdError) as e:
            call()
        assert e.value.status == WGD_E_STATE
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphDestroy", graph)

        def reset(i):
            gpu.write(bufs[2], np.random.default_rng(i).integers(-1, n, batch).astype(np.int32))
            gpu.write(bufs[4], x * (1 + i))
            gpu.write(bufs[5], y)

        want = []
        for i in range(3):
            reset(i)
            call()
            want.append(gpu.read(bufs[5], y.nbytes))
        hip("hipStreamBeginCapture", stream, 2)
        call()
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphInstantiate", ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0))
        for i in (2, 0, 1, 1, 2):
            reset(i)
            hip("hipGraphLaunch", exe, stream)
            assert gpu.read(bufs[5], y.nbytes) == want[i]
            a2, b2, x2, s2 = case(rng, 500 + 200 * i, 2, 64, 64, 32, False)  # larger work between
            run(gpu, up, a2, b2, x2, np.zeros((len(x2), 32), np.float32), np.arange(len(x2)) % 2, s2)
        hip("hipGraphExecDestroy", exe)
        hip("hipGraphDestroy", graph)
    finally:
        up.free()
        gpu.dispose()


def test_refusals(gpu, up):  # noqa: F811
    f = [up(np.zeros(1 << 14, np.uint8)) for _ in range(6)]
    tiny = up(np.zeros(4, np.uint8))
    weights = gpu.upload_weights(8, 64, 4, np.zeros(4 * 2 * 34, np.uint8))  # Q8_0, planar
    f32w = gpu.upload_weights(0, 64, 4, np.zeros(256, np.float32))
    other = Compute().init()
    foreign = other.upload(np.zeros(1 << 14, np.uint8))
    A = lambda type_=0, a=f[0], b=f[1], w=f[2], s=f[3], x=f[4], y=f[5], cols=64, rows=32, rank=4, n=2, stride=32, base=0, batch=3: \
        gpu.adapters(type_, a, b, w, s, x, y, cols, rows, rank, n, stride, base, batch)  # noqa: E731
    bad = [lambda: A(type_=8), lambda: A(type_=30), lambda: A(type_=-1), lambda: A(cols=0), lambda: A(rows=0), lambda: A(rank=0), lambda: A(rank=1025),
           lambda: A(n=0), lambda: A(n=2 ** 31), lambda: A(stride=31), lambda: A(base=1), lambda: A(batch=2 ** 24 + 1), lambda: A(a=tiny), lambda: A(b=tiny),
           lambda: A(w=tiny), lambda: A(s=tiny), lambda: A(x=tiny), lambda: A(y=tiny), lambda: A(y=f[0]), lambda: A(y=f[4]), lambda: A(y=f[2]), lambda: A(y=f[3]),
           lambda: A(a=foreign), lambda: A(y=foreign), lambda: A(a=weights), lambda: A(type_=1, a=f32w, n=1), lambda: A(n=17), lambda: A(cols=2 ** 32 - 1),
           lambda: A(stride=2 ** 32 - 1), lambda: A(batch=1, base=2 ** 32 - 1), lambda: A(rows=2 ** 32 - 1, stride=0, batch=1), lambda: A(batch=65)]
    try:
        for i, call in enumerate(bad):
            with pytest.raises(WgdError) as e:
                call()
            assert e.value.status == WGD_E_INVALID, i
        A(batch=0)
        A()
        A(type_=1)
        A(batch=1, stride=0)
        A(a=f32w, n=1)
        gpu.done()
    finally:
        other.dispose()
        gpu.destroy(weights)
        gpu.destroy(f32w)
