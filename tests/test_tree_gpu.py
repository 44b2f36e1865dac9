"""The drafted-tree operators on the MI355X against the float64 forms of tests/tree_ref.py, and one
decode step over a tree against token-by-token decoding with the operators that were there before.

Tolerances, with e = 2^-24 (half a step of f32):
* rope: each output is a sum of two products of f32 values with a cosine and a sine, which are off
  by at most 2 e each; two products and a sum round once each: 5 e (|l| + |r|) at most, 8 e allowed.
* attention: the f32 dot product of hd terms is off by at most hd e sum|q k|, so a weight by twice
  that and by its own rounding; numerator and denominator are sums of n weights, n e each at most:
  |y - want| <= (2 (hd + 4) e S + 2 (n + 8) e) max|v| with S = scale max sum|q k|. The bound is
  for the worst signs: roundings are independent, so the 2-norm of the difference is held to
  16 e sqrt(hd + n) times the 2-norm of the result as well, with at least 1 for sqrt(S) beside it.
* draws: one token, except where the uniform lies within 1e-9 of a border (tree_ref.draw).
* accepted paths and moved rows: equal.
"""
import ctypes
import math

import numpy as np
import pytest

from tests import tree_ref
from webgpu_amd.gpu import Compute, WgdError, WGD_E_INVALID, WGD_E_STATE
from webgpu_amd.rope import llama3_factors

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
NO_WINDOW = 1 << 30


class Held:
    """Buffers of one test, destroyed at its end."""

    def __init__(self, gpu):
        self.gpu, self.held = gpu, []

    def __call__(self, array, label="test"):
        self.held.append(self.gpu.upload(np.ascontiguousarray(array), label))
        return self.held[-1]

    def free(self):
        for b in self.held:
            self.gpu.destroy(b)


@pytest.fixture
def up(gpu):
    h = Held(gpu)
    yield h
    h.free()


def read(gpu, b, dtype, shape):
    n = int(np.prod(shape))
    return np.frombuffer(gpu.read(b, n * np.dtype(dtype).itemsize), dtype).reshape(shape).copy()


# ------------------------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("heads,hd,rot,batch,adjacent,factors,pad,offset", [
    (1, 2, 2, 1, False, False, 0, 0), (24, 128, 128, 1, False, False, 1024, 0), (40, 128, 128, 64, True, True, 1024, 0),
    (3, 64, 32, 17, False, True, 6, 5), (5, 80, 40, 9, True, False, 1, 3), (2, 96, 96, 256, False, False, 0, 0),
    (1, 256, 256, 33, True, True, 0, 256), (7, 6, 4, 5, False, True, 0, 1), (2, 1040, 1030, 3, False, False, 0, 0),
    (48, 128, 64, 3, False, False, 0, 4), (16, 512, 512, 2, True, False, 0, 0)])
def test_rope_at(gpu, up, heads, hd, rot, batch, adjacent, factors, pad, offset):
    rng = np.random.default_rng(heads * hd + batch)
    stride = heads * hd + pad
    x = rng.standard_normal(offset + batch * stride + 3).astype(np.float32)
    pos = rng.integers(0, 200000, batch).astype(np.int32)
    pos[:2] = [0, -7][:min(2, batch)]
    f = llama3_factors(rot, 5e5, 8.0, 1.0, 4.0, 8192) if factors else None
    xb, pb = up(x), up(pos)
    gpu.rope_at(xb, pb, heads, hd, 5e5, 0.25, rot if rot != hd else 0, batch, adjacent=adjacent,
                factors=up(f) if factors else None, magnitude=1.25, stride=stride if pad else 0, offset=offset)
    got = read(gpu, xb, np.float32, x.shape)
    rows = lambda a: a[offset:offset + batch * stride].reshape(batch, stride)[:, :heads * hd].reshape(batch, heads, hd)  # noqa: E731
    before = rows(x).astype(np.float64)
    want = tree_ref.rope(before, pos, 5e5, 0.25, rot, adjacent, f, 1.25)
    other = before.copy()  # |l| + |r| of each value's pair
    i = np.arange(rot)
    j = i ^ 1 if adjacent else (i + rot // 2) % rot
    other[..., :rot] = np.abs(before[..., i]) + np.abs(before[..., j])
    assert np.all(np.abs(rows(got) - want)[..., :rot] <= 8 * EPS * 1.25 * other[..., :rot])
    assert np.array_equal(rows(got)[..., rot:], rows(x)[..., rot:])
    keep = np.ones(x.size, bool)  # what lies around the heads stays
    keep[offset:offset + batch * stride].reshape(batch, stride)[:, :heads * hd] = False
    assert np.array_equal(got[keep], x[keep])


def test_rope_at_far_positions_and_single_ops_agree(gpu, up):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 2, 128)).astype(np.float32)
    pos = np.array([2 ** 31 - 1, -2 ** 31, 16777217], np.int32)
    xb = up(x)
    gpu.rope_at(xb, up(pos), 2, 128, 1e4, 1.0, 128, 3)
    want = tree_ref.rope(x, pos, 1e4, 1.0, 128, False)
    # the angle itself is known to 2^-52 of it and a few roundings more
    slack = 8 * EPS + 2.0 ** 31 * 2.0 ** -50
    assert np.all(np.abs(read(gpu, xb, np.float32, x.shape) - want) <= slack * 2 * np.abs(x).max())
    # consecutive positions: the operator that takes a start
    x = rng.standard_normal((9, 4, 64)).astype(np.float32)
    for adjacent in (False, True):
        a, b = up(x), up(x)
        gpu.rope_at(a, up(np.arange(500, 509, dtype=np.int32)), 4, 64, 1e6, 0.5, 48, 9, adjacent=adjacent)
        (gpu.rope_adjacent if adjacent else gpu.rope_neox)(b, 4, 64, 500, 1e6, 0.5, 48, 9)
        d = np.abs(read(gpu, a, np.float32, x.shape) - read(gpu, b, np.float32, x.shape))
        assert d.max() <= 16 * EPS * 2 * np.abs(x).max()


def test_rope_at_non_finite_values_stay_in_their_pairs(gpu, up):
    x = np.ones((2, 1, 64), np.float32)
    x[0, 0, 3], x[1, 0, 40] = np.nan, np.inf
    xb = up(x)
    gpu.rope_at(xb, up(np.array([11, 12], np.int32)), 1, 64, 1e4, 1.0, 64, 2)
    bad = ~np.isfinite(read(gpu, xb, np.float32, x.shape))
    want = np.zeros_like(bad)
    want[0, 0, [3, 35]] = want[1, 0, [8, 40]] = True
    assert np.array_equal(bad, want)


# ------------------------------------------------------------------------------- attention

def random_tree(rng, nodes, span=6, pads=0, roots=1):
    parents = [-1] * min(roots, nodes) + [int(rng.integers(max(0, i - span), i)) for i in range(roots, nodes)]
    for i in rng.choice(np.arange(1, nodes), min(pads, nodes - 1), replace=False) if pads else []:
        parents[i] = int(rng.choice([-2, -2 ** 31, i, i + 1, 2 ** 31 - 1]))
    return np.array(parents, np.int32)


def tree_case(rng, heads, kvh, hd, nodes, start, window, extra, kv, qk=1.0):
    cap = min(start, window - 1) + nodes + extra
    q = (rng.standard_normal((nodes, heads, hd)) * qk).astype(np.float32)
    k, v = (rng.standard_normal((cap, kvh, hd)).astype(np.float16 if kv == "f16" else np.float32) for _ in range(2))
    return q, k, v, cap


def run_tree(gpu, up, q, k, v, parents, start, scale, window, tail=0):
    nodes, heads, hd = q.shape
    y = up(np.full(q.size + tail, 77.0, np.float32))
    op = gpu.attention_tree_f16kv if k.dtype == np.float16 else gpu.attention_tree
    op(up(q), up(k), up(v), y, up(parents), heads, k.shape[1], hd, start, scale, window, k.shape[0], nodes)
    got = read(gpu, y, np.float32, q.size + tail)
    assert np.all(got[q.size:] == 77.0)
    return got[:q.size].reshape(q.shape)


def assert_near(got, q, k, v, parents, start, scale, window):
    want = tree_ref.attention(q, k, v, parents, start, scale, window)
    hd, n = q.shape[2], min(start, window) + len(parents)
    group = q.shape[1] // k.shape[1]
    S = scale * max(float((np.abs(q[:, g * group:(g + 1) * group]).reshape(-1, hd).astype(np.float64) @ np.abs(k[:, g].astype(np.float64)).T).max())
                    for g in range(k.shape[1]))
    bound = (2 * (hd + 4) * EPS * S + 2 * (n + 8) * EPS) * float(np.abs(v.astype(np.float64)).max())
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= bound, (np.abs(got - want).max(), bound)
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= 16 * EPS * math.sqrt(hd + n) * max(1, math.sqrt(S)) * norm, np.linalg.norm(got - want) / norm
    pad = [i for i, p in enumerate(tree_ref.paths(parents)) if p is None]
    assert np.all(got[pad] == 0)


CASES = [
    # heads, kv_heads, head_dim, nodes, start, window, slots to spare
    (1, 1, 1, 1, 0, NO_WINDOW, 0), (4, 2, 8, 1, 0, 1, 0), (2, 1, 64, 1, 1, NO_WINDOW, 0), (16, 8, 128, 16, 300, NO_WINDOW, 700),
    (32, 8, 128, 33, 517, NO_WINDOW, 0), (8, 8, 128, 2, 63, NO_WINDOW, 1), (14, 2, 64, 15, 200, NO_WINDOW, 5),
    (3, 1, 128, 17, 64, NO_WINDOW, 0), (20, 1, 64, 7, 130, NO_WINDOW, 0), (34, 2, 128, 5, 40, NO_WINDOW, 0),
    (4, 2, 256, 24, 100, NO_WINDOW, 3), (8, 4, 80, 12, 90, NO_WINDOW, 0), (6, 2, 96, 31, 33, 20, 0), (2, 1, 17, 9, 50, NO_WINDOW, 2),
    (2, 2, 512, 6, 70, NO_WINDOW, 0), (4, 1, 128, 255, 10, NO_WINDOW, 0), (2, 1, 64, 256, 300, NO_WINDOW, 0), (2, 1, 128, 256, 0, 9, 0),
    (8, 4, 128, 40, 1000, 100, 0), (8, 4, 128, 40, 1000, 100, 27), (4, 4, 64, 64, 777, 3, 0), (4, 2, 128, 20, 500, 1, 0),
    (4, 2, 128, 20, 500, 2, 1), (16, 8, 128, 48, 5000, 1024, 80), (7, 1, 128, 64, 3000, NO_WINDOW, 9), (2, 2, 256, 3, 2000, 600, 0),
    (64, 4, 64, 100, 250, NO_WINDOW, 0), (8, 1, 256, 130, 333, NO_WINDOW, 0),
]


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join("w" if v == NO_WINDOW else str(v) for v in c))
def test_attention_tree(gpu, up, case, kv):
    heads, kvh, hd, nodes, start, window, extra = case
    rng = np.random.default_rng(heads * 1000 + nodes + start)
    q, k, v, cap = tree_case(rng, heads, kvh, hd, nodes, start, window, extra, kv)
    parents = random_tree(rng, nodes, pads=nodes // 8, roots=2 if nodes > 20 else 1)
    scale = 1 / math.sqrt(hd)
    got = run_tree(gpu, up, q, k, v, parents, start, scale, window, tail=5)
    assert_near(got, q, k, v, parents, start, scale, window)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("shape", ["chain", "star", "all-roots", "all-padding"])
def test_attention_tree_shapes(gpu, up, shape, kv):
    rng = np.random.default_rng(8)
    n = 37
    parents = {"chain": np.arange(-1, n - 1), "star": np.array([-1] + [0] * (n - 1)), "all-roots": np.full(n, -1),
               "all-padding": np.full(n, -2)}[shape].astype(np.int32)
    for window in (NO_WINDOW, 12):
        q, k, v, cap = tree_case(rng, 8, 2, 128, n, 150, window, 4, kv)
        got = run_tree(gpu, up, q, k, v, parents, 150, 0.09, window)
        if shape == "all-padding":
            assert np.all(got == 0)
        else:
            assert_near(got, q, k, v, parents, 150, 0.09, window)
        if shape == "chain":  # the causal operator over the same ring
            y = up(np.zeros(q.size, np.float32))
            (gpu.attention_f16kv if kv == "f16" else gpu.attention)(up(q), up(k), up(v), y, 8, 2, 128, 150, 0.09, min(window, 4096), cap,
                                                                    cap, n)
            assert np.abs(read(gpu, y, np.float32, q.shape) - got).max() <= 2e-5


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("scale_of", [1e-6, 30.0, 0.0])
def test_attention_tree_magnitudes(gpu, up, hd, kv, scale_of):
    """Scores of one key, all alike, and zero; queries, keys and values of other sizes than 1."""
    rng = np.random.default_rng(hd)
    q, k, v, cap = tree_case(rng, 4, 2, hd, 20, 210, NO_WINDOW, 0, kv)
    q, v = q * np.float32(scale_of), (v.astype(np.float32) * (200 if kv == "f16" else 1e6)).astype(v.dtype)
    k = (k.astype(np.float32) * 0.01).astype(k.dtype)
    parents = random_tree(rng, 20)
    got = run_tree(gpu, up, q, k, v, parents, 210, 3.0, NO_WINDOW)
    assert_near(got, q, k, v, parents, 210, 3.0, NO_WINDOW)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd,heads,kvh", [(128, 8, 2), (64, 4, 4), (256, 4, 2), (40, 2, 1)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_attention_tree_masked_places_reach_nothing(gpu, up, hd, heads, kvh, bad, kv):
    rng = np.random.default_rng(hd + 1)
    nodes, start, window = 40, 230, 64
    q, k, v, cap = tree_case(rng, heads, kvh, hd, nodes, start, window, 9, kv)
    parents = random_tree(rng, nodes)
    paths = tree_ref.paths(parents)
    clean = run_tree(gpu, up, q, k, v, parents, start, 0.1, window)
    # slots that nobody sees
    seen = {t % cap for t in range(start + 1 - window, start + nodes)}
    unseen = [s for s in range(cap) if s not in seen]
    assert unseen
    k1, v1 = k.copy(), v.copy()
    k1[unseen], v1[unseen] = bad, bad
    assert np.array_equal(run_tree(gpu, up, q, k1, v1, parents, start, 0.1, window), clean)
    # a node that some see, and the cached key that only the nodes of depth 0 see
    for slot, sees in (((start + 3) % cap, [3 in p for p in paths]), ((start + 1 - window) % cap, [len(p) == 1 for p in paths])):
        for which in ("v", "k"):
            k1, v1 = k.copy(), v.copy()
            (v1 if which == "v" else k1)[slot, :, hd // 2] = bad
            got = run_tree(gpu, up, q, k1, v1, parents, start, 0.1, window)
            want = tree_ref.attention(q, k1, v1, parents, start, 0.1, window)
            for i in range(nodes):
                if not sees[i]:  # formed another way beside such values, to the same accuracy
                    assert np.abs(got[i] - clean[i]).max() <= 1e-5, (which, i)
                else:
                    assert np.array_equal(np.isnan(got[i]), np.isnan(want[i])), (which, i)
                    inf = np.isinf(want[i])
                    assert np.array_equal(got[i][inf], want[i][inf])
                    fine = np.isfinite(want[i])
                    assert np.allclose(got[i][fine], want[i][fine], rtol=0, atol=1e-3)
    # a query that is not finite spoils its own row alone
    q1 = q.copy()
    q1[5, heads - 1, 0] = bad
    got = run_tree(gpu, up, q1, k, v, parents, start, 0.1, window)
    assert not np.isfinite(got[5, heads - 1]).any()
    got[5, heads - 1] = clean[5, heads - 1]
    assert np.abs(got - clean).max() <= 1e-5


def test_attention_tree_repeats_itself_and_two_contexts_agree(gpu, up):
    rng = np.random.default_rng(12)
    q, k, v, cap = tree_case(rng, 32, 8, 128, 48, 4000, NO_WINDOW, 0, "f16")
    parents = random_tree(rng, 48)
    first = run_tree(gpu, up, q, k, v, parents, 4000, 0.1, NO_WINDOW)
    assert np.array_equal(first, run_tree(gpu, up, q, k, v, parents, 4000, 0.1, NO_WINDOW))
    other = Compute().init()
    try:
        h = Held(other)
        assert np.array_equal(first, run_tree(other, h, q, k, v, parents, 4000, 0.1, NO_WINDOW))
        h.free()
    finally:
        other.dispose()


def test_attention_tree_long_ring_offsets(gpu, up):
    """Rows past 2^32 bytes (and 2^31 elements) of a ring."""
    kvh, hd, cap = 16, 128, (1 << 20) + 64
    big = gpu.buffer(cap * kvh * hd * 2, "long ring")
    try:
        rng = np.random.default_rng(2)
        start, window, nodes = cap - 20, 200, 30
        q, k, v, _ = tree_case(rng, 16, kvh, hd, nodes, start, window, 0, "f16")
        parents = random_tree(rng, nodes)
        slots = [t % cap for t in range(start + 1 - window, start + nodes)]
        ring = {m: np.zeros((len(slots), kvh, hd), np.float16) for m in "k"}
        ring["k"] = rng.standard_normal((len(slots), kvh, hd)).astype(np.float16)
        row = kvh * hd * 2
        split = next(i for i, s in enumerate(slots) if s == 0)
        gpu.write(big, ring["k"][:split], slots[0] * row)
        gpu.write(big, ring["k"][split:], 0)
        y = up(np.zeros(q.size, np.float32))
        gpu.attention_tree_f16kv(up(q), big, big, y, up(parents), 16, kvh, hd, start, 0.1, window, cap, nodes)
        got = read(gpu, y, np.float32, q.shape)
        # the same keys in a ring that holds just them
        small = np.roll(ring["k"], (start + 1 - window) % len(slots), axis=0)
        want = tree_ref.attention(q, small, small, parents, start, 0.1, window)
        assert np.abs(got - want).max() <= 1e-5
    finally:
        gpu.destroy(big)


# ------------------------------------------------------------------------------- draws

def draw_rows(gpu, up, logits, uniforms, t, k, p, m, stride=None):
    rows, n = len(uniforms), logits.shape[1] if stride is None else stride[0]
    tokens = up(np.full(rows + 1, 99, np.int32))
    gpu.sample_rows(up(logits), n, rows, up(np.asarray(uniforms, np.float64)), tokens, t, k, p, m,
                    stride=0 if stride is None else logits.shape[1])
    got = read(gpu, tokens, np.int32, rows + 1)
    assert got[rows] == 99
    return got[:rows].tolist()


def sample_inputs():
    rng = np.random.default_rng(21)
    yield "normal-1000", rng.standard_normal(1000) * 2
    yield "one", np.array([-5.0])
    yield "two", np.array([-5.0, 3.0])
    yield "sixty-three", rng.standard_normal(63) * 3
    yield "slice-2048", rng.standard_normal(2048) * 3
    yield "slice-2049", rng.standard_normal(2049) * 3
    yield "vocab-151936", rng.standard_normal(151936) * 2.5
    yield "vocab-262144", rng.standard_normal(262144)
    yield "flat-262143", rng.standard_normal(262143) * 1e-4
    yield "rounded-ties", np.round(rng.standard_normal(30000) * 2)
    yield "all-equal", np.full(30001, 0.25)
    yield "two-values", np.where(rng.random(20000) < 0.3, 1.0, -1.0)
    yield "one-binade", 0.5 + 0.5 * rng.random(50000)
    yield "huge", rng.standard_normal(3000) * 1e38
    yield "peaked", np.concatenate([[30.0], rng.standard_normal(40000) - 20])
    yield "zeros", np.array([0.0, -0.0, -1.0, 0.0, -0.0, -3.0] * 500)
    l = rng.standard_normal(5000)
    l[rng.integers(0, 5000, 40)] = np.nan
    l[rng.integers(0, 5000, 40)] = np.inf
    l[rng.integers(0, 5000, 40)] = -np.inf
    yield "non-finite", l
    l = np.full(150000, np.nan)
    l[70000:75000] = rng.standard_normal(5000)
    yield "empty-slices", l
    yield "lowest", np.where(rng.random(9000) < 0.9, np.finfo(np.float32).min, rng.standard_normal(9000))


SETTINGS = [(0.7, 40, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (1.5, 0, 1.0, 0.05), (0.3, 200, 1.0, 0.0), (2.0, 3000, 0.9, 0.0),
            (1.0, 3000, 1.0, 0.001), (1.0, 1000, 0.5, 0.1), (0.8, 2, 0.99, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 1e-9, 0.0), (1.0, 0, 1.0, 1.0),
            (0.0, 5, 0.9, 0.5), (1e-3, 0, 0.9, 0.0), (1e-300, 0, 1.0, 0.0), (1.0, 2 ** 32 - 1, 0.999, 1e-30)]


@pytest.mark.parametrize("name,logits", list(sample_inputs()), ids=[n for n, _ in sample_inputs()])
def test_sample_rows_draws_the_formula(gpu, up, name, logits):
    with np.errstate(over="ignore"):
        logits = np.asarray(logits).astype(np.float32)
    rng = np.random.default_rng(logits.size)
    us = np.concatenate([rng.random(10), [1e-12, 1 - 1e-7]])
    rows = np.tile(logits, (len(us), 1))
    for t, k, p, m in SETTINGS:
        got = draw_rows(gpu, up, rows, us, t, k, p, m)
        for g, u, may in zip(got, us, tree_ref.draws(logits, us, t, k, p, m)):
            assert g in may, (name, t, k, p, m, u, g, may)


def test_sample_rows_of_many_rows_apart(gpu, up):
    rng = np.random.default_rng(9)
    rows, n, stride = 530, 700, 777
    logits = (rng.standard_normal((rows, stride)) * 3).astype(np.float32)
    logits[:, n:] = 1e9  # beyond the row
    logits[17, :n] = np.nan
    us = rng.random(rows)
    got = draw_rows(gpu, up, logits, us, 0.9, 50, 0.95, 0.01, stride=(n,))
    for i in range(rows):
        assert got[i] in tree_ref.draw(logits[i, :n], us[i], 0.9, 50, 0.95, 0.01), i
    assert got[17] == -1
    assert draw_rows(gpu, up, logits, us, 0.0, 50, 0.95, 0.0, stride=(n,)) == \
        [-1 if i == 17 else int(np.argmax(logits[i, :n])) for i in range(rows)]


def test_sample_rows_uniforms_outside_the_range_take_the_best(gpu, up):
    logits = np.tile(np.array([0.0, 1.0, 3.0, 2.0], np.float32), (7, 1))
    us = [0.0, 1.0, -0.5, 1.5, np.nan, np.inf, 1 - 2.0 ** -53]
    assert draw_rows(gpu, up, logits, us, 1.0, 0, 1.0, 0.0) == [2] * 6 + [0]


def test_sample_rows_equals_the_single_row_operator(gpu, up):
    rng = np.random.default_rng(31)
    logits = (rng.standard_normal(128256) * 2.5).astype(np.float32)
    from oracle import orc
    us = [orc.uniform(77, i) for i in range(32)]
    lb = up(logits)
    want = [gpu.sample(lb, logits.size, 0.7, 40, 0.9, 77, i) for i in range(32)]
    assert draw_rows(gpu, up, np.tile(logits, (32, 1)), us, 0.7, 40, 0.9, 0.0) == want


# ------------------------------------------------------------------------------- accepted paths

@pytest.mark.parametrize("nodes", [1, 2, 3, 16, 63, 64, 65, 200, 256])
def test_tree_accept(gpu, up, nodes):
    rng = np.random.default_rng(nodes)
    for trial in range(8):
        parents = random_tree(rng, nodes, span=[1, 6, nodes][trial % 3], pads=nodes // 10)
        vocab = [2, 5, 100000][trial % 3]
        drafted, picked = (rng.integers(0, vocab, nodes).astype(np.int32) for _ in range(2))
        if trial % 2:
            inner = (parents >= 0) & (parents < np.arange(nodes))
            hit = inner & (rng.random(nodes) < 0.8)
            drafted[hit] = picked[parents[hit]]
        if trial == 7:
            picked[rng.random(nodes) < 0.2] = -1
            drafted[rng.random(nodes) < 0.2] = -1
        path = up(np.full(nodes + 4, 7, np.int32))
        gpu.tree_accept(up(parents), up(drafted), up(picked), path, nodes)
        got = read(gpu, path, np.int32, nodes + 4).tolist()
        count, token, want = tree_ref.accept(parents, drafted, picked)
        assert got[:2] == [count, token] and got[2:2 + nodes] == want + [-1] * (nodes - count) and got[nodes + 2:] == [7, 7]


def test_tree_accept_without_a_root(gpu, up):
    for first in (-2, 0, 5):
        path = up(np.full(5, 7, np.int32))
        gpu.tree_accept(up(np.array([first, 0, 0], np.int32)), up(np.zeros(3, np.int32)), up(np.zeros(3, np.int32)), path, 3)
        assert read(gpu, path, np.int32, 5).tolist() == [0, -1, -1, -1, -1]


@pytest.mark.parametrize("row,rings,dtype", [(1024 * 4, 2, np.uint8), (1024 * 2, 130, np.uint8), (2, 1, np.uint8), (6, 3, np.uint8),
                                             (20, 2, np.uint8), (80 * 3 * 2, 64, np.uint8), (16, 65, np.uint8), (128 * 40, 4, np.uint8)])
def test_kv_commit(gpu, up, row, rings, dtype):
    rng = np.random.default_rng(row + rings)
    for nodes, capacity, start, count in ((1, 1, 5, 1), (16, 16, 300, 5), (64, 100, 2 ** 31 - 1, 20), (40, 57, 50, 40), (256, 256, 0, 100),
                                          (9, 30, 29, 0)):
        data = rng.integers(0, 256, (rings, capacity, row)).astype(np.uint8)
        path = np.full(nodes + 2, -1, np.int32)
        path[:2] = count, 5
        if count:
            path[2:2 + count] = np.concatenate([[0], np.sort(1 + rng.permutation(nodes - 1)[:count - 1])])
        bufs = [up(d) for d in data]
        gpu.kv_commit(bufs, up(path), row, start, capacity, nodes)
        for d in data:
            for j in range(count):
                d[(start + j) % capacity] = d[(start + int(path[2 + j])) % capacity]
        for b, d in zip(bufs, data):
            assert np.array_equal(read(gpu, b, np.uint8, d.shape), d), (nodes, capacity, count)
    for b in up.held:
        gpu.destroy(b)
    up.held.clear()


def test_kv_commit_of_entries_out_of_range_moves_nothing(gpu, up):
    data = np.arange(10 * 16, dtype=np.uint8).reshape(10, 16)
    for path in ([2 ** 31 - 1, 0, -1, 9, 2 ** 31 - 1, -2 ** 31, 1, 2, 5, 6, 7, 8], [-5, 0] + [3] * 10, [300, 0, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9]):
        b = up(data)
        gpu.kv_commit([b], up(np.array(path, np.int32)), 16, 0, 10, 8)
        assert np.array_equal(read(gpu, b, np.uint8, data.shape), data)


# ------------------------------------------------------------------------------- a whole step

def plain_model(rng, vocab, heads, kvh, hd, hidden):
    w = lambda r, c, s: (rng.standard_normal((r, c)) * s).astype(np.float32)  # noqa: E731
    return {"embd": w(vocab, hidden, 1.0), "qkv": w((heads + 2 * kvh) * hd, hidden, 0.4 / math.sqrt(hidden) * 4),
            "o": w(hidden, heads * hd, 2.0 / math.sqrt(heads * hd)), "out": w(vocab, hidden, 1.5)}


class Step:
    """One attention layer and a head, run with the framework's operators."""

    def __init__(self, gpu, up, rng, half, heads=8, kvh=2, hd=64, hidden=128, vocab=96, capacity=96, window=70):
        self.gpu, self.half, self.window = gpu, half, window
        self.heads, self.kvh, self.hd, self.hidden, self.vocab, self.capacity = heads, kvh, hd, hidden, vocab, capacity
        self.w = {n: up(a, n) for n, a in plain_model(rng, vocab, heads, kvh, hd, hidden).items()}
        size = 2 if half else 4
        self.k, self.v = (gpu.buffer(capacity * kvh * hd * size, n) for n in "kv")
        self.row = kvh * hd

    def project(self, up, ids):
        g, n = self.gpu, len(ids)
        self.x, qkv = (g.buffer(4 * n * m, "work") for m in (self.hidden, (self.heads + 2 * self.kvh) * self.hd))
        up.held += [self.x, qkv]
        g.embed(0, self.w["embd"], up(np.array(ids, np.int32)), self.x, self.hidden, n)
        rows = (self.heads + 2 * self.kvh) * self.hd
        g.matmul(0, self.w["qkv"], self.x, qkv, self.hidden, rows, rows, 0, 0, n)
        return qkv, rows

    def store(self, up, qkv, rows, start, n):
        """K and V of the rows into the ring; q as one batch."""
        q = np.frombuffer(self.gpu.read(qkv, 4 * n * rows), np.float32).reshape(n, rows)
        hq = self.heads * self.hd
        kb, vb = up(q[:, hq:hq + self.row]), up(q[:, hq + self.row:])
        for i in range(n):
            slot = (start + i) % self.capacity
            for src, ring in ((kb, self.k), (vb, self.v)):
                if self.half:
                    self.gpu.kv_store_f16(src, ring, self.row, i * self.row, slot * self.row)
                else:
                    self.gpu.copy(src, ring, 4 * self.row, 4 * i * self.row, 4 * slot * self.row)
        return up(q[:, :hq])

    def logits(self, up, y, n):
        g = self.gpu
        out = g.buffer(4 * n * self.vocab, "logits")
        o = g.buffer(4 * n * self.hidden, "o")
        up.held += [out, o]
        g.matmul(0, self.w["o"], y, o, self.heads * self.hd, self.hidden, self.hidden, 0, 0, n)
        g.add(o, self.x, n * self.hidden)
        g.matmul(0, self.w["out"], self.x, out, self.hidden, self.vocab, self.vocab, 0, 0, n)
        return out

    def one(self, up, token, start):
        """A token with the operators of token-by-token decoding; returns its logits."""
        qkv, rows = self.project(up, [token])
        g = self.gpu
        g.rope_neox(qkv, self.heads + self.kvh, self.hd, start, 1e4, 1.0, self.hd, 1)
        q = self.store(up, qkv, rows, start, 1)
        y = up(np.zeros(self.heads * self.hd, np.float32))
        (g.attention_f16kv if self.half else g.attention)(q, self.k, self.v, y, self.heads, self.kvh, self.hd, start, 0.125, self.window,
                                                         self.capacity, self.capacity, 1)
        return self.logits(up, y, 1)

    def ring(self, slots):
        size = np.float16 if self.half else np.float32
        return [read(self.gpu, b, size, (self.capacity, self.row))[slots].astype(np.float32) for b in (self.k, self.v)]


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_a_step_over_a_tree_equals_token_by_token_decoding(gpu, up, half, temperature):
    rng = np.random.default_rng(41)
    a, b = (Step(gpu, up, np.random.default_rng(6), half) for _ in range(2))
    try:
        prompt = rng.integers(0, a.vocab, 85).tolist()  # the ring wraps inside the tree
        for i, t in enumerate(prompt[:-1]):
            a.one(up, t, i)
            b.one(up, t, i)
        start, depth, token = len(prompt) - 1, 6, prompt[-1]
        us = rng.random(64)
        # token by token: the token at depth d is drawn with the d-th uniform
        tokens, t = [], token
        for d in range(depth):
            out = a.one(up, t, start + d)
            picked = up(np.zeros(1, np.int32))
            gpu.sample_rows(out, a.vocab, 1, up(us[d:d + 1]), picked, temperature, 20, 0.95)
            t = int(read(gpu, picked, np.int32, 1)[0])
            tokens.append(t)
        # the tree: each level holds wrong guesses around the token that will be drawn, the last level only wrong ones
        parents, drafted, depths, at = [-1], [token], [0], 0
        for d in range(depth):
            right = None
            for guess in range(3):
                wrong = (tokens[d] + 1 + guess) % a.vocab
                is_right = guess == d % 3 and d < depth - 1
                parents.append(at)
                drafted.append(tokens[d] if is_right else wrong)
                depths.append(d + 1)
                right = len(parents) - 1 if is_right else right
            at = right
        n = len(parents) + 2  # two nodes of padding
        parents, drafted, depths = (np.array(x + [f] * 2, np.int32) for x, f in ((parents, -2), (drafted, 0), (depths, 0)))
        qkv, rows = b.project(up, drafted.tolist())
        gpu.rope_at(qkv, up(start + depths), b.heads + b.kvh, b.hd, 1e4, 1.0, b.hd, n, stride=rows)
        q = b.store(up, qkv, rows, start, n)
        y = up(np.zeros(n * b.heads * b.hd, np.float32))
        pb, db = up(parents), up(drafted)
        (gpu.attention_tree_f16kv if half else gpu.attention_tree)(q, b.k, b.v, y, pb, b.heads, b.kvh, b.hd, start, 0.125, b.window,
                                                                  b.capacity, n)
        out = b.logits(up, y, n)
        picked, path = up(np.zeros(n, np.int32)), up(np.zeros(n + 2, np.int32))
        gpu.sample_rows(out, b.vocab, n, up(us[depths]), picked, temperature, 20, 0.95)
        gpu.tree_accept(pb, db, picked, path, n)
        gpu.kv_commit([b.k, b.v], path, b.row * (2 if half else 4), start, b.capacity, n)
        got = read(gpu, path, np.int32, n + 2).tolist()
        assert got[0] == depth and got[1] == tokens[-1]
        assert drafted[got[2:2 + depth]].tolist() == [token] + tokens[:-1]
        slots = [(start + j) % b.capacity for j in range(depth)]
        for x, z in zip(a.ring(slots), b.ring(slots)):  # the batch's products and angles round apart; halves may round apart once more
            assert np.abs(x - z).max() <= (2 ** -9 if half else 1e-5) * np.abs(x).max()
    finally:
        for s in (a, b):
            gpu.destroy(s.k)
            gpu.destroy(s.v)


# ------------------------------------------------------------------------------- graphs

class Hip:
    def __init__(self):
        self.l = ctypes.CDLL("libamdhip64.so")

    def __call__(self, name, *args):
        rc = getattr(self.l, name)(*args)
        assert rc == 0, (name, rc)


def test_the_operators_replay_in_a_graph(up):
    gpu = Compute().init()  # a context of its own: its scratch starts empty
    up = Held(gpu)
    hip, stream = Hip(), ctypes.c_void_p(gpu.stream)
    try:
        rng = np.random.default_rng(3)
        nodes, start, vocab = 24, 900, 5000
        q, k, v, cap = tree_case(rng, 16, 4, 128, nodes, start, NO_WINDOW, 0, "f32")
        parents = random_tree(rng, nodes)
        logits = (rng.standard_normal((nodes, vocab)) * 2).astype(np.float32)
        qb, kb, vb, pb, lb = up(q), up(k), up(v), up(parents), up(logits)
        y, ub, tokens, db, path = up(np.zeros_like(q)), up(rng.random(nodes)), up(np.zeros(nodes, np.int32)), \
            up(rng.integers(0, 3, nodes).astype(np.int32)), up(np.zeros(nodes + 2, np.int32))
        posb = up(np.arange(nodes, dtype=np.int32))
        xb = up(q)

        def step():
            gpu.rope_at(xb, posb, 16, 128, 1e4, 1.0, 128, nodes)
            gpu.attention_tree(qb, kb, vb, y, pb, 16, 4, 128, start, 0.08, NO_WINDOW, cap, nodes)
            gpu.sample_rows(lb, vocab, nodes, ub, tokens, 0.8, 0, 0.9, 0.01)
            gpu.tree_accept(pb, db, tokens, path, nodes)
            gpu.kv_commit([kb, vb], path, 4 * 128 * 4, start, cap, nodes)

        # a capture before any call: the scratch cannot grow, and the capture outlives the refusal
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        gpu.done()
        hip("hipStreamBeginCapture", stream, 2)
        gpu.tree_accept(pb, db, tokens, path, nodes)
        with pytest.raises(WgdError) as e:
            gpu.sample_rows(lb, vocab, nodes, ub, tokens, 0.8, 0, 0.9, 0.01)
        assert e.value.status == WGD_E_STATE
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphDestroy", graph)

        def state():
            return [gpu.read(b, s) for b, s in ((xb, q.nbytes), (y, q.nbytes), (tokens, 4 * nodes), (path, 4 * nodes + 8),
                                                (kb, k.nbytes), (vb, v.nbytes))]

        def reset(i):
            gpu.write(xb, q * (i + 1)); gpu.write(qb, q * (1 + 0.1 * i)); gpu.write(kb, k); gpu.write(vb, v)
            gpu.write(ub, np.random.default_rng(i).random(nodes)); gpu.write(tokens, np.zeros(nodes, np.int32))

        want = []
        for i in range(3):
            reset(i)
            step()
            want.append(state())
        gpu.done()
        hip("hipStreamBeginCapture", stream, 2)
        step()
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphInstantiate", ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0))
        for i in (0, 1, 2, 1, 0):
            reset(i)
            hip("hipGraphLaunch", exe, stream)
            assert state() == want[i]
            # larger work of the context between the replays: its scratch grows, the graph's block stays
            big = (rng.standard_normal((64 + 40 * i, vocab))).astype(np.float32)
            b2, u2, t2 = up(big), up(rng.random(len(big))), up(np.zeros(len(big), np.int32))
            gpu.sample_rows(b2, vocab, len(big), u2, t2, 1.0, 0, 0.9)
        hip("hipGraphExecDestroy", exe)
        hip("hipGraphDestroy", graph)
    finally:
        up.free()
        gpu.dispose()


# ------------------------------------------------------------------------------- refusals

def test_refusals(gpu, up):
    f, i32, f64 = (up(np.zeros(1 << 14, np.uint8)) for _ in range(3))
    y, y2 = up(np.zeros(1 << 14, np.uint8)), up(np.zeros(1 << 14, np.uint8))
    tiny = up(np.zeros(4, np.uint8))
    other = Compute().init()
    foreign = other.upload(np.zeros(1 << 14, np.uint8))
    A = lambda q=f, k=i32, v=f64, out=y, par=y2, heads=4, kvh=2, hd=16, start=8, window=64, cap=32, nodes=4: \
        gpu.attention_tree(q, k, v, out, par, heads, kvh, hd, start, 0.1, window, cap, nodes)  # noqa: E731
    R = lambda x=f, pos=i32, heads=2, hd=16, theta=1e4, rot=16, batch=3, **kw: gpu.rope_at(x, pos, heads, hd, theta, 1.0, rot, batch, **kw)  # noqa: E731
    S = lambda l=f, n=16, rows=3, u=f64, t=i32, T=0.5, k=4, p=0.9, m=0.1, **kw: gpu.sample_rows(l, n, rows, u, t, T, k, p, m, **kw)  # noqa: E731
    C = lambda rings, path=y, row=32, start=3, cap=16, nodes=4: gpu.kv_commit(rings, path, row, start, cap, nodes)  # noqa: E731
    P = lambda par=f, d=i32, pk=f64, path=y, nodes=4: gpu.tree_accept(par, d, pk, path, nodes)  # noqa: E731
    bad = [
        lambda: A(heads=3), lambda: A(heads=0), lambda: A(kvh=0), lambda: A(hd=0), lambda: A(hd=513), lambda: A(cap=0), lambda: A(window=0),
        lambda: A(nodes=257, cap=1000), lambda: A(start=2 ** 31), lambda: A(cap=11), lambda: A(window=5, cap=7), lambda: A(q=tiny),
        lambda: A(k=tiny), lambda: A(v=tiny), lambda: A(out=tiny), lambda: A(par=tiny), lambda: A(out=f), lambda: A(out=y2), lambda: A(k=foreign),
        lambda: A(par=foreign), lambda: A(nodes=33, cap=32, start=0), lambda: A(heads=2 ** 31, kvh=1),
        lambda: R(hd=15, rot=14), lambda: R(rot=18), lambda: R(rot=3), lambda: R(hd=0, rot=0), lambda: R(theta=0.0), lambda: R(theta=-1.0),
        lambda: R(theta=math.inf), lambda: R(theta=math.nan), lambda: R(stride=31), lambda: R(x=tiny), lambda: R(pos=tiny), lambda: R(offset=1 << 40),
        lambda: R(offset=4096 - 95), lambda: R(factors=tiny), lambda: R(pos=f), lambda: R(factors=f), lambda: R(heads=2 ** 31, hd=16),
        lambda: R(x=foreign), lambda: R(factors=foreign), lambda: R(batch=2 ** 31),
        lambda: S(n=0), lambda: S(n=2 ** 31), lambda: S(stride=15), lambda: S(T=-0.1), lambda: S(T=2.5), lambda: S(T=math.nan), lambda: S(p=0.0),
        lambda: S(p=1.1), lambda: S(p=math.nan), lambda: S(m=-0.1), lambda: S(m=1.1), lambda: S(m=math.nan), lambda: S(l=tiny), lambda: S(u=tiny),
        lambda: S(t=tiny), lambda: S(t=f), lambda: S(t=f64), lambda: S(u=foreign), lambda: S(rows=2 ** 32 - 1),
        lambda: P(nodes=0), lambda: P(nodes=257), lambda: P(par=tiny), lambda: P(d=tiny), lambda: P(pk=tiny), lambda: P(path=tiny), lambda: P(path=f),
        lambda: P(path=i32), lambda: P(path=f64), lambda: P(pk=foreign),
        lambda: C([f], nodes=0), lambda: C([f], nodes=17), lambda: C([f], row=0), lambda: C([f], row=3), lambda: C([f], cap=4096),
        lambda: C([f, f]), lambda: C([y]), lambda: C([foreign]), lambda: C([f], start=2 ** 31), lambda: C([tiny]), lambda: C([f], path=tiny),
    ]
    try:
        for i, call in enumerate(bad):
            with pytest.raises(WgdError) as e:
                call()
            assert e.value.status == WGD_E_INVALID, i
        # nothing to do is no error
        A(nodes=0)
        R(batch=0)
        R(heads=0)
        S(rows=0)
        C([])
        for call in (A, R, S, P):
            call()
        C([f, f64])
        gpu.done()
        assert gpu.address(f) and gpu.address(f) != gpu.address(y)
    finally:
        other.dispose()


# ------------------------------------------------------------------------------- paths of the launchers

@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("case", [
    # several row groups in a workgroup, the last ones without rows; several splits
    (32, 16, 128, 45, 1071, 1024, 0), (8, 2, 256, 35, 700, NO_WINDOW, 3), (4, 4, 64, 250, 900, NO_WINDOW, 0), (5, 1, 128, 61, 2500, NO_WINDOW, 0),
    (6, 3, 72, 50, 1500, 800, 1),
], ids=lambda c: "-".join("w" if v == NO_WINDOW else str(v) for v in c))
def test_attention_tree_row_groups(gpu, up, case, kv):
    test_attention_tree(gpu, up, case, kv)


@pytest.mark.parametrize("hd,heads,nodes,start", [(128, 7, 64, 3000), (64, 16, 70, 2000), (256, 8, 33, 2500)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_attention_tree_of_many_rows_keeps_masked_places_out(gpu, up, hd, heads, nodes, start, bad):
    rng = np.random.default_rng(hd + nodes)
    q, k, v, cap = tree_case(rng, heads, 1, hd, nodes, start, NO_WINDOW, 4, "f16")
    parents = random_tree(rng, nodes)
    hit = nodes // 2
    free = [i for i, p in enumerate(tree_ref.paths(parents)) if hit not in p]
    assert 0 < len(free) < nodes
    slot = (start + hit) % cap
    k[slot], v[slot] = 0, 0
    want = tree_ref.attention(q, k, v, parents, start, 1 / math.sqrt(hd), NO_WINDOW)
    k[slot], v[slot] = bad, bad
    unused = [(start + nodes + e) % cap for e in range(4)]
    k[unused], v[unused] = bad, bad
    got = run_tree(gpu, up, q, k, v, parents, start, 1 / math.sqrt(hd), NO_WINDOW)
    # |score| <= S: its error is (hd + 4) eps S on either side, a sum of n weights adds (n + 8) eps
    S = float(np.abs(q).max() * np.abs(k[np.isfinite(k)]).max()) * math.sqrt(hd)
    bound = (2 * (hd + 4) * EPS * S + 2 * (start + nodes + 8) * EPS) * float(np.abs(v[np.isfinite(v)]).astype(np.float64).max())
    assert np.isfinite(got[free]).all() and np.abs(got[free] - want[free]).max() <= bound
    assert not np.isfinite(got[hit]).any()


@pytest.mark.parametrize("rows,n,stride", [(300, 5003, 5011), (3, 70001, 70004), (1, 140000, 140000), (40, 33000, 33000)])
@pytest.mark.parametrize("settings", [(0.9, 0, 0.9, 0.01), (1.3, 600, 0.95, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 300, 1.0, 0.0)])
def test_sample_rows_of_different_rows(gpu, up, rows, n, stride, settings):
    rng = np.random.default_rng(rows + n)
    logits = (rng.standard_normal((rows, stride)) * rng.uniform(0.1, 5, (rows, 1))).astype(np.float32)
    logits[:, n:] = 1e9  # beyond the row
    logits[rng.integers(0, rows, 50), rng.integers(0, n, 50)] = np.nan
    logits[rng.integers(0, rows, 50), rng.integers(0, n, 50)] = -np.inf
    if rows > 2:
        logits[1, :n] = -np.inf
        logits[2, :n] = np.round(logits[2, :n])
    us = rng.random(rows)
    got = draw_rows(gpu, up, logits, us, *settings, stride=(n,))
    for i in range(rows):
        assert got[i] in tree_ref.draw(logits[i, :n], us[i], *settings), i
    assert got == draw_rows(gpu, up, logits, us, *settings, stride=(n,))


def test_kv_commit_refuses_more_rings_than_a_call_takes(gpu, up):
    ring, path = up(np.zeros(512, np.uint8)), up(np.zeros(64, np.uint8))
    with pytest.raises(WgdError) as e:
        gpu.kv_commit([ring] * 65537, path, 32, 3, 16, 4)
    assert e.value.status == WGD_E_INVALID
