"""Attention of batches over pages on the MI355X against float64, and steps of a batch with the operators around it.

Tolerance, with e = 2^-24 (half a step of f32), as for single sequences: the f32 dot product of hd terms is off by at most
hd e sum|q k|, so a weight by twice that and by its own rounding; numerator and denominator are sums of n weights, n e each at most:
|y - want| <= (2 (hd + 4) e S + 2 (n + 8) e) max|v| with S = scale max sum|q k|. The bound is for the worst signs: roundings are
independent, so the 2-norm of the difference is held to 16 e sqrt(hd + n) times the 2-norm of the result as well, with at least 1 for
sqrt(S) beside it.
"""
import ctypes
import math

import numpy as np
import pytest

from tests import pages_ref as ref
from tests import tree_ref
from tests.test_pages_gpu import Held, Hip, i32, read, up  # noqa: F401
from webgpu_amd.gpu import Compute, WgdError, WGD_E_INVALID, WGD_E_STATE

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
NO_WINDOW = 1 << 30


class Batch:
    """A batch of random requests, `shared` tokens of which those of `sharers` have in common with the first of them."""

    def __init__(self, rng, heads, kvh, hd, page, lengths, tokens=1, counts=None, shared=0, sharers=(), kv="f32", spare=2, qk=1.0):
        self.heads, self.shared, self.tokens, self.page = heads, shared, tokens, page
        self.lengths, self.counts = i32(lengths), None if counts is None else i32(counts)
        R = len(lengths)
        held = [ref.held(max(0, n), page) for n in lengths]
        width, first = max(held + [1]) + spare, shared // page
        self.pages = int(sum(held)) + first + spare
        order = rng.permutation(self.pages).tolist()
        self.table = rng.integers(-9, self.pages + 9, (R, width)).astype(np.int32)  # what lies behind a request is no page of its own
        common = [order.pop() for _ in range(first)]
        for r in range(R):
            ids = common if r in sharers else []
            ids = (ids + [order.pop() for _ in range(held[r] - len(ids))])[:held[r]]
            self.table[r, :held[r]] = ids
        self.q = (rng.standard_normal((R, tokens, heads, hd)) * qk).astype(np.float32)
        self.k, self.v = (rng.standard_normal((self.pages, page, kvh, hd)).astype(np.float16 if kv == "f16" else np.float32) for _ in range(2))

    def want(self, scale, window=NO_WINDOW):
        return ref.attention(self.q, self.k, self.v, self.table, self.lengths, self.counts, scale, window)

    def run(self, gpu, up, scale, window=NO_WINDOW, shared=None, owner=0):  # noqa: F811
        y = up(np.full(self.q.size + 5, 77.0, np.float32))
        (gpu.attention_pages_f16kv if self.k.dtype == np.float16 else gpu.attention_pages)(
            up(self.q), up(self.k), up(self.v), y, up(self.table), up(self.lengths), self.heads, self.k.shape[2], self.k.shape[3], scale, window,
            self.page, self.table.shape[1], self.pages, len(self.lengths), self.tokens, counts=None if self.counts is None else up(self.counts),
            shared=self.shared if shared is None else shared, owner=owner)
        got = read(gpu, y, self.q.size + 5, np.float32)
        assert np.all(got[self.q.size:] == 77.0)
        return got[:self.q.size].reshape(self.q.shape)

    def bound(self, scale, window=NO_WINDOW):
        hd = self.q.shape[3]
        q, k, v = (np.abs(np.where(np.isfinite(x), x, 0)).astype(np.float64) for x in (self.q, self.k, self.v))
        S = scale * math.sqrt((q ** 2).sum(-1).max() * (k ** 2).sum(-1).max())
        n = min(int(max(self.lengths.max(), 1)), window)
        return S, n, (2 * (hd + 4) * EPS * S + 2 * (n + 8) * EPS) * float(v.max())

    def check(self, got, scale, window=NO_WINDOW):
        want = self.want(scale, window)
        S, n, bound = self.bound(scale, window)
        assert np.isfinite(got).all()
        assert np.abs(got - want).max() <= bound, (np.abs(got - want).max(), bound)
        assert np.linalg.norm(got - want) <= 16 * EPS * math.sqrt(self.q.shape[3] + n) * max(1, math.sqrt(S)) * np.linalg.norm(want)
        assert np.all(got[np.all(want == 0, -1)] == 0)


CASES = [
    # heads, kv_heads, head_dim, page, lengths, tokens, window
    (1, 1, 1, 1, [1], 1, NO_WINDOW), (4, 2, 8, 4, [0, 1, 3, 4, 5], 1, NO_WINDOW), (2, 1, 64, 16, [0], 1, NO_WINDOW), (16, 8, 128, 16, [300, 7, 64, 65], 1, NO_WINDOW),
    (32, 8, 128, 32, [517, 1, 0, 1200, 33], 1, NO_WINDOW), (8, 8, 128, 1, [63, 130], 1, NO_WINDOW), (14, 2, 64, 2, [200, 31, 32], 1, NO_WINDOW),
    (3, 1, 128, 64, [1000], 1, NO_WINDOW), (20, 1, 64, 8, [130, 5000], 1, NO_WINDOW), (34, 2, 128, 128, [40, 600], 1, NO_WINDOW),
    (4, 2, 256, 16, [100, 700, 3], 1, NO_WINDOW), (8, 4, 80, 16, [90, 333], 1, NO_WINDOW), (6, 2, 96, 4, [33, 2100], 1, NO_WINDOW), (2, 1, 17, 16, [50, 9], 1, NO_WINDOW),
    (2, 2, 512, 16, [70, 20], 1, NO_WINDOW), (4, 2, 128, 1024, [1500, 1024, 1025], 1, NO_WINDOW), (8, 2, 128, 16, [500, 90, 3], 1, 50), (8, 2, 64, 8, [500, 90, 3], 1, 1),
    (8, 2, 128, 16, [500, 90, 3], 5, NO_WINDOW), (8, 2, 128, 16, [500, 90, 3, 0], 7, 40), (4, 4, 64, 4, [40, 41], 33, NO_WINDOW), (8, 1, 128, 32, [300, 800], 40, NO_WINDOW),
    (32, 8, 128, 16, [700, 100], 64, NO_WINDOW), (4, 2, 256, 64, [260, 129], 70, 100), (8, 2, 80, 16, [300, 50], 17, NO_WINDOW), (6, 3, 40, 2, [90, 30], 21, 25),
    (16, 2, 128, 16, [2000], 128, NO_WINDOW), (16, 2, 64, 16, [3000, 200], 90, 1000), (2, 2, 128, 32, [64] * 70, 1, NO_WINDOW), (4, 1, 64, 8, list(range(0, 140)), 2, NO_WINDOW),
    (1, 1, 64, 16, [20000], 1, NO_WINDOW), (2, 1, 128, 16, [9000, 1, 4000], 1, 8000), (24, 8, 64, 16, [300, 77], 1, NO_WINDOW), (7, 1, 72, 16, [300, 77], 3, NO_WINDOW),
]


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) if not isinstance(v, list) else "%dx%d" % (len(v), max(v)) for v in c))
def test_attention_pages(gpu, up, case, kv):  # noqa: F811
    heads, kvh, hd, page, lengths, tokens, window = case
    rng = np.random.default_rng(heads * 1000 + hd + len(lengths))
    counts = None if tokens == 1 and len(lengths) % 2 else rng.integers(-1, tokens + 2, len(lengths))
    if counts is not None:
        counts[0] = tokens
    b = Batch(rng, heads, kvh, hd, page, lengths, tokens, counts, kv=kv)
    b.check(b.run(gpu, up, 1 / math.sqrt(hd), window), 1 / math.sqrt(hd), window)


PREFIXES = [
    # heads, kv_heads, head_dim, page, shared, lengths behind it, tokens, sharers of them
    (8, 2, 128, 16, 64, [1, 5, 30], 1, 3), (32, 8, 128, 32, 1024, [1] * 20, 1, 20), (16, 8, 128, 16, 512, [40, 3, 700, 9], 1, 2), (4, 4, 64, 8, 8, [1, 1], 1, 2),
    (8, 1, 256, 64, 2048, [10, 200, 1], 1, 3), (6, 2, 80, 16, 320, [7, 9, 11], 2, 3), (8, 2, 128, 16, 3200, list(range(1, 41)), 1, 38), (4, 2, 17, 4, 40, [3, 8], 3, 2),
    (8, 2, 128, 16, 640, [20, 30, 40, 50], 16, 4), (8, 1, 64, 2, 514, [1] * 130, 1, 130), (4, 1, 128, 1, 300, [2, 1, 5], 1, 3), (32, 8, 128, 64, 4096, [5] * 9, 9, 8),
    (2, 2, 512, 16, 64, [3, 4], 1, 2), (8, 2, 128, 16, 64, [1, 5, 30], 1, 1), (16, 1, 128, 16, 6400, [30, 4] * 40, 1, 80),
]


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("case", PREFIXES, ids=lambda c: "-".join(str(v) if not isinstance(v, list) else "%dx%d" % (len(v), max(v)) for v in c))
def test_attention_pages_with_a_shared_prefix(gpu, up, case, kv):  # noqa: F811
    heads, kvh, hd, page, shared, behind, tokens, n = case
    rng = np.random.default_rng(shared + len(behind))
    scale = 1 / math.sqrt(hd)
    lengths = [shared + x for x in behind]
    counts = np.minimum(rng.integers(0, tokens + 1, len(behind)), behind)
    counts[:2] = np.minimum(tokens, behind[:2])
    b = Batch(rng, heads, kvh, hd, page, lengths, tokens, counts, shared, range(n), kv)
    got = b.run(gpu, up, scale)
    b.check(got, scale)
    assert np.array_equal(got, b.run(gpu, up, scale))
    b.check(b.run(gpu, up, scale, owner=n - 1), scale)
    # a window that hides a part of the prefix, or of all but it
    for window in (shared + 1, max(1, shared // 2)):
        b.check(b.run(gpu, up, scale, window), scale, window)
    # requests that have less than the prefix or no new token, an owner without one, and one that is too short
    b.lengths[-1], b.counts[0] = max(1, shared - 3), 0
    b.check(b.run(gpu, up, scale), scale)
    b.lengths[0] = max(0, shared - 1)
    b.check(b.run(gpu, up, scale), scale)


def test_attention_pages_shares_what_a_smaller_prefix_names(gpu, up):  # noqa: F811
    rng = np.random.default_rng(2)
    b = Batch(rng, 8, 2, 128, 16, [333, 340, 500], shared=320, sharers=range(3), kv="f16")
    for shared in (0, 16, 160, 320):
        b.check(b.run(gpu, up, 0.09, shared=shared), 0.09)
    for owner in (1, 2):
        b.check(b.run(gpu, up, 0.09, owner=owner), 0.09)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd,heads,kvh", [(128, 8, 2), (64, 4, 4), (256, 4, 2), (40, 2, 1)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_masked_places_reach_nothing(gpu, up, hd, heads, kvh, bad, kv):  # noqa: F811
    rng = np.random.default_rng(hd + 1)
    window, tokens = 64, 9
    b = Batch(rng, heads, kvh, hd, 16, [128 + 40, 128 + 21, 128 + 9], tokens, [9, 4, 1], 128, range(3), kv)
    b2 = Batch(rng, heads, kvh, hd, 16, [230, 77], tokens, [9, 4], kv=kv)
    for batch, win in ((b, NO_WINDOW), (b2, window)):
        clean = batch.run(gpu, up, 0.1, win)
        # slots behind a request's last token, and pages that nobody has
        seen = np.zeros((batch.pages, 16), bool)
        for r, n in enumerate(batch.lengths):
            for t in range(max(0, n - batch.counts[r] + 1 - win), n):
                seen[batch.table[r, t // 16], t % 16] = True
        k, v = batch.k.copy(), batch.v.copy()
        batch.k[~seen], batch.v[~seen] = bad, bad
        assert np.array_equal(batch.run(gpu, up, 0.1, win), clean)
        batch.k, batch.v = k, v
        # a key that only later queries of the request see, in K or in V
        n = int(batch.lengths[0])
        for which in "kv":
            data = getattr(batch, which)
            kept = data.copy()
            data[batch.table[0, (n - 3) // 16], (n - 3) % 16, :, hd // 2] = bad
            got, want = batch.run(gpu, up, 0.1, win), batch.want(0.1, win)
            hit = np.zeros(got.shape[:2], bool)
            hit[0, 6:9] = True
            assert np.abs(got[~hit] - clean[~hit]).max() <= 1e-5  # formed another way beside such values, to the same accuracy
            assert np.array_equal(np.isnan(got[hit]), np.isnan(want[hit]))
            inf = np.isinf(want[hit])
            assert np.array_equal(got[hit][inf], want[hit][inf])
            fine = np.isfinite(want[hit])
            assert np.allclose(got[hit][fine], want[hit][fine], rtol=0, atol=1e-3)
            setattr(batch, which, kept)
        # a query that is not finite spoils its own row alone
        q = batch.q.copy()
        batch.q[0, 5, heads - 1, 0] = bad
        batch.q[1, 5:] = bad  # no query of the request
        got = batch.run(gpu, up, 0.1, win)
        assert not np.isfinite(got[0, 5, heads - 1]).any()
        got[0, 5, heads - 1] = clean[0, 5, heads - 1]
        assert np.abs(got - clean).max() <= 1e-5
        batch.q = q


@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_pages_that_are_none_are_not_seen(gpu, up, kv):  # noqa: F811
    rng = np.random.default_rng(6)
    for hd in (128, 48):
        b = Batch(rng, 8, 2, hd, 16, [700, 90, 33, 16, 40], 3, [3, 3, 1, 2, 3], kv=kv)
        b.table[0, 5], b.table[0, 43], b.table[1, 2], b.table[2, :3], b.table[3, 0], b.table[4, 2] = b.pages, -1, -2 ** 31, -5, 2 ** 31 - 1, -1
        got = b.run(gpu, up, 0.1)
        b.check(got, 0.1)
        assert np.all(got[2:4] == 0)
        b = Batch(rng, 8, 2, hd, 16, [330, 323], shared=320, sharers=(0, 1), kv=kv)
        b.table[:, 7] = b.pages + 3  # in the prefix
        b.check(b.run(gpu, up, 0.1), 0.1)
        b.table[:, 19] = -1  # its last column
        b.check(b.run(gpu, up, 0.1), 0.1)
    # a column of the prefix that is none in tables that have nothing else in common
    b = Batch(rng, 8, 2, 128, 16, [330, 323], kv=kv)
    b.table[:, 19] = -1
    b.check(b.run(gpu, up, 0.1, shared=320), 0.1)


def test_lengths_beyond_the_table_count_as_its_end(gpu, up):  # noqa: F811
    rng = np.random.default_rng(7)
    b = Batch(rng, 4, 2, 64, 8, [40, 40, 40], spare=0)
    b.lengths = i32([41, -3, 2 ** 31 - 1])
    got = b.run(gpu, up, 0.1)
    b.check(got, 0.1)
    assert np.all(got[1] == 0) and not np.all(got[2] == 0)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 48])
@pytest.mark.parametrize("scale_of", [1e-6, 30.0, 0.0])
def test_magnitudes(gpu, up, hd, kv, scale_of):  # noqa: F811
    """Scores of one key, all alike, and zero; queries, keys and values of other sizes than 1."""
    rng = np.random.default_rng(hd)
    b = Batch(rng, 4, 2, hd, 16, [310, 130, 140], 4, [4, 2, 1], 128, range(3), kv, qk=scale_of)
    b.v = (b.v.astype(np.float32) * (200 if kv == "f16" else 1e6)).astype(b.v.dtype)
    b.k = (b.k.astype(np.float32) * 0.01).astype(b.k.dtype)
    b.check(b.run(gpu, up, 3.0), 3.0)


def test_offsets_pass_32_bits(gpu, up):  # noqa: F811
    """Pages behind 2^32 bytes (and 2^31 elements) of a pool, for own pages and a shared prefix."""
    kvh, hd, page, pages = 16, 128, 16, (1 << 16) + 90
    big = gpu.buffer(pages * page * kvh * hd * 2, "large pool")
    try:
        rng = np.random.default_rng(8)
        b = Batch(rng, 16, kvh, hd, page, [333, 322], shared=320, sharers=(0, 1), kv="f16", spare=0)
        b.v = b.k
        for p in range(b.pages):
            gpu.write(big, b.k[p], (pages - b.pages + p) * page * kvh * hd * 2)
        y = up(np.zeros(b.q.size, np.float32))
        for shared in (0, 320):
            gpu.attention_pages_f16kv(up(b.q), big, big, y, up(b.table + i32(pages - b.pages)), up(b.lengths), 16, kvh, hd, 0.1, NO_WINDOW, page,
                                      b.table.shape[1], pages, 2, shared=shared)
            b.check(read(gpu, y, b.q.shape, np.float32), 0.1)
    finally:
        gpu.destroy(big)


@pytest.mark.parametrize("tokens", [1360, 1400])
def test_millions_of_rows_of_one_kv_head(gpu, up, tokens):  # noqa: F811
    """Rows of a shared prefix up to what a launch takes (65535 blocks of 64) and beyond. Zero queries weigh all their keys alike: with V 0 in
    the prefix and r + 1 in the request's own tokens, query t of request r gives (t + 1) (r + 1) / (16 + t + 1)."""
    R, heads, hd, page = 1024, 3, 8, 16
    own = ref.held(tokens, page)
    pages = 1 + R * own
    table = np.concatenate([np.zeros((R, 1)), 1 + np.arange(R * own).reshape(R, own)], 1).astype(np.int32)
    v = np.repeat(np.concatenate([[0], 1 + np.arange(R * own) // own]), page * hd).astype(np.float32)
    q, y = gpu.buffer(R * tokens * heads * hd * 4), gpu.buffer(R * tokens * heads * hd * 4)
    try:
        gpu.attention_pages(q, up(np.zeros_like(v)), up(v), y, up(table), up(np.full(R, 16 + tokens, np.int32)), heads, 1, hd, 0.3, NO_WINDOW, page,
                            own + 1, pages, R, tokens, shared=16)
        got = read(gpu, y, (R, tokens, heads * hd), np.float32)
    finally:
        gpu.destroy(q)
        gpu.destroy(y)
    t, r = np.arange(tokens)[None] + 1.0, np.arange(R)[:, None] + 1.0
    want = t * r / (16 + t)
    # equal weights: their sums are whole numbers in f32, the products and the quotient round
    assert np.abs(got - want[..., None]).max() <= (tokens + 16 + 8) * EPS * R


def test_many_requests_repeat_themselves_and_two_contexts_agree(gpu, up):  # noqa: F811
    rng = np.random.default_rng(12)
    b = Batch(rng, 8, 2, 64, 16, rng.integers(0, 300, 1024), counts=rng.integers(0, 2, 1024), kv="f16")
    first = b.run(gpu, up, 0.1)
    b.check(first, 0.1)
    assert np.array_equal(first, b.run(gpu, up, 0.1))
    other = Compute().init()
    try:
        h = Held(other)
        assert np.array_equal(first, b.run(other, h, 0.1))
        h.free()
    finally:
        other.dispose()


# ------------------------------------------------------------------------------- steps of a batch

@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_a_batch_agrees_with_each_request_alone(gpu, up, kv):  # noqa: F811
    """Prompts in chunks, decoded tokens, a fork, a rollback and a compaction, with adapters beside a shared projection:
    every step's attention is that of the request alone over a ring, by the operators for one sequence."""
    rng = np.random.default_rng(20)
    R, heads, kvh, hd, page, width, pages, hidden, rank = 5, 8, 2, 64, 8, 12, 40, 96, 4
    row, qkv = kvh * hd, heads * hd + 2 * kvh * hd
    half = kv == "f16"
    z = lambda n, kind=np.int32: up(np.zeros(n, kind))  # noqa: E731
    table, lengths, refs, table_to, moved = z(R * width), z(R), z(pages), z(R * width), z(pages)
    k, v = (z(pages * page * row, np.float16 if half else np.float32) for _ in range(2))
    W = (rng.standard_normal((qkv, hidden)) / math.sqrt(hidden)).astype(np.float32)
    a = (rng.standard_normal((3, rank, hidden)) / math.sqrt(hidden)).astype(np.float32)
    bb = (rng.standard_normal((3, qkv, rank)) / math.sqrt(rank)).astype(np.float32)
    which, scales = np.array([0, 2, -1, 1, 0]), np.array([0.5, 1.0, 2.0], np.float32)
    Wb, ab, bbb, sb = up(W), up(a), up(bb), up(scales)
    tokens = [[] for _ in range(R)]  # every request's inputs so far
    adapters = which.copy()

    def project(x, w):  # one token in float32, as the f64 formula rounds
        y = W.astype(np.float64) @ x
        if w >= 0:
            y += float(scales[w]) * (bb[w].astype(np.float64) @ (a[w].astype(np.float64) @ x))
        return y.reshape(-1, hd)

    keys = [[] for _ in range(R)]  # rotated keys and values of every request, in float64

    def step(T, counts):
        x = rng.standard_normal((R * T, hidden)).astype(np.float32)
        added, positions, slots, y = z(R), z(R * T), z(R * T), z(R * T * qkv, np.float32)
        gpu.pages_extend(table, lengths, refs, added, positions, slots, R, T, page, width, pages, counts=up(i32(counts)))
        gpu.matmul(0, Wb, up(x), y, hidden, qkv, qkv, 0, 0, R * T)
        gpu.adapters(0, ab, bbb, up(i32(np.repeat(adapters, T))), sb, up(x), y, hidden, qkv, rank, 3, qkv, 0, R * T)
        gpu.rope_at(y, positions, heads + kvh, hd, 1e4, 1.0, 0, R * T, stride=qkv)
        (gpu.pages_store_f16kv if half else gpu.pages_store)(y, y, k, v, slots, row, R * T, pages * page, stride=qkv, k_offset=heads * hd,
                                                             v_offset=heads * hd + row)
        q = z(R * T * heads * hd, np.float32)
        for t in range(R * T):
            gpu.copy(y, q, heads * hd * 4, t * qkv * 4, t * heads * hd * 4)
        out = z(R * T * heads * hd, np.float32)
        (gpu.attention_pages_f16kv if half else gpu.attention_pages)(q, k, v, out, table, lengths, heads, kvh, hd, 0.125, NO_WINDOW, page, width, pages, R, T,
                                                                     counts=added)
        got = read(gpu, out, (R, T, heads, hd), np.float32)
        assert read(gpu, added, R).tolist() == list(counts)
        for r in range(R):
            for t in range(counts[r]):
                pos = len(keys[r])
                p = project(x[r * T + t].astype(np.float64), adapters[r])
                rot = tree_ref.rope(p[None, :heads + kvh], [pos], 1e4, 1.0, hd, False)[0]
                kk, vv = rot[heads:], p[heads + kvh:]
                keys[r].append((kk, vv))
                K, V = (np.stack([e[i] for e in keys[r]]) for i in range(2))
                if half:
                    K, V = (m.astype(np.float32).astype(np.float16).astype(np.float64) for m in (K, V))
                for h in range(heads):
                    s = K[:, h // (heads // kvh)] @ rot[h] * 0.125
                    w = np.exp(s - s.max())
                    want = w @ V[:, h // (heads // kvh)] / w.sum()
                    # f16 rings may round a value that lies next to a border the other way: one step of 2^-10 in 4
                    assert np.abs(got[r, t, h] - want).max() <= (2e-3 if half else 5e-5), (r, t, h)
            assert np.all(got[r, max(0, counts[r]):] == 0)

    def fork(origin, keep):
        copies = z(2 * R + 1)
        gpu.pages_fork(table, lengths, refs, up(i32(origin)), copies, R, page, width, pages, keep=up(i32(keep)))
        gpu.pages_copy([k, v], copies, R, page * row * (2 if half else 4), pages)
        assert read(gpu, copies, 1)[0] >= 0
        old = [list(e) for e in keys]
        for r in range(R):
            keys[r] = old[origin[r]][:keep[r]] if origin[r] >= 0 else []
            adapters[r] = which[origin[r]] if origin[r] >= 0 else which[r]

    step(17, [17, 3, 9, 0, 1])
    step(5, [5, 0, 1, 5, 2])
    step(1, [1, 1, 1, 1, 1])
    fork([0, 0, 2, -1, 0], [99, 21, 99, 0, 16])
    step(1, [1, 1, 1, 0, 1])
    step(6, [2, 6, 3, 6, 1])
    fork([0, 1, 2, 3, 4], [99, 22, 3, 99, 99])  # drafted tokens go back
    copies = z(pages // 2 * 2 + 1)
    gpu.pages_compact(table, refs, table, refs, moved, copies, R, width, pages)
    gpu.pages_copy([k, v], copies, pages // 2, page * row * (2 if half else 4), pages)
    n = read(gpu, refs, pages)
    assert np.all(n[:int((n > 0).sum())] > 0)
    step(4, [4, 3, 2, 1, 4])


def test_attention_pages_replay_in_a_graph():
    """Replays at lengths that grow, and after work between them that grows the context's scratch."""
    gpu = Compute().init()
    up = Held(gpu)  # noqa: F811
    hip, stream = Hip(), ctypes.c_void_p(gpu.stream)
    try:
        rng = np.random.default_rng(14)
        b = Batch(rng, 8, 2, 128, 16, [3200, 3300, 3230, 10], shared=3200 - 16, sharers=(0, 1, 2), kv="f16")
        bufs = [up(x) for x in (b.q, b.k, b.v, np.zeros_like(b.q), b.table, b.lengths)]
        call = lambda: gpu.attention_pages_f16kv(*bufs, 8, 2, 128, 0.09, NO_WINDOW, 16, b.table.shape[1], b.pages, 4, shared=b.shared)  # noqa: E731
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        gpu.done()
        hip("hipStreamBeginCapture", stream, 2)
        with pytest.raises(WgdError) as e:
            call()
        assert e.value.status == WGD_E_STATE
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphDestroy", graph)
        lengths = [b.lengths - i32([0, 0, 0, i]) for i in (9, 3, 0)] + [i32([3199, 0, 3230, 1])]
        want = []
        for n in lengths:
            gpu.write(bufs[5], n)
            call()
            want.append(gpu.read(bufs[3], b.q.nbytes))
        hip("hipStreamBeginCapture", stream, 2)
        call()
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphInstantiate", ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0))
        for i in (0, 1, 2, 3, 0):
            gpu.write(bufs[5], lengths[i])
            hip("hipGraphLaunch", exe, stream)
            assert gpu.read(bufs[3], b.q.nbytes) == want[i]
            more = Batch(rng, 8, 2, 64, 16, [200 + 900 * i] * 30, 2, kv="f16")
            more.run(gpu, up, 0.1)
        hip("hipGraphExecDestroy", exe)
        hip("hipGraphDestroy", graph)
    finally:
        up.free()
        gpu.dispose()


def test_refusals(gpu, up):  # noqa: F811
    f = [up(np.zeros(1 << 15, np.uint8)) for _ in range(7)]
    tiny = up(np.zeros(4, np.uint8))
    other = Compute().init()
    foreign = other.upload(np.zeros(1 << 15, np.uint8))
    A = lambda q=f[0], k=f[1], v=f[2], y=f[3], t=f[4], n=f[5], heads=4, kvh=2, hd=16, window=64, page=4, width=8, pages=32, R=3, T=2, **kw: \
        gpu.attention_pages(q, k, v, y, t, n, heads, kvh, hd, 0.1, window, page, width, pages, R, T, **kw)  # noqa: E731
    H = lambda pages=32, **kw: gpu.attention_pages_f16kv(f[0], f[1], f[2], f[3], f[4], f[5], 4, 2, 16, 0.1, 64, 4, 8, pages, 3, 2, **kw)  # noqa: E731
    bad = [lambda: A(heads=3), lambda: A(heads=0), lambda: A(kvh=0), lambda: A(hd=0), lambda: A(hd=513), lambda: A(window=0), lambda: A(page=0),
           lambda: A(page=24), lambda: A(page=2048), lambda: A(width=0), lambda: A(pages=0), lambda: A(R=1025), lambda: A(T=0), lambda: A(T=2 ** 20 + 1, R=1),
           lambda: A(heads=2 ** 21, kvh=1), lambda: A(heads=2 ** 20, kvh=2, T=32), lambda: A(heads=2 ** 20, kvh=1, T=2, R=1), lambda: A(width=2 ** 29),
           lambda: A(pages=2 ** 29), lambda: A(pages=65), lambda: H(pages=129), lambda: A(q=tiny), lambda: A(k=tiny), lambda: A(v=tiny), lambda: A(y=tiny),
           lambda: A(t=tiny), lambda: A(n=tiny), lambda: A(counts=tiny), lambda: A(y=f[0]), lambda: A(y=f[1]), lambda: A(y=f[4]), lambda: A(y=f[5]),
           lambda: A(counts=f[3]), lambda: A(q=foreign), lambda: A(t=foreign), lambda: A(counts=foreign), lambda: A(shared=2), lambda: A(shared=36),
           lambda: A(shared=4, owner=3), lambda: H(shared=6), lambda: A(R=1024, T=64), lambda: A(T=86)]
    try:
        for i, call in enumerate(bad):
            with pytest.raises(WgdError) as e:
                call()
            assert e.value.status == WGD_E_INVALID, i
        A(R=0)
        A()
        H(pages=128)
        A(counts=f[6], shared=32, owner=2)
        A(k=f[1], v=f[1], q=f[1])
        gpu.done()
    finally:
        other.dispose()
