"""Attention over pages at the ends of what its arguments can say: ranges of keys on more pages than a workgroup holds the
numbers of, and prefixes of more threads than a launch takes, and what a call allocates. The sizes of the ranges are worked out here as the launch's plan does, and
asserted."""
import math

import numpy as np
import pytest

from tests import pages_ref as ref
from tests.test_attention_pages_gpu import Batch, NO_WINDOW
from tests.test_pages_gpu import Held, i32, read, up  # noqa: F401
from webgpu_amd.gpu import Compute

pytestmark = pytest.mark.gpu
CUS, IDS = 256, 1024  # page numbers that a workgroup holds at a time


class Thin(Batch):
    """Requests whose tables name the same few pages again and again, so that long ones need little memory."""

    def __init__(self, rng, heads, kvh, hd, page, lengths, tokens=1, counts=None, kv="f32", pages=97):
        super().__init__(rng, heads, kvh, hd, page, [pages * page], tokens, None, kv=kv, spare=0)
        self.lengths, self.counts = i32(lengths), None if counts is None else i32(counts)
        self.table = rng.integers(0, self.pages, (len(lengths), max(ref.held(n, page) for n in lengths))).astype(np.int32)
        self.q = rng.standard_normal((len(lengths), tokens, heads, hd)).astype(np.float32)

    def want(self, scale, window=NO_WINDOW):
        """tests/pages_ref.py's formula, the queries of a request and kv head at once."""
        y = np.zeros(self.q.shape)
        page, kvh, hd = self.k.shape[1:]
        group = self.heads // kvh
        for r, n in enumerate(self.lengths):
            asked = min(int(n), self.tokens if self.counts is None else max(0, min(int(self.counts[r]), self.tokens)))
            if not asked:
                continue
            j = np.arange(n)
            ids = self.table[r, j // page]
            on = (ids >= 0) & (ids < self.pages)
            pos = int(n) - asked + np.arange(asked)[:, None]
            sees = ((j <= pos) & (j > pos - window) & on)[:, None]
            at = np.where(on, ids, 0), j % page
            for h in range(kvh):
                k, v = (m[at[0], at[1], h].astype(np.float64) for m in (self.k, self.v))
                s = self.q[r, :asked, h * group:(h + 1) * group].astype(np.float64) @ k.T * scale
                s = np.where(sees, s, -np.inf)
                top = s.max(-1, keepdims=True)
                p = np.where(sees, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                total = p.sum(-1, keepdims=True)
                y[r, :asked, h * group:(h + 1) * group] = p @ v / np.where(total > 0, total, 1)
        return y


def longest_range(b, unit, target):
    """Pages of the longest range of keys of a workgroup: chunks of whole units, as many as `target` makes of the batch."""
    units = [ref.held(int(n), unit) for n in b.lengths]
    chunk = math.ceil(sum(units) / target)
    return max(ref.held(ref.held(u, ref.held(u, chunk)) * unit if u > chunk else int(n), b.page) for u, n in zip(units, b.lengths))


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("page,lengths", [(1, [2500, 1025, 1024, 1, 0, 3100, 2049, 700] * 4), (2, [5000, 4097, 3, 2100] * 8)])
@pytest.mark.parametrize("hd", [8, 64, 20])
def test_direct_ranges_of_more_pages_than_are_held(gpu, up, hd, page, lengths, kv):  # noqa: F811
    rng = np.random.default_rng(page + hd)
    b = Thin(rng, 32, 32, hd, page, lengths, kv=kv)
    # one row of a kv head: 32 workgroups a chunk, four a CU (head dims of no multiple of 8: tiles of keys that fit 50000 bytes)
    unit = (32 if kv == "f16" else 16) * 4 if hd % 8 == 0 else 64
    assert longest_range(b, unit, 4 * CUS // 32) > IDS
    b.check(b.run(gpu, up, 0.3), 0.3)
    for window in (1100, 40):
        b.check(b.run(gpu, up, 0.3, window), 0.3, window)
    # pages that are none, the first of them behind those that are held first
    kept = b.table.copy()
    b.table[0, 1030], b.table[1, b.table.shape[1] - 5], b.table[5 % len(lengths), 1500] = -1, 2 ** 31 - 1, b.pages
    b.check(b.run(gpu, up, 0.3), 0.3)
    b.table[0, 7] = -2
    b.check(b.run(gpu, up, 0.3), 0.3)
    # a value that is not finite there, which all see
    b.table = kept
    b.v[int(b.table[0, 1040]), 0, 3, hd - 1] = np.inf
    got, want = b.run(gpu, up, 0.3), b.want(0.3)
    assert np.array_equal(np.isinf(got), np.isinf(want)) and not np.isnan(got).any()
    fine = np.isfinite(want)
    assert np.abs(got[fine] - want[fine]).max() <= b.bound(0.3)[2]


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_staged_ranges_of_more_pages_than_are_held(gpu, up, hd):  # noqa: F811
    rng = np.random.default_rng(hd)
    heads, tokens = 64, 128
    lengths, counts = [2300, 1100, 700, 40], [128, 127, 100, 40]
    b = Thin(rng, heads, heads, hd, 1, lengths, tokens, counts, kv="f16")
    rows = 64 if hd == 256 else 128
    wgs = heads * tokens // rows
    at_once = CUS // wgs
    target = at_once - 2 if len(lengths) <= at_once else max(1, 2 * CUS // wgs)
    assert longest_range(b, 128, target) > IDS
    scale = 1 / math.sqrt(hd)
    b.check(b.run(gpu, up, scale), scale)
    b.check(b.run(gpu, up, scale, 1200), scale, 1200)
    b.table[0, 1100], b.table[1, 1090] = -1, b.pages
    b.check(b.run(gpu, up, scale), scale)
    b.table[2, 3] = -7
    b.check(b.run(gpu, up, scale, 1200), scale, 1200)


@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_a_prefix_of_more_threads_than_a_launch_takes(gpu, up, kv):  # noqa: F811
    """2^20 kv heads over a prefix of 16368 pages: parts of fewer than 1024 page numbers would be more than 2^32 threads along x. The
    prefix is one page again and again, computed apart; the pages behind it hold other values."""
    heads, hd, shared, tail = 1 << 20, 8, 16368, 3
    kind, half = (np.float16, True) if kv == "f16" else (np.float32, False)
    values = np.arange(1, 4, dtype=kind)[:, None] * np.ones(heads * hd, kind)  # page p holds p + 1
    table = np.zeros((2, shared + tail), np.int32)
    table[:, shared:] = [[1], [2]]
    lengths = i32([shared + 1, shared + tail])
    held = [gpu.buffer(n) for n in (2 * heads * hd * 4, values.nbytes, 2 * heads * hd * 4)]  # zero queries and keys: equal weights
    try:
        q, k, y = held
        for owner in (0, 1):
            (gpu.attention_pages_f16kv if half else gpu.attention_pages)(q, k, up(values), y, up(table), up(lengths), heads, heads, hd, 1.0, NO_WINDOW, 1,
                                                                         shared + tail, 3, 2, shared=shared, owner=owner)
            got = read(gpu, y, (2, heads * hd), np.float32)
            want = np.array([(shared + 2) / (shared + 1), (shared + 3 * tail) / (shared + tail)])
            # equal weights: their sums are whole numbers in f32, the values' products with them and the quotient round
            assert np.abs(got - want[:, None]).max() <= 4 * 2.0 ** -24 * want.max()
    finally:
        for b in held:
            gpu.destroy(b)


@pytest.mark.parametrize("kv,heads,hd,tokens,lengths,mib", [("f32", 128, 8, 512, [512], 10), ("f16", 128, 8, 320, [330, 17, 320, 0], 14), ("f16", 32, 64, 1024, [1024], 26),
                                                            ("f32", 128, 20, 100, [160, 90, 130], 16)])
def test_prompts_that_are_not_cut_need_no_scratch(kv, heads, hd, tokens, lengths, mib):
    """So many blocks of rows that one chunk for each request is all that is wanted: nothing is kept for a join, and a budget that has room
    for the buffers alone suffices."""
    gpu = Compute(mib).init()
    up = Held(gpu)  # noqa: F811
    try:
        b = Batch(np.random.default_rng(tokens), heads, heads, hd, 16, lengths, tokens, kv=kv)
        before = gpu.allocated
        got = b.run(gpu, up, 0.2)
        assert gpu.allocated - before == sum(x.size for x in up.held)
        b.check(got, 0.2)
    finally:
        up.free()
        gpu.dispose()


def test_lengths_that_are_none(gpu, up):  # noqa: F811
    """extend refuses such requests whatever their count, fork and attention take the nearest end."""
    page, width, pages = 4, 3, 12
    table = i32(np.arange(12).reshape(4, 3))
    lengths, refs = i32([-1, 13, -2 ** 31, 2 ** 31 - 1]), i32([0, 0, 0, 1, 1, 1, 0, 0, 0, 1, 1, 1])
    b = [up(x) for x in (table, lengths, refs)]
    outs = [up(np.full(n, 77, np.int32)) for n in (4, 8, 8)]
    for counts in ([0] * 4, [1, 0, 2, 1]):
        gpu.pages_extend(*b, *outs, 4, 2, page, width, pages, counts=up(i32(counts)))
        for x, want in zip(b + outs, (table, lengths, refs, i32([-1] * 4), i32([-1] * 8), i32([-1] * 8))):
            assert np.array_equal(read(gpu, x, want.shape), want)
    copies = up(np.zeros(9, np.int32))
    gpu.pages_fork(*b, up(i32([0, 0, 3, 3])), copies, 4, page, width, pages)
    t, n, c, pairs = ref.fork(table, lengths, refs, [0, 0, 3, 3], None, page)
    assert n.tolist() == [-1, 0, 12, 2 ** 31 - 1] and pairs == []
    for x, want in zip(b, (t, n, c)):
        assert np.array_equal(read(gpu, x, want.shape), want)
