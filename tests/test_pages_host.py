"""The plain forms of tests/pages_ref.py against a cache that keeps every request's tokens as a list: whatever a batch
extends, forks, drops and compacts, the pages hold each request's tokens, nobody writes into shared ones, and the
counts are those of the table."""
import numpy as np
import pytest

from tests import pages_ref as ref


class Cache:
    """Tokens with their values in a pool, driven by the plain forms, and lists beside it."""

    def __init__(self, R, width, page, pages):
        self.page, self.pages = page, pages
        self.table, self.lengths, self.refs = np.zeros((R, width), np.int32), np.zeros(R, np.int32), np.zeros(pages, np.int32)
        self.pool = np.full((pages, page), -1)
        self.lists = [[] for _ in range(R)]
        self.next = 0

    def extend(self, counts, tokens):
        self.table, self.lengths, self.refs, added, positions, slots = ref.extend(self.table, self.lengths, self.refs, counts, tokens, self.page)
        for r, n in enumerate(added):
            for t in range(max(0, n)):
                assert positions[r, t] == len(self.lists[r])
                self.lists[r].append(self.next)
                self.pool.ravel()[slots[r, t]] = self.next
                self.next += 1
            assert np.all(slots[r, max(0, n):] == -1) and np.all(positions[r, max(0, n):] == -1)
        return added

    def fork(self, origin, keep):
        out = ref.fork(self.table, self.lengths, self.refs, origin, keep, self.page)
        self.table, self.lengths, self.refs, pairs = out
        if pairs is not None:
            self.copy(pairs)
            old = self.lists
            self.lists = [list(old[o][:len(old[o]) if keep is None else max(0, keep[r])]) if 0 <= o < len(old) else [] for r, o in enumerate(origin)]
        return pairs

    def copy(self, pairs):
        sources, targets = {a for a, _ in pairs}, [b for _, b in pairs]
        assert len(set(targets)) == len(targets) and not sources & set(targets)
        for a, b in pairs:
            self.pool[b] = self.pool[a]

    def compact(self):
        self.table, self.refs, moved, pairs = ref.compact(self.table, self.refs)
        self.copy(pairs)
        n = int((self.refs > 0).sum())
        assert np.all(self.refs[:n] > 0) and np.all(self.refs[n:] <= 0)

    def check(self):
        holders = np.zeros(self.pages, int)
        for r, tokens in enumerate(self.lists):
            assert self.lengths[r] == len(tokens)
            ids = self.table[r, :ref.held(len(tokens), self.page)]
            np.add.at(holders, ids, 1)
            assert self.pool[ids].ravel()[:len(tokens)].tolist() == tokens
            if len(tokens) % self.page:  # the page that is written next
                assert self.refs[ids[-1]] == 1
        assert np.array_equal(holders, self.refs)


@pytest.mark.parametrize("seed", range(12))
def test_random_steps_keep_every_request(seed):
    rng = np.random.default_rng(seed)
    R, page = int(rng.integers(1, 9)), int(rng.choice([1, 2, 4, 16]))
    width = int(rng.integers(1, 12))
    c = Cache(R, width, page, int(rng.integers(1, R * width + 3)))
    refused = 0
    for _ in range(60):
        step = rng.integers(0, 5)
        if step < 3:
            T = int(rng.integers(1, 2 * page + 2))
            refused += int((c.extend(rng.integers(-1, T + 2, R) if step else None, T) < 0).sum())
        elif step == 3:
            origin = np.where(rng.random(R) < 0.5, np.arange(R), rng.integers(-1, R + 1, R))
            keep = None if rng.random() < 0.5 else rng.integers(-1, width * page + 1, R)
            c.fork(origin, keep)
        else:
            c.compact()
        c.check()
    assert refused or R * width * page > 100


def test_extend_goes_in_order_and_takes_the_lowest():
    table, lengths, refs = np.zeros((4, 3), np.int32), np.array([3, 4, 0, 8], np.int32), np.array([1, 0, 1, 0, 1, 0, 1, 1, 0], np.int32)
    table[0, 0], table[1, 0], table[3, :2] = 0, 2, (4, 6)
    t, n, c, added, positions, slots = ref.extend(table, lengths, refs, np.array([6, 1, 13, 4]), 13, 4)
    assert added.tolist() == [6, 1, -1, 4] and n.tolist() == [9, 5, 0, 12]
    assert t.tolist() == [[0, 1, 3], [2, 5, 0], [0, 0, 0], [4, 6, 8]] and c.tolist() == [1] * 9
    assert positions[0, :7].tolist() == [3, 4, 5, 6, 7, 8, -1] and slots[0, :6].tolist() == [3, 4, 5, 6, 7, 12]


def test_extend_without_pages_refuses_one_and_serves_the_next():
    table, lengths, refs = np.zeros((3, 4), np.int32), np.array([0, 0, 0], np.int32), np.array([0, 1, 0], np.int32)
    _, n, c, added, _, slots = ref.extend(table, lengths, refs, np.array([9, 4, 2]), 9, 4)
    assert added.tolist() == [-1, 4, 2] and n.tolist() == [0, 4, 2] and c.tolist() == [1, 1, 1]
    assert slots[1, :4].tolist() == [0, 1, 2, 3] and slots[2, :2].tolist() == [8, 9]


def test_fork_keeps_a_last_page_with_its_first_heir():
    table, lengths, refs = np.full((4, 2), -1, np.int32), np.array([6, 0, 0, 3], np.int32), np.array([1, 1, 1, 0, 0, 0], np.int32)
    table[0], table[3, 0] = (0, 1), 2
    t, n, c, pairs = ref.fork(table, lengths, refs, np.array([-1, 0, 0, 3]), None, 4)
    assert n.tolist() == [0, 6, 6, 3] and pairs == [(1, 3)]
    assert t.tolist() == [[-1, -1], [0, 1], [0, 3], [2, -1]] and c.tolist() == [2, 1, 1, 1, 0, 0]


def test_reference_attention_of_one_request_is_causal_attention():
    from oracle import orc
    rng = np.random.default_rng(3)
    n, heads, kvh, hd, page, window = 5, 4, 2, 8, 4, 7
    start = 11
    k, v = (rng.standard_normal((6, page, kvh, hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((1, n, heads, hd)).astype(np.float32)
    table = np.array([[3, 0, 5, 2]], np.int32)
    got = ref.attention(q, k, v, table, np.array([start + n]), None, 0.3, window)
    flat = [a[table[0]].reshape(-1, kvh, hd).ravel() for a in (k, v)]
    want = orc.attention(q.ravel(), *flat, heads, kvh, hd, start, 0.3, window, 16, n)
    assert np.abs(got.ravel() - want).max() < 1e-5
