"""Caches in pages on the MI355X against the plain forms of tests/pages_ref.py: tables, lengths, counts, positions, slots
and copies are equal, rows and pages moved are equal, f16 rows equal the rounding to nearest even."""
import ctypes

import numpy as np
import pytest

from tests import pages_ref as ref
from webgpu_amd.gpu import Compute, WgdError, WGD_E_INVALID, WGD_E_STATE

pytestmark = pytest.mark.gpu


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


def read(gpu, b, shape, dtype=np.int32):
    n = int(np.prod(shape))
    return np.frombuffer(gpu.read(b, n * np.dtype(dtype).itemsize), dtype).reshape(shape).copy()


def i32(a):
    return np.asarray(a, np.int32)


def random_state(rng, R, width, page, pages, share=0.3):
    """Rows of ragged lengths whose full pages may be shared, with the counts of their holders."""
    table, lengths, refs = rng.integers(-5, pages + 5, (R, width)).astype(np.int32), np.zeros(R, np.int32), np.zeros(pages, np.int32)
    order = rng.permutation(pages).tolist()
    for r in range(R):
        n = int(rng.integers(0, width * page + 1))
        for c in range(ref.held(n, page)):
            if r and (c + 1) * page <= min(n, lengths[r - 1]) and rng.random() < share:
                table[r, c] = table[r - 1, c]
            elif order:
                table[r, c] = order.pop()
            else:
                n = c * page
                break
            refs[table[r, c]] += 1
        lengths[r] = n
    return table, lengths, refs


SHAPES = [(1, 1, 1, 1), (1, 3, 16, 2), (3, 5, 4, 12), (8, 64, 16, 700), (64, 17, 1, 400), (7, 9, 1024, 40), (33, 300, 2, 20000),
          (1024, 3, 8, 2000), (5, 4000, 32, 70001), (100, 40, 64, 1)]


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_extend(gpu, up, shape, seed):
    R, width, page, pages = shape
    rng = np.random.default_rng(seed + R)
    T = [1, int(rng.integers(2, 40)), min(2 * page * width + 3, 2 ** 24 // R, 3000)][seed]
    table, lengths, refs = random_state(rng, R, width, page, pages)
    counts = rng.integers(-1, T + 2, R).astype(np.int32) if seed else None
    if seed == 2 and R > 3:
        lengths[1], lengths[2] = -3, width * page + 1  # no lengths
    b = [up(x) for x in (table, lengths, refs)]
    outs = [up(np.full(n + 3, 77, np.int32)) for n in (R, R * T, R * T)]
    cb = up(counts) if counts is not None else None
    for _ in range(3):  # again and again, until pages run short
        gpu.pages_extend(*b, *outs, R, T, page, width, pages, counts=cb)
        want = ref.extend(table, lengths, refs, counts, T, page)
        table, lengths, refs = want[:3]
        for x, w in zip(b, want):
            assert np.array_equal(read(gpu, x, w.shape), w)
        for x, w in zip(outs, want[3:]):
            got = read(gpu, x, w.size + 3)
            assert np.array_equal(got[:w.size], w.ravel()) and np.all(got[w.size:] == 77)


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_fork(gpu, up, shape, seed):
    R, width, page, pages = shape
    rng = np.random.default_rng(10 * seed + R)
    table, lengths, refs = random_state(rng, R, width, page, pages)
    origin = [np.arange(R), np.zeros(R), np.full(R, -1), rng.integers(-2, R + 2, R), np.arange(R) // 3 * 3, rng.permutation(R)][seed].astype(np.int32)
    keep = rng.integers(-3, width * page + 5, R).astype(np.int32) if seed % 2 else None
    pinned = rng.integers(0, pages, max(1, pages // 10))
    refs[pinned] += 1  # the host's own lists
    b = [up(x) for x in (table, lengths, refs)]
    copies, ob, kb = up(np.full(2 * R + 4, 77, np.int32)), up(origin), up(keep) if keep is not None else None
    for _ in range(2):
        gpu.pages_fork(*b, ob, copies, R, page, width, pages, keep=kb)
        t, n, c, pairs = ref.fork(table, lengths, refs, origin, keep, page)
        got = read(gpu, copies, 2 * R + 4)
        assert np.all(got[1 + 2 * R:] == 77)
        flat = [x for p in pairs or [] for x in p]
        assert got[:1 + 2 * R].tolist() == [-1 if pairs is None else len(pairs)] + flat + [-1] * (2 * R - len(flat))
        for x, w in zip(b, (t, n, c)):
            assert np.array_equal(read(gpu, x, w.shape), w)
        table, lengths, refs = t, n, c


def test_fork_without_pages_changes_nothing(gpu, up):
    rng = np.random.default_rng(5)
    R, width, page = 16, 6, 8
    table = np.arange(R * width).reshape(R, width).astype(np.int32)
    lengths, refs = np.full(R, width * page - 3, np.int32), np.ones(R * width, np.int32)
    lengths[7] = 0
    refs[7 * width:8 * width] = [1, 1, 0, 1, 1, 0]  # two pages are left, the third row would free no more
    origin = np.zeros(R, np.int32)
    origin[8:] = np.arange(8, R)
    b = [up(x) for x in (table, lengths, refs)]
    keep = np.full(R, width * page, np.int32)
    keep[1:7] = 5
    refs_held = refs.copy()
    refs_held[width:7 * width] += 1  # held elsewhere too: freeing rows 1 to 6 gives nothing back
    gpu.write(b[2], refs_held)
    copies = up(np.zeros(2 * R + 1, np.int32))
    want = ref.fork(table, lengths, refs_held, origin, keep, page)
    assert want[3] is None
    gpu.pages_fork(*b, up(origin), copies, R, page, width, R * width, keep=up(keep))
    assert read(gpu, copies, 2 * R + 1).tolist() == [-1] * (2 * R + 1)
    for x, w in zip(b, (table, lengths, refs_held)):
        assert np.array_equal(read(gpu, x, w.shape), w)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("R,width,pages,used", [(1, 1, 1, 0), (1, 1, 1, 1), (2, 3, 2, 1), (4, 9, 33, 20), (8, 64, 1000, 999), (8, 64, 1000, 1),
                                                (3, 50000, 100003, 60000), (64, 40, 16385, 9000), (1024, 4, 16384, 8192)])
def test_compact(gpu, up, R, width, pages, used, inplace):
    rng = np.random.default_rng(R + pages)
    table = rng.integers(-3, pages + 3, (R, width)).astype(np.int32)
    refs = np.zeros(pages, np.int32)
    refs[rng.permutation(pages)[:used]] = rng.integers(1, 9, used)
    refs[rng.integers(0, pages, 2)] -= 2 if used < pages // 2 else 0
    tb, rb, moved, copies = up(table), up(refs), up(np.full(pages + 1, 77, np.int32)), up(np.full(pages // 2 * 2 + 3, 77, np.int32))
    to, ro = (tb, rb) if inplace else (up(np.full(table.size + 1, 77, np.int32)), up(np.full(pages + 1, 77, np.int32)))
    gpu.pages_compact(tb, rb, to, ro, moved, copies, R, width, pages)
    t, c, m, pairs = ref.compact(table, refs)
    assert np.array_equal(read(gpu, to, t.shape), t)
    got, free = read(gpu, ro, pages), c <= 0
    assert np.array_equal(got[~free], c[~free]) and np.all(got[free] <= 0)
    assert np.array_equal(read(gpu, moved, pages), m)
    flat = [int(x) for p in pairs for x in p]
    assert read(gpu, copies, pages // 2 * 2 + 1).tolist() == [len(pairs)] + flat + [-1] * (pages // 2 * 2 - len(flat))
    if not inplace:
        assert np.array_equal(read(gpu, tb, table.shape), table) and np.array_equal(read(gpu, rb, pages), refs)
        assert read(gpu, to, table.size + 1)[-1] == 77 and read(gpu, ro, pages + 1)[-1] == 77
    assert read(gpu, moved, pages + 1)[-1] == 77 and np.all(read(gpu, copies, pages // 2 * 2 + 3)[-2:] == 77)


@pytest.mark.parametrize("pages", [1024, 1025, 2050, 4095, 4096, 4097, 5001])
def test_pools_around_the_pages_of_a_thread(gpu, up, pages):
    """A thread has one page of a pool, four or sixteen: pools at and beside where that changes."""
    for used in (pages // 2, pages - 1):
        for inplace in (False, True):
            test_compact(gpu, up, 8, 200, pages, used, inplace)
    test_extend(gpu, up, (6, 1000, 1, pages), 0)
    test_fork(gpu, up, (6, 900, 2, pages), 0)


@pytest.mark.parametrize("pools,pages,bytes_,n", [(1, 2, 2, 1), (3, 9, 6, 4), (2, 40, 4100, 17), (130, 12, 64, 5), (2, 300, 32768, 130),
                                                  (1, 5, 50002, 2), (1, 6000, 16, 3000)])
def test_copy(gpu, up, pools, pages, bytes_, n):
    rng = np.random.default_rng(pages)
    data = rng.integers(0, 256, (pools, pages, bytes_), dtype=np.uint8)
    order = rng.permutation(pages)
    pairs = np.stack([order[:n], order[n:2 * n]], 1)
    listed = np.concatenate([[n], pairs.ravel(), [0, 1]]).astype(np.int32)  # what lies behind the count is not carried out
    bufs = [up(d) for d in data]
    gpu.pages_copy(bufs, up(listed), n + 1, bytes_, pages)
    want = data.copy()
    want[:, pairs[:, 1]] = data[:, pairs[:, 0]]
    for b, w in zip(bufs, want):
        assert np.array_equal(read(gpu, b, w.shape, np.uint8), w)


def test_copy_takes_no_pairs_outside_the_pool(gpu, up):
    data = np.arange(40, dtype=np.int32).reshape(5, 8)
    pool = up(data)
    for listed in ([4, -1, 2, 0, -1, 5, 1, 2, 5], [-1, 0, 1, 0, 2, 0, 3, 0, 4], [-2 ** 31] + [1] * 8, [2, 2 ** 31 - 1, 0, 0, -2 ** 31, 0, 1, 0, 1]):
        gpu.pages_copy([pool], up(i32(listed)), 4, 32, 5)
        assert np.array_equal(read(gpu, pool, data.shape), data)
    gpu.pages_copy([pool], up(i32([9, 0, 1, 0, 2])), 2, 32, 5)  # no more than `most`
    data[1] = data[2] = data[0]
    assert np.array_equal(read(gpu, pool, data.shape), data)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("row,rows,stride,ko,vo,slots", [(1, 1, 0, 0, 0, 1), (4, 3, 0, 0, 0, 7), (1024, 9, 3200, 1024, 2048, 64), (6, 50, 20, 3, 11, 60),
                                                         (128, 2000, 384, 128, 256, 4096), (100, 33, 301, 100, 200, 40), (2052, 5, 0, 0, 0, 5)])
def test_store(gpu, up, row, rows, stride, ko, vo, slots, half):
    rng = np.random.default_rng(row)
    step = stride or row
    src = (rng.standard_normal(max(ko, vo) + rows * step) * 100).astype(np.float32)
    src[:3] = ([65519.99, 1e-9, np.nan] if half else [np.inf, -0.0, np.nan])[:src.size]
    kind = np.float16 if half else np.float32
    at = rng.permutation(slots)[:rows] if rows <= slots else rng.permutation(slots)
    at = np.concatenate([at, np.full(rows - len(at), -1)]).astype(np.int32)
    if rows > 4:
        at[1], at[3] = slots, -2 ** 31
    pools = [np.full((slots + 1, row), 7, kind) for _ in range(2)]
    sb, kb, vb = up(src), up(pools[0]), up(pools[1])
    other = up(src[::-1].copy()) if not stride else sb
    (gpu.pages_store_f16kv if half else gpu.pages_store)(sb, other, kb, vb, up(at), row, rows, slots, stride=stride, k_offset=ko, v_offset=vo)
    for buf, pool, off, data in ((kb, pools[0], ko, src), (vb, pools[1], vo, src if stride else src[::-1])):
        for t in range(rows):
            if 0 <= at[t] < slots:
                with np.errstate(over="ignore"):
                    pool[at[t]] = data[off + t * step:off + t * step + row].astype(kind)
        assert np.array_equal(read(gpu, buf, pool.shape, kind), pool, equal_nan=True)


def test_store_offsets_pass_32_bits(gpu, up):
    """Slots behind 2^32 bytes and 2^31 elements of a pool."""
    row, slots = 2048, (1 << 20) + 70
    big, other = gpu.buffer(slots * row * 4, "large pool"), gpu.buffer(slots * row * 4, "large pool")
    try:
        src = np.arange(3 * row, dtype=np.float32).reshape(3, row)
        at = i32([slots - 1, 1 << 20, 5])
        gpu.pages_store(up(src), up(src * 2), big, other, up(at), row, 3, slots)
        for t in range(3):
            got = np.frombuffer(gpu.read(big, row * 4, int(at[t]) * row * 4), np.float32)
            assert np.array_equal(got, src[t])
            got = np.frombuffer(gpu.read(other, row * 4, int(at[t]) * row * 4), np.float32)
            assert np.array_equal(got, 2 * src[t])
    finally:
        gpu.destroy(big)
        gpu.destroy(other)


# ------------------------------------------------------------------------------- graphs

class Hip:
    def __init__(self):
        self.l = ctypes.CDLL("libamdhip64.so")

    def __call__(self, name, *args):
        rc = getattr(self.l, name)(*args)
        assert rc == 0, (name, rc)


def test_a_batch_grows_forks_and_shrinks_in_a_graph():
    """Replays go on from the state that the last one left, as eager calls do."""
    gpu = Compute().init()
    up = Held(gpu)
    hip, stream = Hip(), ctypes.c_void_p(gpu.stream)
    try:
        R, width, page, pages, row, T = 6, 40, 4, 300, 16, 3
        rng = np.random.default_rng(9)
        origin = i32([0, 0, 2, 3, -1, 5])
        src = rng.standard_normal((R * T, row)).astype(np.float32)

        def fresh():
            z = lambda n: up(np.zeros(n, np.int32))  # noqa: E731
            return dict(table=z(R * width), lengths=z(R), refs=z(pages), added=z(R), positions=z(R * T), slots=z(R * T), copies=z(2 * R + 1),
                        table_to=z(R * width), refs_to=z(pages), moved=z(pages), more=z(pages // 2 * 2 + 1), k=up(np.zeros((pages * page, row), np.float32)),
                        v=up(np.zeros((pages * page, row), np.float32)))

        ob, sb, cb = up(origin), up(src), up(i32([3, 2, 1, 0, 3, 2]))

        def step(s):
            state = (s["table"], s["lengths"], s["refs"])
            gpu.pages_extend(*state, s["added"], s["positions"], s["slots"], R, T, page, width, pages, counts=cb)
            gpu.pages_store(sb, sb, s["k"], s["v"], s["slots"], row, R * T, pages * page)
            gpu.pages_fork(*state, ob, s["copies"], R, page, width, pages)
            gpu.pages_copy([s["k"], s["v"]], s["copies"], R, page * row * 4, pages)
            gpu.pages_compact(s["table"], s["refs"], s["table"], s["refs"], s["moved"], s["more"], R, width, pages)
            gpu.pages_copy([s["k"], s["v"]], s["more"], pages // 2, page * row * 4, pages)

        state = lambda s: [gpu.read(b, b.size) for b in s.values()]  # noqa: E731
        a, b = fresh(), fresh()
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        gpu.done()
        hip("hipStreamBeginCapture", stream, 2)
        with pytest.raises(WgdError) as e:  # no call has made its scratch yet; the capture outlives that
            gpu.pages_fork(b["table"], b["lengths"], b["refs"], ob, b["copies"], R, page, width, pages)
        assert e.value.status == WGD_E_STATE
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphDestroy", graph)
        want = []
        for _ in range(8):
            step(a)
            want.append(state(a))
        hip("hipStreamBeginCapture", stream, 2)
        step(b)
        hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        hip("hipGraphInstantiate", ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0))
        for w in want:
            hip("hipGraphLaunch", exe, stream)
            assert state(b) == w
            big = up(np.zeros((64, 4000), np.int32))  # larger work between: the context's scratch grows
            gpu.pages_fork(big, up(np.zeros(64, np.int32)), up(np.zeros(9, np.int32)), up(np.zeros(64, np.int32)), up(np.zeros(129, np.int32)), 64, 1, 4000, 9)
        assert want[0] != want[-1]
        hip("hipGraphExecDestroy", exe)
        hip("hipGraphDestroy", graph)
    finally:
        up.free()
        gpu.dispose()


# ------------------------------------------------------------------------------- refusals

def refusal_calls(gpu, f):
    """Calls that name wrong sizes, aliases and missing buffers; f makes buffers of 16 KB."""
    b = [f(1 << 14) for _ in range(9)]
    t, n, c, ad, ps, sl, og, kp, cp = b
    tiny = f(4)
    E = lambda t=t, n=n, c=c, ad=ad, ps=ps, sl=sl, R=4, T=5, page=4, width=8, pages=64, **kw: \
        gpu.pages_extend(t, n, c, ad, ps, sl, R, T, page, width, pages, **kw)  # noqa: E731
    F = lambda t=t, n=n, c=c, og=og, cp=cp, R=4, page=4, width=8, pages=64, **kw: gpu.pages_fork(t, n, c, og, cp, R, page, width, pages, **kw)  # noqa: E731
    K = lambda t=t, c=c, to=ad, ro=ps, mv=sl, cp=cp, R=4, width=8, pages=64: gpu.pages_compact(t, c, to, ro, mv, cp, R, width, pages)  # noqa: E731
    P = lambda pools=(t, n), cp=cp, most=4, size=64, pages=16: gpu.pages_copy(list(pools), cp, most, size, pages)  # noqa: E731
    S = lambda k=t, v=n, kp=c, vp=ad, sl=sl, row=8, rows=4, slots=64, half=False, **kw: \
        (gpu.pages_store_f16kv if half else gpu.pages_store)(k, v, kp, vp, sl, row, rows, slots, **kw)  # noqa: E731
    bad = [
        lambda: E(R=1025), lambda: E(T=0), lambda: E(T=2 ** 23), lambda: E(page=0), lambda: E(page=3), lambda: E(page=2048), lambda: E(width=0),
        lambda: E(pages=0), lambda: E(width=2 ** 29), lambda: E(pages=2 ** 29), lambda: E(t=tiny), lambda: E(n=tiny), lambda: E(c=tiny), lambda: E(ad=tiny),
        lambda: E(ps=tiny), lambda: E(sl=tiny), lambda: E(counts=tiny), lambda: E(counts=ad), lambda: E(t=n), lambda: E(ps=sl), lambda: E(sl=c),
        lambda: F(R=1025), lambda: F(page=12), lambda: F(width=2 ** 30), lambda: F(pages=5000), lambda: F(t=tiny), lambda: F(n=tiny), lambda: F(c=tiny),
        lambda: F(og=tiny), lambda: F(cp=tiny), lambda: F(keep=tiny), lambda: F(og=n), lambda: F(keep=n), lambda: F(cp=t), lambda: F(t=c),
        lambda: K(R=1025), lambda: K(pages=0), lambda: K(pages=2 ** 31), lambda: K(width=0), lambda: K(t=tiny), lambda: K(c=tiny), lambda: K(to=tiny),
        lambda: K(ro=tiny), lambda: K(mv=tiny), lambda: K(cp=tiny), lambda: K(to=c), lambda: K(ro=t), lambda: K(mv=c), lambda: K(cp=t), lambda: K(mv=cp),
        lambda: K(to=ps), lambda: P(size=0), lambda: P(size=7), lambda: P(size=2 ** 30 + 2), lambda: P(pages=0), lambda: P(pages=257), lambda: P(most=2048),
        lambda: P(pools=(t, t)), lambda: P(pools=(t, cp)), lambda: P(pools=(tiny,)), lambda: P(cp=tiny), lambda: P(most=2 ** 31), lambda: P(pools=[t] * 65537),
        lambda: S(row=0), lambda: S(stride=7), lambda: S(rows=2000), lambda: S(slots=2 ** 31), lambda: S(slots=513), lambda: S(slots=1025, half=True),
        lambda: S(k=tiny), lambda: S(v=tiny), lambda: S(kp=tiny), lambda: S(vp=tiny), lambda: S(sl=tiny), lambda: S(kp=t), lambda: S(vp=c), lambda: S(vp=sl),
        lambda: S(k_offset=4096 - 31), lambda: S(v_offset=2 ** 63), lambda: S(rows=2 ** 32 - 1, stride=2 ** 32 - 1),
    ]
    fine = [lambda: E(R=0), lambda: F(R=0), lambda: K(R=0), lambda: P(pools=()), lambda: P(most=0), lambda: S(rows=0), lambda: S(slots=0),
            lambda: S(slots=1024, half=True), E, F, K, P, S, lambda: K(to=t, ro=c), lambda: S(k=t, v=t)]
    return b, bad, fine


def test_refusals(gpu, up):
    b, bad, fine = refusal_calls(gpu, lambda n: up(np.zeros(n, np.uint8)))
    other = Compute().init()
    try:
        foreign = other.upload(np.zeros(1 << 14, np.uint8))
        t, n, c, ad, ps, sl, og, kp, cp = b
        bad += [lambda: gpu.pages_extend(foreign, n, c, ad, ps, sl, 4, 5, 4, 8, 64), lambda: gpu.pages_fork(t, n, c, foreign, cp, 4, 4, 8, 64),
                lambda: gpu.pages_compact(t, foreign, ad, ps, sl, cp, 4, 8, 64), lambda: gpu.pages_copy([foreign], cp, 4, 64, 16),
                lambda: gpu.pages_store(t, n, foreign, ad, sl, 8, 4, 64)]
        for i, call in enumerate(bad):
            with pytest.raises(WgdError) as e:
                call()
            assert e.value.status == WGD_E_INVALID, i
        for call in fine:
            call()
        gpu.done()
    finally:
        other.dispose()
