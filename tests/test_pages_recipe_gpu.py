"""The step of a batch as the guide for hosts writes it down: its lines are run as they stand, over prompts, decoded tokens, a fork and
a compaction, and every request's attention is held to float64 over its tokens alone."""
import math
import os
import re

import numpy as np
import pytest

from tests import tree_ref
from tests.test_pages_gpu import i32, read, up  # noqa: F401

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HALF = 2.0 ** -11  # a rounding to f16


def blocks():
    with open(os.path.join(ROOT, "INTEGRATION.md"), encoding="utf-8") as f:
        text = f.read()
    section = text[text.index("## 3d."):]
    return re.findall(r"```python\n(.*?)```", section[:section.index("\n## ")], re.S)


def test_the_written_step_runs_and_answers(gpu, up):  # noqa: F811
    step, between = blocks()
    assert "attention_pages_f16kv" in step and "pages_fork" in between
    rng = np.random.default_rng(31)
    requests, tokens, heads, kv_heads, hd, page, max_pages, pages, hidden, rank, adapters = 4, 6, 8, 2, 64, 8, 10, 64, 128, 8, 3
    row, theta, scale = kv_heads * hd, 1e4, 1 / math.sqrt(hd)
    z = lambda n, kind=np.int32: up(np.zeros(n, kind))  # noqa: E731
    matrix = lambda r, c: (rng.standard_normal((r, c)) / math.sqrt(c)).astype(np.float32)  # noqa: E731
    W = {"q": matrix(heads * hd, hidden), "kv": matrix(2 * row, hidden)}
    A, B = ({n: np.stack([matrix(r, c) for _ in range(adapters)]).astype(np.float16) for n, r, c in shapes}
            for shapes in ((("q", rank, hidden), ("v", rank, hidden)), (("q", heads * hd, rank), ("v", row, rank))))
    scales = np.array([0.5, 1.0, 2.0], np.float32)
    env = dict(gpu=gpu, type=0, requests=requests, tokens=tokens, heads=heads, kv_heads=kv_heads, hd=hd, page=page, max_pages=max_pages, pages=pages,
               hidden=hidden, rank=rank, adapters=adapters, row=row, theta=theta, scale=scale, window=1 << 30, shared=8, owner=0,
               page_bytes=page * row * 2, table=z(requests * max_pages), lengths=z(requests), refs=z(pages), added=z(requests),
               positions=z(requests * tokens), slots=z(requests * tokens), copies=z(max(2 * requests + 1, 2 * (pages // 2) + 1)), moved=z(pages),
               k_pool=z(pages * page * row, np.float16), v_pool=z(pages * page * row, np.float16), w_q=up(W["q"]), w_kv=up(W["kv"]), q_a=up(A["q"]),
               q_b=up(B["q"]), v_a=up(A["v"]), v_b=up(B["v"]), scales=up(scales), q=z(requests * tokens * heads * hd, np.float32),
               kv=z(requests * tokens * 2 * row, np.float32), y=z(requests * tokens * heads * hd, np.float32))
    env["pools"] = [env["k_pool"], env["v_pool"]]
    which = [0, -1, 2, 1]
    cached = [[] for _ in range(requests)]  # rotated keys and values, as the pools hold them

    def low_rank(name, x, w):
        return 0 if w < 0 else float(scales[w]) * (B[name][w].astype(np.float64) @ (A[name][w].astype(np.float64) @ x))

    def run(counts, requests=requests, tokens=tokens):
        x = rng.standard_normal((requests * tokens, hidden)).astype(np.float32)
        env.update(x=up(x), counts=up(i32(counts)), which=up(i32(np.repeat(which[:requests], tokens))), requests=requests, tokens=tokens)
        exec(step, env)
        assert read(gpu, env["added"], requests).tolist() == list(counts)
        y = read(gpu, env["y"], (requests, tokens, heads, hd), np.float32)
        for r in range(requests):
            for t in range(counts[r]):
                xt = x[r * tokens + t].astype(np.float64)
                at = [len(cached[r])]
                q = tree_ref.rope((W["q"].astype(np.float64) @ xt + low_rank("q", xt, which[r])).reshape(1, heads, hd), at, theta, 1.0, hd, False)[0]
                both = W["kv"].astype(np.float64) @ xt
                both[row:] += low_rank("v", xt, which[r])
                k = tree_ref.rope(both[:row].reshape(1, kv_heads, hd), at, theta, 1.0, hd, False)[0]
                cached[r].append([m.astype(np.float32).astype(np.float16).astype(np.float64) for m in (k, both[row:].reshape(kv_heads, hd))])
                K, V = (np.stack([e[i] for e in cached[r]]) for i in range(2))
                for h in range(heads):
                    g = h // (heads // kv_heads)
                    s = K[:, g] @ q[h] * scale
                    p = np.exp(s - s.max())
                    # a value beside a border of f16 may be rounded the other way, by 2^-11 of itself more: a key so changes a score by
                    # 2 HALF of its largest sum of magnitudes S, a weight by twice that; f32's own roundings are far below
                    S = (np.abs(K[:, g]) @ np.abs(q[h]) * scale).max()
                    assert np.abs(y[r, t, h] - p @ V[:, g] / p.sum()).max() <= (4 * S + 2) * HALF * np.abs(V[:, g]).max(), (r, t, h)
            assert np.all(y[r, max(0, counts[r]):] == 0)

    run([6, 2, 0, 5])
    run([6, 1, 3, 1])
    run([1, 1, 1, 1])
    env.update(origin=up(i32([0, 0, -1, 3])), keep=up(i32([13, 11, 0, 7])))
    env.update(requests=requests)
    exec(between, env)
    cached[:] = [cached[0], cached[0][:11], [], cached[3][:7]]
    which[:] = [0, 0, 2, 1]
    used = read(gpu, env["refs"], pages) > 0
    assert used[:used.sum()].all()
    run([1, 1, 4, 1])
    run([2, 6, 1, 0])
    run([6, 3], requests=2)  # those with a chunk are the table's first rows: two batches
    run([0, 0, 1, 1], tokens=1)
