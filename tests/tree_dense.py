"""Tree attention in float64 as a product per kv head under a mask, for rings too long for the form of
tests/tree_ref.py, and the bounds that outputs are held to.

Bounds, with e = 2^-24 (half a step of f32), n keys and S = scale max sum|q k|: the f32 dot product of hd terms is off by
at most hd e sum|q k|, so a weight by twice that and by its own rounding; numerator and denominator are sums of n
weights, n e each at most. So each output is within (2 (hd + 4) e S + 2 (n + 8) e) max|v|. That is for the worst
signs: roundings are independent, so the 2-norm of the difference is held to 16 e sqrt(hd + n) max(1, sqrt(S)) times
the result's as well.
"""
import math

import numpy as np

from tests import tree_ref

EPS = 2.0 ** -24
NO_WINDOW = 1 << 30

# heads, kv_heads, head_dim, nodes, start, window, slots to spare, with f16 rings: all are shapes for the kernel
# that stages keys in LDS. What the plan makes of them on 256 CUs:
STAGED = [
    # two row groups, one stage a workgroup, the window's first keys hidden; the ring wraps inside a stage
    (8, 1, 128, 64, 9001, 2500, 0), (8, 1, 128, 64, 9001, 2500, 27), (8, 1, 64, 64, 5000, 1500, 0), (4, 1, 256, 32, 6000, 2100, 27),
    # the wrap among the nodes
    (8, 1, 128, 64, 7659, 2500, 0),
    # four to sixteen stages a workgroup: the stages change places, the last one is cut by the split's end
    (32, 8, 128, 64, 9001, 4000, 0), (128, 16, 128, 64, 9001, 4000, 27), (64, 16, 64, 64, 9000, 4000, 5), (32, 16, 256, 40, 9000, 4100, 9),
    # more than 64 nodes: paths in LDS in place of registers
    (2, 1, 128, 256, 5000, 1024, 0), (32, 4, 128, 256, 5000, 1024, 0),
    # four row groups: a ring that does not wrap, and windows over one that does
    (4, 1, 128, 64, 8100, NO_WINDOW, 0), (4, 1, 64, 64, 8000, NO_WINDOW, 0), (4, 1, 256, 16, 8050, NO_WINDOW, 3), (64, 16, 128, 64, 9000, NO_WINDOW, 0),
    (4, 1, 128, 64, 20011, 8200, 0), (4, 1, 256, 16, 16200, 8100, 0), (64, 16, 128, 64, 15000, 8200, 27), (64, 16, 64, 64, 19000, 8200, 5),
    (32, 8, 256, 64, 20000, 8101, 0),
    # a long window whose splits are 25 stages long
    (48, 16, 128, 64, 31000, 16000, 40),
]


def inputs(case, pads):
    """q, K and V rings of f16, parents, what the nodes see, the first key and the scale."""
    heads, kvh, hd, nodes, start, window, extra = case
    rng = np.random.default_rng(sum(case))
    cap = min(start, window - 1) + nodes + extra
    q = rng.standard_normal((nodes, heads, hd)).astype(np.float32)
    k, v = (rng.standard_normal((cap, kvh, hd)).astype(np.float16) for _ in range(2))
    parents = np.array([-1, -1][:nodes] + [int(rng.integers(max(0, i - 6), i)) for i in range(2, nodes)], np.int32)
    for i in rng.choice(np.arange(1, nodes), pads, replace=False):
        parents[i] = int(rng.choice([-2, -2 ** 31, i, i + 1, 2 ** 31 - 1]))
    return q, k, v, parents, *visible(parents, start, window), 1 / math.sqrt(hd)


def visible(parents, start, window):
    """Which of the keys [first, start + nodes) each node sees, and the first one."""
    nodes, first = len(parents), start - min(start, window - 1)
    sees = np.zeros((nodes, start + nodes - first), bool)
    for i, path in enumerate(tree_ref.paths(parents)):
        if path is not None:
            pos = start + len(path) - 1
            sees[i, max(first, pos + 1 - window) - first:start - first] = True
            sees[i, [start - first + a for a in path[:window]]] = True
    return sees, first


def attention(q, k, v, sees, first, scale):
    """Outputs [nodes][heads][hd], zeros where a node sees nothing, and S. What a masked place holds is not used."""
    nodes, heads, hd = q.shape
    cap, kvh, _ = k.shape
    group, slots = heads // kvh, np.arange(first, first + sees.shape[1]) % cap
    y, S = np.zeros(q.shape), 0.0
    for g in range(kvh):
        kg, vg = k[slots, g].astype(np.float64), v[slots, g].astype(np.float64)
        qg = q[:, g * group:(g + 1) * group].astype(np.float64).reshape(-1, hd)
        mask = np.repeat(sees, group, 0)
        s = np.where(mask, qg @ kg.T * scale, -np.inf)
        with np.errstate(invalid="ignore"):
            p = np.where(mask, np.exp(s - s.max(1, keepdims=True)), 0)
            out = p @ vg / p.sum(1, keepdims=True)
        y[:, g * group:(g + 1) * group] = np.where(mask.any(1)[:, None], out, 0).reshape(nodes, group, hd)
        S = max(S, scale * float((np.abs(qg) @ np.abs(kg).T).max()))
    return y, S


def bounds(want, S, keys, most):
    """Of each output, and of the 2-norm; `most` is max|v|."""
    hd = want.shape[-1]
    return ((2 * (hd + 4) * EPS * S + 2 * (keys + 8) * EPS) * most,
            16 * EPS * math.sqrt(hd + keys) * max(1, math.sqrt(S)) * float(np.linalg.norm(want)))


def within(got, want, S, keys, most):
    each, norm = bounds(want, S, keys, most)
    return bool(np.isfinite(got).all() and np.abs(got - want).max() <= each and np.linalg.norm(got - want) <= norm)
