"""Plain float64 forms of the drafted-tree operators (include/wgd.h), one token at a time."""
import math

import numpy as np


def rope(x, positions, theta, scale, rot, adjacent, factors=None, magnitude=1.0):
    """x [batch][heads][hd] in float64, rotated."""
    x = np.array(x, np.float64)
    for t, pos in enumerate(positions):
        for j in range(rot // 2):
            a = float(pos) * float(np.float32(scale)) * float(np.float32(theta)) ** (-2 * j / rot)
            if factors is not None:
                a /= float(factors[j])
            c, s = math.cos(a) * float(np.float32(magnitude)), math.sin(a) * float(np.float32(magnitude))
            i, k = (2 * j, 2 * j + 1) if adjacent else (j, j + rot // 2)
            l, r = x[t, :, i].copy(), x[t, :, k].copy()
            x[t, :, i], x[t, :, k] = l * c - r * s, l * s + r * c
    return x


def paths(parents):
    """Every node's path to the root, itself first; None for padding."""
    out = []
    for i, p in enumerate(parents):
        up = [] if p == -1 else out[p] if 0 <= p < i else None
        out.append(None if up is None else [i] + up)
    return out


def attention(q, k, v, parents, start, scale, window):
    """q [nodes][heads][hd]; k, v rings [capacity][kvh][hd]; zeros for padding."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    cap, kvh, hd = k.shape
    heads = q.shape[1]
    y = np.zeros(q.shape)
    for i, path in enumerate(paths(parents)):
        if path is None:
            continue
        pos = start + len(path) - 1
        slots = [t % cap for t in range(max(0, pos + 1 - window), start)] + [(start + a) % cap for a in path[:window]]
        for h in range(heads):
            g = h // (heads // kvh)
            with np.errstate(invalid="ignore", over="ignore"):
                s = k[slots, g] @ q[i, h] * scale
                p = np.exp(s - s.max())
                y[i, h] = p @ v[slots, g] / p.sum()
    return y


def draws(logits, us, temperature, top_k, top_p, min_p):
    """For each uniform the tokens that a draw may give: one, or two where it lies within 1e-9 of a border."""
    idx = np.flatnonzero(np.isfinite(logits))
    if not len(idx):
        return [{-1} for _ in us]
    order = idx[np.argsort(-logits[idx].astype(np.float64), kind="stable")]
    l = logits[order].astype(np.float64)
    with np.errstate(over="ignore", under="ignore", divide="ignore", invalid="ignore"):
        p = np.exp((l - l[0]) / temperature) if temperature else np.zeros(len(l))
    if top_k:
        p = p[:top_k]
    cum = np.cumsum(p)
    out = [set() for _ in us]
    for dp in (-1e-9, 0, 1e-9):
        # shares never fall, so the first that reaches top_p is found by bisection
        cut = min(int(np.searchsorted(cum / cum[-1], top_p * (1 + dp), "left")) + 1, len(p)) if temperature and top_p < 1 else len(p)
        kept = min(cut, int(np.sum(p >= min_p)))
        for i, u in enumerate(us):
            if temperature == 0 or not 0 <= u < 1:
                out[i].add(int(order[0]))
                continue
            for du in (-1e-9, 0, 1e-9):
                out[i].add(int(order[min(int(np.searchsorted(cum[:kept], (u + du) * cum[kept - 1], "left")), kept - 1)]))
    return out


def draw(logits, u, temperature, top_k, top_p, min_p):
    return draws(logits, [u], temperature, top_k, top_p, min_p)[0]


def accept(parents, drafted, picked):
    """(count, next token, nodes) of the confirmed path."""
    if parents[0] != -1:
        return 0, -1, []
    nodes = [0]
    while True:
        c = nodes[-1]
        child = [i for i in range(c + 1, len(parents)) if parents[i] == c and drafted[i] == picked[c] and picked[c] >= 0]
        if not child:
            return len(nodes), int(picked[c]), nodes
        nodes.append(child[0])
