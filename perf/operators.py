"""The operators of a decode step over a tree of drafted tokens, as a list of timed cases.

A small model, or extra heads, draft a tree of continuations; the large model reads all of its
nodes in one batch. Beside the products that the framework has, such a step takes: rotary
positions given token by token (siblings share one), attention of every node over the cached keys
and its own ancestors, a token drawn at every node, the walk that finds the drafted path which the
draws confirm, and the move of that path's keys and values to the places that they keep.

Where ``own`` is false, ``run`` computes these with plain torch; where it is true, with the
framework's operators on the framework's buffers. ``exact`` restates them in float64.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token of the small model, query and key heads of one row: the launch counts
        {"name": "rope_one_0.6b", "kind": "rope", "heads": 24, "head_dim": 128, "rotary": 128, "stride": 4096, "batch": 1,
         "theta": 1e6, "adjacent": False, "factors": False, "magnitude": 1.0},
        # a full tree of the 8B model with the long-context frequencies, inside rows of q | k | v
        {"name": "rope_tree_8b", "kind": "rope", "heads": 40, "head_dim": 128, "rotary": 128, "stride": 6144, "batch": 64,
         "theta": 5e5, "adjacent": True, "factors": True, "magnitude": 1.0},
        # a short chat with the small model, sixteen drafted tokens
        {"name": "tree_0.6b_short", "kind": "attention", "heads": 16, "kv_heads": 8, "head_dim": 128, "start": 300,
         "window": 1 << 30, "capacity": 1024, "nodes": 16, "pad": 0, "kv": "f32"},
        # a local layer of the 27B model: the ring has wrapped many times, the tree is padded
        {"name": "tree_27b_window", "kind": "attention", "heads": 32, "kv_heads": 16, "head_dim": 128, "start": 8191,
         "window": 1024, "capacity": 1151, "nodes": 48, "pad": 3, "kv": "f32"},
        # the 8B model deep in a long document with half-precision rings
        {"name": "tree_8b_32k", "kind": "attention", "heads": 32, "kv_heads": 8, "head_dim": 128, "start": 31000,
         "window": 1 << 30, "capacity": 32768, "nodes": 64, "pad": 0, "kv": "f16"},
        # one row of the small model's logits with the default settings
        {"name": "sample_one_0.6b", "kind": "sample", "vocab": 151936, "rows": 1, "temperature": 0.7, "top_k": 40,
         "top_p": 0.9, "min_p": 0.0},
        # every node of a tree of the 8B model, the default settings with min-p
        {"name": "sample_tree_8b", "kind": "sample", "vocab": 128256, "rows": 64, "temperature": 0.7, "top_k": 40,
         "top_p": 0.9, "min_p": 0.02},
        # the whole vocabulary of the 27B model without top-k
        {"name": "sample_whole_27b", "kind": "sample", "vocab": 262144, "rows": 16, "temperature": 1.0, "top_k": 0,
         "top_p": 0.95, "min_p": 0.0},
        # the walk down a small tree, and down the largest
        {"name": "accept_16", "kind": "accept", "nodes": 16, "pad": 0},
        {"name": "accept_256", "kind": "accept", "nodes": 256, "pad": 5},
        # three accepted tokens in the rings of the small model's 28 layers
        {"name": "commit_0.6b", "kind": "commit", "layers": 28, "row": 1024, "capacity": 512, "start": 300, "nodes": 16,
         "accepted": 4, "kv": "f32"},
        # a long accepted path across the wrap of the 8B model's half-precision rings
        {"name": "commit_8b", "kind": "commit", "layers": 32, "row": 1024, "capacity": 4096, "start": 4070, "nodes": 64,
         "accepted": 12, "kv": "f16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["rope", "attention", "attention", "attention", "sample", "sample", "sample", "accept", "commit"])
    if kind == "rope":
        hd = rng.choice([64, 80, 96, 128, 128, 256])
        heads = _spread(rng, 1, 48)
        return {"kind": "rope", "heads": heads, "head_dim": hd, "rotary": rng.choice([hd, hd, hd // 2]),
                "stride": heads * hd + rng.choice([0, 2, 1024]), "batch": _spread(rng, 1, 256), "theta": rng.choice([1e4, 5e5, 1e6]),
                "adjacent": rng.random() < 0.5, "factors": rng.random() < 0.5, "magnitude": rng.choice([1.0, 1.0, 0.9])}
    if kind == "attention":
        kvh, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 4, 7, 8])
        hd, kv = rng.choice([64, 80, 128, 128, 128, 256]), rng.choice(["f32", "f16"])
        nodes, start = _spread(rng, 1, 256), rng.choice([0, _spread(rng, 1, 31000), _spread(rng, 100, 31000)])
        while nodes * kvh * group * (start + nodes) * hd > 8e9 or (start + nodes) * kvh * hd * (8 if kv == "f32" else 4) > 1.3e8:
            nodes, start = max(1, nodes // 2), start * 3 // 4
        window = rng.choice([1 << 30, 1 << 30, _spread(rng, 1, 4096)])
        return {"kind": "attention", "heads": kvh * group, "kv_heads": kvh, "head_dim": hd,
                "start": start, "window": window, "capacity": min(start, window - 1) + nodes + rng.choice([0, 1, 100]),
                "nodes": nodes, "pad": min(nodes - 1, rng.choice([0, 0, 3])), "kv": kv}
    if kind == "sample":
        vocab = _spread(rng, 1000, 262144)
        return {"kind": "sample", "vocab": vocab, "rows": _spread(rng, 1, max(1, min(256, 8_000_000 // vocab))),
                "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), "top_k": rng.choice([0, 0, 1, 40, _spread(rng, 2, 1000)]),
                "top_p": rng.choice([1.0, 0.9, 0.95, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}
    nodes = _spread(rng, 2, 256)
    if kind == "accept":
        return {"kind": "accept", "nodes": nodes, "pad": min(nodes - 1, rng.choice([0, 0, 3]))}
    start = _spread(rng, 1, 8000)
    return {"kind": "commit", "layers": rng.randint(1, 32), "row": 64 * _spread(rng, 1, 32), "capacity": nodes + _spread(rng, 1, 1000),
            "start": start, "nodes": nodes, "accepted": min(nodes, _spread(rng, 1, 20)), "kv": rng.choice(["f32", "f16"])}


# ------------------------------------------------------------------------------- inputs

def _gen(seed, tag):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1_000_003 + tag * 7919 + 17) & 0x7FFFFFFFFFFF)


def _tree(nodes, pad, seed):
    """Parents of a drafted tree in the order drafted (-1: follows the cached tokens; -2: padding), a
    random recent node each, so both long paths and many siblings occur."""
    rng = np.random.default_rng(seed)
    parents = [-1] + [int(rng.integers(max(0, i - 8), i)) for i in range(1, nodes - pad)]
    return np.array(parents + [-2] * pad, np.int32)


def _ancestors(parents):
    """The nodes that each one sees, itself among them, and the depths (host)."""
    n = len(parents)
    sees = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= -1:
            sees[i] = sees[p] if p >= 0 else False
            sees[i, i] = True
    return sees, np.maximum(sees.sum(1) - 1, 0).astype(np.int32)


def _slots(case):
    """Ring slots of the cached keys that some node sees, then of the nodes."""
    first = max(0, case["start"] + 1 - case["window"])
    return torch.arange(first, case["start"] + case["nodes"], device="cuda") % case["capacity"]


def _rope_inputs(case, seed):
    x = torch.randn(case["batch"], case["stride"], generator=_gen(seed, 0), device="cuda")
    p = torch.randint(0, 8, (case["batch"],), generator=_gen(seed, 1), device="cuda", dtype=torch.int32)
    p = p + int(np.random.default_rng(seed).integers(1, 130000))
    f = None
    if case["factors"]:  # low frequencies interpolated by 8, high ones kept, a ramp between
        wave = 2 * math.pi * case["theta"] ** (torch.arange(0, case["rotary"], 2, device="cuda").double() / case["rotary"])
        smooth = ((8192 / wave - 1) / 3).clamp(0, 1)
        f = (1 / ((1 - smooth) / 8 + smooth)).float()
    return {"x": x, "positions": p.to(torch.int32), "factors": f}


def _attention_inputs(case, seed):
    half = torch.float16 if case["kv"] == "f16" else torch.float32
    q = torch.randn(case["nodes"], case["heads"], case["head_dim"], generator=_gen(seed, 0), device="cuda") * 1.5
    k, v = (torch.randn(case["capacity"], case["kv_heads"], case["head_dim"], generator=_gen(seed, 1 + i), device="cuda").to(half)
            for i in range(2))
    parents = _tree(case["nodes"], case["pad"], seed)
    sees, depth = _ancestors(parents)
    up = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    return {"q": q, "k": k, "v": v, "y": torch.zeros_like(q), "parents": up(parents), "sees": up(sees), "depth": up(depth)}


def _sample_inputs(case, seed):
    logits = 2.5 * torch.randn(case["rows"], case["vocab"], generator=_gen(seed, 0), device="cuda")
    return {"logits": logits, "uniforms": torch.rand(case["rows"], generator=_gen(seed, 1), device="cuda", dtype=torch.float64),
            "tokens": torch.zeros(case["rows"], device="cuda", dtype=torch.int32)}


def _accept_inputs(case, seed):
    parents = _tree(case["nodes"], case["pad"], seed)
    rng = np.random.default_rng(seed + 1)
    picked, drafted = (rng.integers(0, 150000, case["nodes"]).astype(np.int32) for _ in range(2))
    inner = parents >= 0  # a third of the drafted tokens are what the model draws at their parents
    hit = inner & (rng.random(case["nodes"]) < 0.35)
    drafted[hit] = picked[parents[hit]]
    sees, _ = _ancestors(parents)
    up = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    return {"parents": up(parents), "drafted": up(drafted), "picked": up(picked), "sees": up(sees),
            "path": torch.zeros(case["nodes"] + 2, dtype=torch.int32, device="cuda")}


def _commit_inputs(case, seed):
    half = torch.float16 if case["kv"] == "f16" else torch.float32
    rings = torch.randn(2 * case["layers"], case["capacity"], case["row"], generator=_gen(seed, 0), device="cuda").to(half)
    rng = np.random.default_rng(seed)
    path = np.full(case["nodes"] + 2, -1, np.int32)
    path[0], path[1] = case["accepted"], rng.integers(0, 150000)
    path[3:2 + case["accepted"]] = np.sort(1 + rng.permutation(case["nodes"] - 1)[:case["accepted"] - 1])
    path[2] = 0
    return {"rings": rings, "path": torch.from_numpy(path).cuda()}


_INPUTS = {"rope": _rope_inputs, "attention": _attention_inputs, "sample": _sample_inputs, "accept": _accept_inputs,
           "commit": _commit_inputs}


# ------------------------------------------------------------------------------- the framework's buffers

_compute = None


def _connect():
    """The framework's context. Its stream becomes torch's current one, so that what torch does with the buffers, before
    the operators run or with what they wrote, keeps its place among their launches; a caller who makes another
    stream the current one orders it after this one."""
    global _compute
    if _compute is None:
        from webgpu_amd.gpu import Compute
        _compute = Compute().init()
    if torch.cuda.current_stream().cuda_stream != _compute.stream:
        torch.cuda.synchronize()
        torch.cuda.set_stream(torch.cuda.ExternalStream(_compute.stream))


class _View:
    """The CUDA array interface of a framework buffer that lives as long as the tensors over it."""

    def __init__(self, label, like):
        kind = {torch.float32: "<f4", torch.float16: "<f2", torch.float64: "<f8", torch.int32: "<i4"}[like.dtype]
        self.buffer = _compute.buffer(like.numel() * like.element_size(), label)
        self.__cuda_array_interface__ = {"data": (_compute.address(self.buffer), False), "shape": tuple(like.shape), "typestr": kind,
                                         "version": 3}

    def __del__(self):
        _compute.destroy(self.buffer)


class _Buffers:
    """The inputs of a case in buffers of the framework, and torch tensors over the same memory."""

    def __init__(self, inputs):
        self.at, self.tensor = {}, {}
        for name, t in inputs.items():
            if name in ("sees", "depth") or t is None:
                continue
            pairs = [self.place(name, x) for x in (t.unbind(0) if name == "rings" else [t])]
            self.at[name], self.tensor[name] = ([p[i] for p in pairs] for i in range(2))
            if name != "rings":
                self.at[name], self.tensor[name] = self.at[name][0], self.tensor[name][0]
        torch.cuda.synchronize()

    def place(self, name, t):
        view = _View(name, t)
        _compute.done()  # the new buffer's zeros come before its values
        tensor = torch.as_tensor(view, device="cuda")
        tensor.copy_(t)
        return view.buffer, tensor


# ------------------------------------------------------------------------------- the plain forms

def _rope_plain(case, s):
    rot, hd, B = case["rotary"], case["head_dim"], case["batch"]
    j = torch.arange(0, rot, 2, device="cuda").double()
    freq = torch.tensor(case["theta"], device="cuda", dtype=torch.float64) ** (-j / rot)
    if s["factors"] is not None:
        freq = freq / s["factors"].double()
    angle = s["positions"].double()[:, None] * freq
    cos = (torch.cos(angle) * case["magnitude"]).float()[:, None]
    sin = (torch.sin(angle) * case["magnitude"]).float()[:, None]
    x = s["x"][:, :case["heads"] * hd].view(B, case["heads"], hd)
    l, r = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["adjacent"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = l * cos - r * sin, l * sin + r * cos
    l.copy_(a)
    r.copy_(b)
    return {"x": s["x"]}


def _attention_plain(case, s):
    n, heads, kvh, hd = case["nodes"], case["heads"], case["kv_heads"], case["head_dim"]
    at = _slots(case)
    k, v = (s[m][at].float().transpose(0, 1).contiguous() for m in "kv")  # [kvh][keys][hd]
    q = s["q"].view(n, kvh, heads // kvh, hd).permute(1, 2, 0, 3).reshape(kvh, -1, hd)
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).view(kvh, -1, n, at.numel()) * case["scale"]
    pos = case["start"] + s["depth"]
    key = torch.arange(at.numel(), device="cuda") + (case["start"] + n - at.numel())
    valid = s["sees"].diagonal()
    cached = valid[:, None] & (key[None, :-n] > pos[:, None] - case["window"])
    drafted = s["sees"] & (pos[None] > pos[:, None] - case["window"])
    mask = torch.cat([cached, drafted], 1)
    scores = scores.masked_fill(~mask, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = torch.where(mask, p, torch.zeros((), device="cuda"))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(kvh, -1, at.numel()), v).view(kvh, -1, n, hd) / total
    o = torch.where(valid[:, None], o, torch.zeros((), device="cuda"))
    return {"y": o.permute(2, 0, 1, 3).reshape(n, heads, hd)}


def _sample_plain(case, s):
    top, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    if case["temperature"] == 0:
        return {"tokens": order[:, 0].to(torch.int32)}
    K = min(case["top_k"] or case["vocab"], case["vocab"])
    top, order = top[:, :K].double(), order[:, :K]
    p = torch.exp((top - top[:, :1]) / case["temperature"])
    cum = torch.cumsum(p, 1)
    before = cum / cum[:, -1:] < case["top_p"]  # a prefix; the first one outside it stays
    kept = torch.minimum(before.sum(1) + 1, (p >= case["min_p"]).sum(1)).clamp(max=K)
    target = s["uniforms"][:, None] * cum.gather(1, kept[:, None] - 1)
    at = (cum < target).sum(1, keepdim=True)
    return {"tokens": order.gather(1, at)[:, 0].to(torch.int32)}


def _accept_plain(case, s):
    n, parents = case["nodes"], s["parents"].long()
    up = parents.clamp(min=0)
    hit = (parents >= 0) & (s["drafted"] == s["picked"][up])
    index = torch.arange(n, device="cuda")
    first = torch.full((n,), n, device="cuda").scatter_reduce(0, up, torch.where(hit, index, n), "amin")
    ok = (index == 0) | (hit & (first[up] == index))
    taken = s["sees"][:, 0] & ~(s["sees"] & ~ok).any(1)
    count = taken.sum()
    nodes = torch.sort(torch.where(taken, index, n)).values
    path = torch.cat([count[None], s["picked"][(torch.where(taken, index, 0)).amax()][None], torch.where(nodes < n, nodes, -1)])
    return {"path": path.to(torch.int32)}


def _commit_plain(case, s):
    n, rings = case["nodes"], s["rings"]
    j = torch.arange(n, device="cuda")
    source = torch.where(j < s["path"][0], s["path"][2:], j)
    rings[:, (case["start"] + j) % case["capacity"]] = rings[:, (case["start"] + source) % case["capacity"]]
    return {"rings": list(rings.unbind(0))}


_PLAIN = {"rope": _rope_plain, "attention": _attention_plain, "sample": _sample_plain, "accept": _accept_plain, "commit": _commit_plain}


# ------------------------------------------------------------------------------- the framework's operators

def _own(case, s):
    c, b, t, kind = _compute, s.at, s.tensor, case["kind"]
    if kind == "rope":
        c.rope_at(b["x"], b["positions"], case["heads"], case["head_dim"], case["theta"], 1.0, case["rotary"], case["batch"],
                  adjacent=case["adjacent"], factors=b.get("factors"), magnitude=case["magnitude"], stride=case["stride"])
        return {"x": t["x"]}
    if kind == "attention":
        op = c.attention_tree if case["kv"] == "f32" else c.attention_tree_f16kv
        op(b["q"], b["k"], b["v"], b["y"], b["parents"], case["heads"], case["kv_heads"], case["head_dim"], case["start"],
           case["scale"], case["window"], case["capacity"], case["nodes"])
        return {"y": t["y"]}
    if kind == "sample":
        c.sample_rows(b["logits"], case["vocab"], case["rows"], b["uniforms"], b["tokens"], case["temperature"], case["top_k"],
                      case["top_p"], case["min_p"])
        return {"tokens": t["tokens"]}
    if kind == "accept":
        c.tree_accept(b["parents"], b["drafted"], b["picked"], b["path"], case["nodes"])
        return {"path": t["path"]}
    size = 4 if case["kv"] == "f32" else 2
    c.kv_commit(b["rings"], b["path"], size * case["row"], case["start"], case["capacity"], case["nodes"])
    return {"rings": t["rings"]}


# ------------------------------------------------------------------------------- the interface

def _full(case):
    return dict(case, scale=1 / math.sqrt(case["head_dim"])) if case["kind"] == "attention" else case


def prepare(case, seed):
    if own:
        _connect()
    inputs = _INPUTS[case["kind"]](case, seed)
    return _full(case), _Buffers(inputs) if own else inputs


def run(state):
    case, held = state
    return _own(case, held) if own else _PLAIN[case["kind"]](case, held)


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["batch"] * case["heads"] * case["rotary"]
        return {"bytes": 8.0 * n + 4.0 * case["batch"], "flops": 3.0 * n}
    if kind == "attention":
        n, size = case["nodes"], 4 if case["kv"] == "f32" else 2
        keys = min(case["start"], case["window"] - 1)
        # at least the cached keys of its window and itself, for every node that is no padding
        return {"bytes": 2.0 * (keys + n) * case["kv_heads"] * case["head_dim"] * size + 8.0 * n * case["heads"] * case["head_dim"] + 4.0 * n,
                "flops": 4.0 * (n - case["pad"]) * (keys + 1) * case["heads"] * case["head_dim"]}
    if kind == "sample":
        return {"bytes": case["rows"] * (4.0 * case["vocab"] + 12), "flops": 2.0 * case["rows"] * case["vocab"]}
    if kind == "accept":
        return {"bytes": 16.0 * case["nodes"] + 8, "flops": 2.0 * case["nodes"]}
    size = 4 if case["kv"] == "f32" else 2
    return {"bytes": 4.0 * case["layers"] * max(1, case["accepted"] - 1) * case["row"] * size, "flops": 0.0}


def exact(case, seed):
    case, s = _full(case), _INPUTS[case["kind"]](case, seed)
    kind = case["kind"]
    if kind == "rope":
        x, rot, hd = s["x"].double(), case["rotary"], case["head_dim"]
        for i in range(rot // 2):
            turn = s["positions"].double() * math.exp(-2 * i / rot * math.log(case["theta"]))
            if s["factors"] is not None:
                turn = turn / float(s["factors"][i])
            z = torch.polar(torch.full_like(turn, case["magnitude"]), turn)[:, None]
            a, b = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + rot // 2)
            h = torch.arange(case["heads"], device="cuda") * hd
            w = torch.complex(x[:, h + a], x[:, h + b]) * z
            x[:, h + a], x[:, h + b] = w.real, w.imag
        return {"x": x}
    if kind == "attention":
        y = torch.zeros(case["nodes"], case["heads"], case["head_dim"], dtype=torch.float64, device="cuda")
        parents, group = s["parents"].tolist(), case["heads"] // case["kv_heads"]
        cached = torch.arange(max(0, case["start"] + 1 - case["window"]), case["start"], device="cuda") % case["capacity"]
        own_at = [(case["start"] + i) % case["capacity"] for i in range(case["nodes"])]
        k, v = s["k"].double(), s["v"].double()
        kc, vc = k[cached], v[cached]
        for i in range(case["nodes"]):
            if parents[i] < -1:
                continue
            chain, a = [], i
            while a >= 0:
                chain.append(a)
                a = parents[a]
            hidden = min(len(cached), max(0, len(chain) + case["start"] - case["window"] - (case["start"] - len(cached))))
            tree = torch.tensor([own_at[a] for a in chain[:case["window"]]], device="cuda")
            ki, vi = (torch.cat([c[hidden:], r[tree]]).repeat_interleave(group, 1) for c, r in ((kc, k), (vc, v)))
            p = torch.softmax((ki * s["q"][i].double()).sum(-1) * case["scale"], 0)
            y[i] = (p[..., None] * vi).sum(0)
        return {"y": y}
    if kind == "commit":
        rings, path = s["rings"].double(), s["path"].tolist()
        for j, node in enumerate(path[2:2 + path[0]]):
            rings[:, (case["start"] + j) % case["capacity"]] = rings[:, (case["start"] + node) % case["capacity"]].clone()
        return {"rings": list(rings.unbind(0))}
    return None
