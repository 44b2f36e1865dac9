"""The operators of a decode step of many requests, as a list of timed cases.

Requests keep their keys and values in pages of one pool per layer, and requests that come from one another share
pages. Beside the products, rotary positions and draws that the framework has for batches, a step of such a
batch takes: places in the pages for the new tokens and the move of their keys and values there, a batch that
forks (beams, several answers to one prompt) or drops requests, pools that are compacted, attention of every
request over its own pages with a prefix that many share computed once, and low-rank adapters, each
request's own, beside a projection that all share.

Where ``own`` is false, ``run`` computes these with plain torch; where it is true, with the framework's operators on
the framework's buffers. ``exact`` restates what is computed in float64.
"""
import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------------------- the cases

def listed():
    return [
        # eight chats of the small model, four drafted tokens each, all of them rejected: the launches count
        {"name": "draft_0.6b", "kind": "draft", "requests": 8, "tokens": 4, "shortest": 40, "longest": 900, "page": 16,
         "max_pages": 64, "pages": 700, "row": 1024, "kv": "f32"},
        # a chunk of 512 tokens for each of eight prompts of the 8B model, ragged at their ends
        {"name": "draft_prompts_8b", "kind": "draft", "requests": 8, "tokens": 512, "shortest": 0, "longest": 4000, "page": 32,
         "max_pages": 256, "pages": 1200, "row": 1024, "kv": "f16"},
        # eight beams of the small model, four of which go on twice
        {"name": "fork_beams_0.6b", "kind": "fork", "requests": 8, "shortest": 300, "longest": 300, "page": 16, "max_pages": 64,
         "pages": 256, "row": 1024, "pools": 56, "heirs": 2, "freed": 0, "kv": "f32"},
        # a batch of the 8B model deep in long documents: one in four starts three others, some end
        {"name": "fork_long_8b", "kind": "fork", "requests": 64, "shortest": 3000, "longest": 16000, "page": 64, "max_pages": 256,
         "pages": 12000, "row": 128, "pools": 2, "heirs": 4, "freed": 3, "kv": "f16"},
        # a small pool after a few chats ended
        {"name": "compact_small", "kind": "compact", "requests": 8, "max_pages": 64, "pages": 128, "used": 70, "page": 16, "row": 1024,
         "pools": 8, "kv": "f32"},
        # the pool of a layer of the 8B model, half of it free in between
        {"name": "compact_8b", "kind": "compact", "requests": 64, "max_pages": 128, "pages": 4000, "used": 2100, "page": 32,
         "row": 1024, "pools": 2, "kv": "f16"},
        # four chats of the small model
        {"name": "attend_0.6b", "kind": "attention", "heads": 16, "kv_heads": 8, "head_dim": 128, "requests": 4, "tokens": 1, "empty": 0,
         "shared": 0, "strangers": 0, "shortest": 40, "longest": 500, "page": 16, "window": 1 << 30, "kv": "f32"},
        # a ragged batch of the 8B model, one row of it unused
        {"name": "attend_ragged_8b", "kind": "attention", "heads": 32, "kv_heads": 8, "head_dim": 128, "requests": 32, "tokens": 1,
         "empty": 1, "shared": 0, "strangers": 0, "shortest": 100, "longest": 4000, "page": 32, "window": 1 << 30, "kv": "f16"},
        # sixty-four questions about one long document, and two requests without it
        {"name": "attend_prefix_8b", "kind": "attention", "heads": 32, "kv_heads": 8, "head_dim": 128, "requests": 66, "tokens": 1,
         "empty": 0, "shared": 8192, "strangers": 2, "shortest": 10, "longest": 1000, "page": 64, "window": 1 << 30, "kv": "f16"},
        # three chats of the small model with adapters of rank 8 and one without, at the query projection
        {"name": "adapt_0.6b", "kind": "adapters", "batch": 4, "adapters": 3, "rank": 8, "cols": 1024, "rows": 2048, "run": 1, "type": "f32"},
        # a batch of the 8B model with two dozen adapters at the gate projection
        {"name": "adapt_mixed_8b", "kind": "adapters", "batch": 64, "adapters": 24, "rank": 16, "cols": 4096, "rows": 14336, "run": 1,
         "type": "f16"},
        # four prompts of 512 tokens of the 8B model, three of them with an adapter of rank 64 each, at the output projection
        {"name": "adapt_prompts_8b", "kind": "adapters", "batch": 2048, "adapters": 4, "rank": 64, "cols": 4096, "rows": 4096, "run": 512,
         "type": "f16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["draft", "fork", "compact", "attention", "attention", "attention", "attention", "adapters", "adapters", "adapters"])
    kv = rng.choice(["f32", "f16"])
    if kind == "draft":
        R, T, page = _spread(rng, 1, 128), rng.choice([1, 1, _spread(rng, 2, 512)]), 1 << rng.randint(0, 7)
        while R * T > 2048:
            R, T = max(1, R // 2), max(1, T * 2 // 3)
        longest = max(1, min(_spread(rng, 1, 8000), 50000 // R))
        width = -(-(longest + T) // page) + rng.randint(0, 3)
        return {"kind": kind, "requests": R, "tokens": T, "shortest": rng.randint(0, longest), "longest": longest, "page": page,
                "max_pages": width, "pages": R * width + rng.randint(0, 50), "row": rng.choice([1, 6, 64, 100, 128, 256, 512]), "kv": kv}
    if kind == "fork":
        R, page = _spread(rng, 1, 128), 1 << rng.randint(2, 7)
        longest = max(1, min(_spread(rng, 1, 16000), 300000 // R))
        width = -(-longest // page) + rng.randint(0, 3)
        row, pools = 2 * _spread(rng, 1, 64), _spread(rng, 1, 16)
        while R * (width + 1) * page * row * pools > 1.2e7 and (row > 2 or pools > 1):
            row, pools = max(2, row // 4 * 2), max(1, pools // 2)
        return {"kind": kind, "requests": R, "shortest": rng.randint(1, longest), "longest": longest, "page": page, "max_pages": width,
                "pages": R * (width + 1), "row": row, "pools": 2 * pools,
                "heirs": rng.randint(1, 4), "freed": rng.randint(0, 3), "kv": kv}
    if kind == "compact":
        pages, page, row = _spread(rng, 2, 20000), 1 << rng.randint(2, 6), 2 * _spread(rng, 1, 512)
        while pages * page * row > 1.6e7:
            page, row = max(1, page // 2), max(2, row // 4 * 2)
        R = _spread(rng, 1, 64)
        return {"kind": kind, "requests": R, "max_pages": -(-pages // R) + rng.randint(0, 9), "pages": pages, "used": rng.randint(1, pages),
                "page": page, "row": row, "pools": 2 * rng.randint(1, 4), "kv": kv}
    if kind == "attention":
        kvh, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 3, 4, 4, 7, 8])
        hd, page = rng.choice([64, 80, 128, 128, 128, 256]), 1 << rng.randint(2, 8)
        R, T = _spread(rng, 1, 128), rng.choice([1, 1, 1, 1, 2, 5, _spread(rng, 2, 128)])
        shared, longest = rng.choice([0, 0, _spread(rng, 64, 16000)]), _spread(rng, max(2, T), 8000)
        while R * T * kvh * group * (shared + longest) * hd > 2.2e9 or (shared + R * longest) * kvh * hd > 2e7 \
                or R * (shared + longest) * kvh * hd > 6e8:
            if R > 8 or (R > 1 and T == 1 and longest <= 16):
                R //= 2
            else:
                T, longest, shared = max(1, T // 2), max(2, T // 2, longest * 2 // 3), shared * 2 // 3
        shared = shared // page * page if R > 1 else 0
        return {"kind": kind, "heads": kvh * group, "kv_heads": kvh, "head_dim": hd, "requests": R, "tokens": T,
                "empty": rng.choice([0, 0, min(1, R - 1)]), "shared": shared, "strangers": rng.choice([0, 0, min(2, R - 1)]) if shared else 0,
                "shortest": rng.randint(T, max(T, longest)), "longest": max(T, longest), "page": page,
                "window": rng.choice([1 << 30, 1 << 30, 1 << 30, _spread(rng, 1, 4096)]), "kv": kv}
    cols, rows, rank = 8 * _spread(rng, 8, 1792), 8 * _spread(rng, 8, 1792), rng.choice([1, 4, 8, 16, 16, 32, 64, _spread(rng, 2, 128)])
    batch, adapters = _spread(rng, 1, 2048), _spread(rng, 1, 64)
    while batch * (cols + rows) > 1.2e7 or batch * rank * (cols + rows) > 1e9:
        batch = batch * 2 // 3
    while adapters * rank * (cols + rows) > 1.2e7:
        adapters = adapters * 2 // 3
    return {"kind": "adapters", "batch": max(1, batch), "adapters": max(1, adapters), "rank": rank, "cols": cols + rng.choice([0, 0, 0, 1, 4]),
            "rows": rows + rng.choice([0, 0, 0, 1, 4]), "run": rng.choice([1, 1, _spread(rng, 2, 512)]), "type": kv}


# ------------------------------------------------------------------------------- inputs

def _gen(seed, tag):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1_000_003 + tag * 7919 + 31) & 0x7FFFFFFFFFFF)


def _up(a, kind=np.int32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, kind))).cuda()


def _ragged(n, lo, hi):
    """n whole numbers of [lo, hi] that go through it unevenly; the first is the largest."""
    turns = (1 - 1e-9 - np.arange(n) * 0.6180339887498949) % 1.0
    return (lo + np.floor(turns * (hi - lo + 1))).astype(np.int64)


def _half(case):
    return torch.float16 if case["kv"] == "f16" else torch.float32


def _pools(case, seed, n):
    return torch.randn(n, case["pages"], case["page"] * case["row"], generator=_gen(seed, 9), device="cuda").to(_half(case))


def _tables(lengths, page, width, pages, seed):
    """Rows of pages that no two requests share, in no order, and the pages' counts of holders."""
    order = np.random.default_rng(seed).permutation(pages)
    table, refs, at = np.full((len(lengths), width), -1), np.zeros(pages), 0
    for r, n in enumerate(-(-np.asarray(lengths) // page)):
        table[r, :n] = order[at:at + n]
        refs[order[at:at + n]] = 1
        at += n
    return table, refs


def _draft_inputs(case, seed):
    R, T, row = case["requests"], case["tokens"], case["row"]
    lengths = _ragged(R, case["shortest"], case["longest"])
    table, refs = _tables(lengths, case["page"], case["max_pages"], case["pages"], seed)
    pools = _pools(case, seed, 2)
    qkv = torch.randn(R * T, 3 * row, generator=_gen(seed, 1), device="cuda")  # query, key and value side by side
    return {"table": _up(table), "lengths": _up(lengths), "refs": _up(refs), "counts": _up(_ragged(R, 1, T)), "origin": _up(np.arange(R)),
            "keep": _up(lengths), "qkv": qkv, "k": pools[0].clone(), "v": pools[1].clone(), "added": _up(np.zeros(R)),
            "positions": _up(np.zeros(R * T)), "slots": _up(np.zeros(R * T)), "copies": _up(np.zeros(1 + 2 * R))}


def _fork_inputs(case, seed):
    R = case["requests"]
    lengths = _ragged(R, case["shortest"], case["longest"])
    table, refs = _tables(lengths, case["page"], case["max_pages"], case["pages"], seed)
    origin = np.arange(R) // case["heirs"] * case["heirs"]  # the first of every few goes on as all of them
    origin[R - min(case["freed"], R - 1):] = -1
    keep = np.maximum(1, lengths[origin] - np.random.default_rng(seed + 1).integers(0, 2, R) * (np.arange(R) % 3))
    keep[origin == np.arange(R)] = lengths[origin == np.arange(R)]
    return {"table": _up(table), "lengths": _up(lengths), "refs": _up(refs), "origin": _up(origin), "keep": _up(keep),
            "copies": _up(np.zeros(1 + 2 * R)), "pools": _pools(case, seed, case["pools"])}


def _compact_inputs(case, seed):
    rng, R, W = np.random.default_rng(seed), case["requests"], case["max_pages"]
    used = rng.permutation(case["pages"])[:case["used"]]
    refs, table = np.zeros(case["pages"]), np.full(R * W, -1)
    refs[used] = 1
    table[rng.permutation(R * W)[:min(R * W, case["used"])]] = used[:R * W]
    again = rng.integers(0, R * W, R)  # a few pages that a second request holds
    again = again[table[again] < 0]
    table[again] = used[rng.integers(0, min(R * W, case["used"]), len(again))]
    np.add.at(refs, table[again], 1)
    return {"table": _up(table.reshape(R, W)), "refs": _up(refs), "table_to": _up(np.zeros((R, W))), "refs_to": _up(np.zeros(case["pages"])),
            "moved": _up(np.zeros(case["pages"])), "copies": _up(np.zeros(1 + case["pages"] // 2 * 2)),
            "pools": _pools(case, seed, case["pools"])}


def _sizes(case):
    """Lengths of the requests and how many tokens each of them asks for; which ones share the prefix."""
    R = case["requests"]
    own_tokens = _ragged(R, case["shortest"], case["longest"])
    shares = np.arange(R) < R - case["strangers"]
    lengths = own_tokens + np.where(shares, case["shared"], 0)
    counts = np.minimum(_ragged(R, 1, case["tokens"]), own_tokens)
    if case["empty"]:
        lengths[1:1 + case["empty"]] = counts[1:1 + case["empty"]] = 0
    return lengths, counts, shares & (lengths > 0)


def _attention_inputs(case, seed):
    lengths, counts, shares = _sizes(case)
    R, page, first = case["requests"], case["page"], case["shared"] // case["page"]
    held = -(-lengths // page)
    pages, width = int(first + held.sum() + 3), int(held.max()) + 2
    order = np.random.default_rng(seed).permutation(pages)
    table, at = np.full((R, width), -1), first
    for r in range(R):
        skip = first if shares[r] else 0
        table[r, :skip] = order[:skip]
        table[r, skip:held[r]] = order[at:at + held[r] - skip]
        at += held[r] - skip
    q = torch.randn(R, case["tokens"], case["heads"], case["head_dim"], generator=_gen(seed, 0), device="cuda") * 1.5
    k, v = (torch.randn(pages, page, case["kv_heads"], case["head_dim"], generator=_gen(seed, 1 + i), device="cuda").to(_half(case))
            for i in range(2))
    return {"q": q, "k": k, "v": v, "y": torch.zeros_like(q), "table": _up(table), "lengths": _up(lengths), "counts": _up(counts)}


def _which(case):
    """The adapter of every row: runs of one, every seventh run without."""
    i = np.arange(case["batch"]) // case["run"]
    return np.where(i % 7 == 3, -1, (i * 5 + i // 3) % case["adapters"])


def _adapters_inputs(case, seed):
    kind = torch.float16 if case["type"] == "f16" else torch.float32
    n, rank = case["adapters"], case["rank"]
    a = (torch.randn(n, rank, case["cols"], generator=_gen(seed, 0), device="cuda") / math.sqrt(case["cols"])).to(kind)
    b = (torch.randn(n, case["rows"], rank, generator=_gen(seed, 1), device="cuda") / math.sqrt(rank)).to(kind)
    return {"a": a, "b": b, "x": torch.randn(case["batch"], case["cols"], generator=_gen(seed, 2), device="cuda"),
            "y": torch.randn(case["batch"], case["rows"], generator=_gen(seed, 3), device="cuda"), "which": _up(_which(case)),
            "scales": torch.rand(n, generator=_gen(seed, 4), device="cuda") * 2}


_INPUTS = {"draft": _draft_inputs, "fork": _fork_inputs, "compact": _compact_inputs, "attention": _attention_inputs, "adapters": _adapters_inputs}


# ------------------------------------------------------------------------------- the framework's buffers

_compute = None


def _connect():
    """The framework's context. Its stream becomes torch's current one, so that what torch does with the buffers, before
    the operators run or with what they wrote, keeps its place among their launches."""
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
        kind = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4"}[like.dtype]
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
            pairs = [self.place(name, x) for x in (t.unbind(0) if name == "pools" else [t])]
            self.at[name], self.tensor[name] = ([p[i] for p in pairs] for i in range(2))
            if name != "pools":
                self.at[name], self.tensor[name] = self.at[name][0], self.tensor[name][0]
        torch.cuda.synchronize()

    def place(self, name, t):
        view = _View(name, t)
        _compute.done()  # the new buffer's zeros come before its values
        tensor = torch.as_tensor(view, device="cuda")
        tensor.copy_(t)
        return view.buffer, tensor


# ------------------------------------------------------------------------------- the plain forms

def _free(refs):
    """The pages, those that nobody holds first, each part in order."""
    return torch.sort((refs != 0).to(torch.int32), stable=True).indices


def _count(refs, pages, mask, by):
    """refs[p] += by for every page p of the masked places."""
    p = torch.where(mask, pages, 0).reshape(-1).long()
    refs.index_add_(0, p, torch.where(mask, by, 0).reshape(-1).to(torch.int32))


def _extend_plain(case, s):
    page, T = case["page"], case["tokens"]
    table, lengths, counts = s["table"], s["lengths"].long(), s["counts"].long()
    have, want = (lengths + page - 1) // page, (lengths + counts + page - 1) // page
    first = torch.cumsum(want - have, 0) - want  # rank of column c of request r among the pages taken: first + c
    col = torch.arange(case["max_pages"], device="cuda")[None]
    new = (col >= have[:, None]) & (col < want[:, None])
    ids = _free(s["refs"])[(first[:, None] + col).clamp(0, case["pages"] - 1)].to(torch.int32)
    table.copy_(torch.where(new, ids, table))
    _count(s["refs"], table, new, 1)
    t = torch.arange(T, device="cuda")[None]
    at, there = lengths[:, None] + t, t < counts[:, None]
    at = torch.where(there, at, 0)
    slot = table.gather(1, at // page).long() * page + at % page
    s["positions"].copy_(torch.where(there, at, -1).reshape(-1))
    s["slots"].copy_(torch.where(there, slot, -1).reshape(-1))
    s["added"].copy_(counts)
    s["lengths"].copy_(lengths + counts)


def _store_plain(case, s):
    row = case["row"]
    there = s["slots"] >= 0
    at = s["slots"][there].long()
    for i, name in enumerate("kv"):
        s[name].view(-1, row)[at] = s["qkv"][there, (1 + i) * row:(2 + i) * row].to(s[name].dtype)


def _fork_plain(case, s):
    page, R = case["page"], case["requests"]
    old, lengths, origin = s["table"].clone(), s["lengths"].long(), s["origin"].long()
    col, me = torch.arange(case["max_pages"], device="cuda")[None], torch.arange(R, device="cuda")
    src = origin.clamp(min=0)
    kept = torch.where(origin >= 0, torch.minimum(s["keep"].long(), lengths[src]), 0)
    changed = (origin != me) | (kept < lengths)
    refs = s["refs"].clone()
    _count(refs, old, changed[:, None] & (col < ((lengths + page - 1) // page)[:, None]), -1)
    full, rows = kept // page, old[src]
    _count(refs, rows, changed[:, None] & (col < full[:, None]), 1)
    last = changed & (kept % page > 0)
    p = torch.where(last, rows.gather(1, full.clamp(max=case["max_pages"] - 1)[:, None])[:, 0].long(), 0)
    heir = torch.full((case["pages"],), R, device="cuda").scatter_reduce(0, p, torch.where(last, me, R), "amin")
    stays = last & (refs[p] == 0) & (heir[p] == me)
    refs.index_add_(0, p, stays.to(torch.int32))
    copied = last & ~stays
    rank = torch.cumsum(copied, 0) - 1
    to = _free(refs)[rank.clamp(min=0)]
    refs.index_add_(0, to, copied.to(torch.int32))
    end = torch.where(copied, to, p).to(torch.int32)[:, None]
    rows = torch.where(col < full[:, None], rows, torch.where((col == full[:, None]) & last[:, None], end, -1))
    s["table"].copy_(torch.where(changed[:, None], rows, old))
    s["lengths"].copy_(torch.where(changed, kept, lengths))
    s["refs"].copy_(refs)
    pairs = torch.full((R + 1, 2), -1, dtype=torch.int64, device="cuda")
    pairs[torch.where(copied, rank, R)] = torch.stack([p, to], 1)
    s["copies"][0] = copied.sum()
    s["copies"][1:] = torch.where(me[:, None] < copied.sum(), pairs[:R], -1).reshape(-1)


def _copy_plain(pools, copies):
    pairs = copies[1:].view(-1, 2).long()
    pairs = pairs[pairs[:, 0] >= 0]
    for pool in pools:
        pool[pairs[:, 1]] = pool[pairs[:, 0]]


def _draft_plain(case, s):
    _extend_plain(case, s)
    _store_plain(case, s)
    _fork_plain(case, s)
    return {name: s[name] for name in ("table", "lengths", "refs", "added", "positions", "slots", "copies", "k", "v")}


def _fork_and_copy_plain(case, s):
    _fork_plain(case, s)
    _copy_plain(s["pools"], s["copies"])
    return {"pools": list(s["pools"].unbind(0)), **{name: s[name] for name in ("table", "lengths", "refs", "copies")}}


def _compact_plain(case, s):
    refs, n = s["refs"], case["pages"]
    page, used = torch.arange(n, device="cuda"), refs > 0
    count = used.sum()
    move, hole = used & (page >= count), ~used & (page < count)
    src, dst = page[move], page[hole]
    to = torch.where(used, page, -1)
    to[src] = dst
    s["moved"].copy_(to)
    table = s["table"]
    there = (table >= 0) & (table < n)
    s["table_to"].copy_(torch.where(there, to[table.clamp(0, n - 1).long()].to(torch.int32), table))
    after = torch.where(move, 0, refs)
    after[dst] = refs[src]
    s["refs_to"].copy_(after)
    s["copies"].fill_(-1)
    s["copies"][0] = src.numel()
    s["copies"][1:1 + 2 * src.numel()] = torch.stack([src, dst], 1).reshape(-1).to(torch.int32)
    _copy_plain(s["pools"], s["copies"])
    return {"pools": list(s["pools"].unbind(0)), **{name: s[name] for name in ("table_to", "refs_to", "moved", "copies")}}


def _attention_plain(case, s):
    R, T, H, kvh, hd, page = (case[n] for n in ("requests", "tokens", "heads", "kv_heads", "head_dim", "page"))
    lengths, counts = s["lengths"].long(), s["counts"].long()
    width = s["table"].shape[1]
    k, v = (s[m][s["table"].clamp(min=0).long()].view(R, width * page, kvh, hd).permute(0, 2, 1, 3).float().reshape(R * kvh, -1, hd) for m in "kv")
    q = s["q"].view(R, T, kvh, H // kvh, hd).permute(0, 2, 1, 3, 4).reshape(R * kvh, -1, hd)
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).view(R, kvh, T, H // kvh, width * page) * case["scale"]
    t, key = torch.arange(T, device="cuda")[None, :, None], torch.arange(width * page, device="cuda")[None, None]
    pos = (lengths - counts)[:, None, None] + t
    mask = ((t < counts[:, None, None]) & (key <= pos) & (key > pos - case["window"]))[:, None, :, None]
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(mask, torch.exp(scores - torch.where(top == -math.inf, 0, top)), torch.zeros((), device="cuda"))
    total = p.sum(-1, keepdim=True)
    y = torch.bmm(p.view(R * kvh, -1, width * page), v).view(R, kvh, T, H // kvh, hd) / torch.where(total > 0, total, 1)
    return {"y": y.permute(0, 2, 1, 3, 4).reshape(R, T, H, hd)}


def _adapters_plain(case, s):
    for w in range(case["adapters"]):
        at = torch.nonzero(s["which"] == w)[:, 0]
        h = torch.mm(s["x"][at], s["a"][w].float().t())
        s["y"][at] += s["scales"][w] * torch.mm(h, s["b"][w].float().t())
    return {"y": s["y"]}


_PLAIN = {"draft": _draft_plain, "fork": _fork_and_copy_plain, "compact": _compact_plain, "attention": _attention_plain,
          "adapters": _adapters_plain}


# ------------------------------------------------------------------------------- the framework's operators

def _own(case, s):
    c, b, t, kind = _compute, s.at, s.tensor, case["kind"]
    half = case.get("kv") == "f16"
    if kind == "draft":
        R, T, row, shape = case["requests"], case["tokens"], case["row"], (case["page"], case["max_pages"], case["pages"])
        c.pages_extend(b["table"], b["lengths"], b["refs"], b["added"], b["positions"], b["slots"], R, T, *shape, counts=b["counts"])
        store = c.pages_store_f16kv if half else c.pages_store
        store(b["qkv"], b["qkv"], b["k"], b["v"], b["slots"], row, R * T, case["pages"] * case["page"], stride=3 * row, k_offset=row,
              v_offset=2 * row)
        c.pages_fork(b["table"], b["lengths"], b["refs"], b["origin"], b["copies"], R, *shape, keep=b["keep"])
        return {name: t[name] for name in ("table", "lengths", "refs", "added", "positions", "slots", "copies", "k", "v")}
    bytes_ = case.get("page", 0) * case.get("row", 0) * (2 if half else 4)
    if kind == "fork":
        c.pages_fork(b["table"], b["lengths"], b["refs"], b["origin"], b["copies"], case["requests"], case["page"], case["max_pages"],
                     case["pages"], keep=b["keep"])
        c.pages_copy(b["pools"], b["copies"], case["requests"], bytes_, case["pages"])
        return {"pools": t["pools"], **{name: t[name] for name in ("table", "lengths", "refs", "copies")}}
    if kind == "compact":
        c.pages_compact(b["table"], b["refs"], b["table_to"], b["refs_to"], b["moved"], b["copies"], case["requests"], case["max_pages"],
                        case["pages"])
        c.pages_copy(b["pools"], b["copies"], case["pages"] // 2, bytes_, case["pages"])
        return {"pools": t["pools"], **{name: t[name] for name in ("table_to", "refs_to", "moved", "copies")}}
    if kind == "attention":
        pages, width = t["k"].shape[0], t["table"].shape[1]
        (c.attention_pages_f16kv if half else c.attention_pages)(
            b["q"], b["k"], b["v"], b["y"], b["table"], b["lengths"], case["heads"], case["kv_heads"], case["head_dim"], case["scale"],
            case["window"], case["page"], width, pages, case["requests"], case["tokens"], counts=b["counts"], shared=case["shared"], owner=0)
        return {"y": t["y"]}
    c.adapters(1 if case["type"] == "f16" else 0, b["a"], b["b"], b["which"], b["scales"], b["x"], b["y"], case["cols"], case["rows"],
               case["rank"], case["adapters"], case["rows"], 0, case["batch"])
    return {"y": t["y"]}


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
    kind, size = case["kind"], 2 if case.get("kv", case.get("type")) == "f16" else 4
    if kind == "draft":
        R, T = case["requests"], case["tokens"]
        n, held = float(_ragged(R, 1, T).sum()), float((-(-_ragged(R, case["shortest"], case["longest"]) // case["page"])).sum())
        return {"bytes": n * case["row"] * 2 * (4 + size) + 8.0 * R * T + 8.0 * held + 24.0 * R, "flops": 0.0}
    if kind == "fork":
        R, page = case["requests"], case["page"]
        lengths, origin = _ragged(R, case["shortest"], case["longest"]), np.arange(R) // case["heirs"] * case["heirs"]
        live = np.arange(R) < R - min(case["freed"], R - 1)
        heirs = live & (origin != np.arange(R))
        moved = float((heirs & (lengths[origin] % page > 0)).sum()) * page * case["row"] * size * case["pools"]
        return {"bytes": 2 * moved + 16.0 * float((-(-lengths[origin] // page))[heirs].sum()) + 16.0 * R, "flops": 0.0}
    if kind == "compact":
        moved = case["used"] * (1 - case["used"] / case["pages"])  # of pages used at random, those behind the first `used`
        return {"bytes": 2.0 * moved * case["page"] * case["row"] * size * case["pools"] + 8.0 * case["requests"] * case["max_pages"]
                + 12.0 * case["pages"] + 8.0 * moved, "flops": 0.0}
    if kind == "attention":
        lengths, counts, shares = _sizes(case)
        seen = np.minimum(lengths, case["window"] + counts - 1) * (counts > 0)
        asked = np.minimum(lengths - (counts - 1) / 2, case["window"]) * counts
        once = seen.sum() - (max(0, int(shares.sum()) - 1) * case["shared"] if case["window"] >= lengths.max() else 0)
        return {"bytes": 2.0 * float(once) * case["kv_heads"] * case["head_dim"] * size
                + 8.0 * case["requests"] * case["tokens"] * case["heads"] * case["head_dim"],
                "flops": 4.0 * float(asked.sum()) * case["heads"] * case["head_dim"]}
    w = _which(case)
    n, kinds = float((w >= 0).sum()), len(set(w[w >= 0]))
    both = case["cols"] + case["rows"]
    return {"bytes": kinds * case["rank"] * both * float(size) + 4.0 * n * (both + case["rows"]), "flops": 2.0 * n * case["rank"] * both}


def exact(case, seed):
    if case["kind"] not in ("attention", "adapters"):
        return None
    case, s = _full(case), _INPUTS[case["kind"]](case, seed)
    if case["kind"] == "adapters":
        y = s["y"].double()
        for i, w in enumerate(s["which"].tolist()):
            if w >= 0:
                y[i] += float(s["scales"][w]) * (s["b"][w].double() @ (s["a"][w].double() @ s["x"][i].double()))
        return {"y": y}
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lengths, counts, _ = _sizes(case)
    group = case["heads"] // case["kv_heads"]
    for r in range(case["requests"]):
        n, asked = int(lengths[r]), int(counts[r])
        ids = s["table"][r, :-(-n // case["page"])].long()
        k, v = (s[m][ids].reshape(-1, case["kv_heads"], case["head_dim"])[:n].double() for m in "kv")
        end = torch.arange(n - asked, n, device="cuda")[:, None] + 1
        key = torch.arange(n, device="cuda")[None]
        hidden = ((key >= end) | (key < end - case["window"]))[:, None]
        for h in range(case["kv_heads"] if asked else 0):
            score = s["q"][r, :asked, h * group:(h + 1) * group].double() @ k[:, h].t() * case["scale"]
            y[r, :asked, h * group:(h + 1) * group] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[:, h]
    return {"y": y}
