"""The operators that serve a batch of continuations from one paged cache, as they
are timed: their inputs, a plain form of each, and the same in 64 bits.

A server that answers several requests over one long prompt keeps the keys and
values in pages.  A page is [kv_heads, page, head_dim] f16 in each of a pool's
planes (keys and values of every layer); a slot (a sequence in the batch) names
its pages in a row of the table and its length in ``lens`` (-1: not in use);
``refs`` counts the slots that hold a page.  A step of the batch is

* ``append``: rotary embedding of the step's queries and keys, each row at its
  own position, and the new keys and values written to their pages;
* ``attn``: attention of the step's queries over the pages, those that all slots
  share read once for all;
* ``softmax``: the logits' probabilities at each request's temperature;
* ``verify``: drafted tokens kept or refused by the target's probabilities and
  given random numbers, and the token that follows;
* ``pages``: slots freed, forked and given room, or the pool's pages moved
  together.

Shapes are those of the repository's decoder configurations (Qwen2.5-0.5B heads
14 / 2 of 64, vocabulary 151936; Llama-3-8B heads 32 / 8 of 128, vocabulary
128256) and generic ones between them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

SLAB_BYTES = 64 << 20   # scratch that a serving program keeps for its calls
THETA = 1e6
_ctx = None


def _hip():
    """The process's context, on torch's current stream as a torch program runs it."""
    global _ctx
    if _ctx is None:
        from cima_amd.hip import HipCtx

        _ctx = HipCtx(0)
    _ctx.use_torch_stream()
    return _ctx


# -------------------------------------------------------------------- cases

def _attn(name, seqs, n_new, q_heads, kv_heads, dim, page, prefix, own_max, window=0):
    c = {"op": "attn", "seqs": seqs, "n_new": n_new, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
         "page": page, "prefix": prefix, "own_max": own_max, "window": window}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few answers to one question by the small model: what a step costs in latency
        _attn("attn few", 4, 1, 14, 2, 64, 16, 512, 61),
        # a batch of samples over one document
        _attn("attn batch", 32, 1, 32, 8, 128, 64, 8000, 1023),
        # a full batch over a very long document
        _attn("attn long", 128, 1, 32, 8, 128, 128, 65536, 500),
        # drafted tokens checked in one step, with a sliding window that ends inside the prefix
        _attn("attn drafts", 24, 5, 14, 2, 64, 32, 4096, 700, 4000),
        # rotary embedding and cache write of one token of a few slots, and of drafts of a large batch
        {"name": "append few", "op": "append", "seqs": 4, "n_new": 1, "q_heads": 14, "kv_heads": 2, "dim": 64,
         "page": 16, "max_pos": 4000},
        {"name": "append drafts", "op": "append", "seqs": 256, "n_new": 8, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "max_pos": 120000},
        # eight more answers branch off a running one: slots freed, forked and given room
        {"name": "pages branch", "op": "branch", "layers": 24, "kv_heads": 2, "dim": 64, "page": 16, "pages": 1024,
         "forks": 8, "length": 4003, "room": 20},
        # the pool's live pages moved together after requests ended
        {"name": "pages compact", "op": "compact", "layers": 16, "kv_heads": 8, "dim": 128, "page": 64, "pages": 250,
         "seqs": 40, "length": 550},
        # one request sampled, and every row of a batch with drafts
        {"name": "softmax one", "op": "softmax", "reqs": 1, "rows": 1, "vocab": 151936, "f32": False, "cap": 0.0},
        {"name": "softmax batch", "op": "softmax", "reqs": 64, "rows": 6, "vocab": 128256, "f32": False, "cap": 0.0},
        {"name": "verify few", "op": "verify", "seqs": 2, "drafts": 3, "vocab": 151936, "greedy": False},
        {"name": "verify batch", "op": "verify", "seqs": 192, "drafts": 5, "vocab": 128256, "greedy": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "append", "pages", "softmax", "verify"])
    heads = rng.choice([(14, 2, 64), (32, 8, 128), (28, 4, 128), (12, 12, 64), (16, 1, 128), (24, 8, 64)])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "attn":
        seqs, n_new = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 3, 5, 8])
        prefix = _log(rng, 16, 65536) if rng.random() < 0.85 else 0
        while seqs * n_new * heads[0] * heads[2] * prefix > 128 * 32 * 128 * 65536:  # no dearer than the largest
            prefix = prefix * 3 // 4
        window = _log(rng, 30, 2 * (prefix + 500)) if rng.random() < 0.25 else 0
        return _attn(None, seqs, n_new, *heads, page, prefix // page * page, _log(rng, 2, 2000), window)
    if op == "append":
        return {"op": "append", "seqs": _log(rng, 1, 256), "n_new": rng.randint(1, 8), "q_heads": heads[0],
                "kv_heads": heads[1], "dim": heads[2], "page": page, "max_pos": _log(rng, 1000, 120000)}
    if op == "pages":
        layers, page = rng.randint(2, 16), min(page, 64)
        if rng.random() < 0.5:
            forks, length = rng.randint(1, 16), _log(rng, 3, 4000)
            return {"op": "branch", "layers": layers, "kv_heads": heads[1], "dim": heads[2], "page": page,
                    "pages": -(-length // page) + 40 + rng.randint(4, 20) * forks, "forks": forks, "length": length,
                    "room": rng.randint(1, 3 * page)}
        return {"op": "compact", "layers": layers, "kv_heads": min(heads[1], 8), "dim": heads[2], "page": page,
                "pages": rng.randint(40, 250), "seqs": rng.randint(2, 40), "length": _log(rng, 30, 550)}
    if op == "softmax":
        rows = rng.randint(1, 6)
        return {"op": "softmax", "reqs": _log(rng, 1, 64), "rows": rows, "vocab": _log(rng, 500, 128256),
                "f32": rng.random() < 0.3, "cap": 30.0 if rng.random() < 0.3 else 0.0}
    return {"op": "verify", "seqs": _log(rng, 1, 192), "drafts": rng.randint(0, 5), "vocab": _log(rng, 500, 128256),
            "greedy": rng.random() < 0.25}


# ------------------------------------------------------------------- inputs

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt * 7919) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(shape, seed, salt, dtype=torch.float16):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda", dtype=torch.float32).to(dtype)


def _ints(v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


def _pool(layers, pages, kv_heads, page, dim, seed):
    """Planes of keys and values, made a plane at a time (a pool may be large)."""
    t = torch.empty((2 * layers, pages, kv_heads, page, dim), dtype=torch.float16, device="cuda")
    g = _gen(seed, 1)
    for plane in t:
        plane.copy_(torch.randn(plane.shape, generator=g, device="cuda", dtype=torch.float32))
    return t


def _cache(pool, refs, table, lens):
    """The tensors of a paged cache, and the framework's handle on them."""
    s = {"pool": pool, "refs": _ints(refs), "table": _ints(table), "lens": _ints(lens)}
    if own:
        from cima_amd.paged import PagedKV

        s["kv"] = PagedKV(s["pool"], s["refs"], s["table"], s["lens"])
    return s


def _attn_case(c, seed):
    r = np.random.default_rng([seed, 3])
    page, pp = c["page"], c["prefix"] // c["page"]
    S, n = c["seqs"], c["n_new"]
    own_len = r.integers(0, c["own_max"], S)      # a slot's own tokens before the step
    own_len[r.integers(0, S)] = c["own_max"] - 1
    lens = c["prefix"] + own_len
    held = -(-(own_len + n) // page)              # its own pages
    stride = pp + int(held.max()) + 2
    pages = pp + int(held.sum()) + 5
    ids = r.permutation(pages)
    table = np.full((S, stride), -1)
    table[:, :pp] = ids[:pp]
    at = pp
    for s in range(S):
        table[s, pp:pp + held[s]] = ids[at:at + held[s]]
        at += held[s]
    refs = np.zeros(pages)
    np.add.at(refs, table[table >= 0], 1)
    s = _cache(_pool(1, pages, c["kv_heads"], page, c["dim"], seed), refs, table, lens)
    s |= {"case": c, "q": _normal((S * n, c["q_heads"], c["dim"]), seed, 2),
          "prefix_pages": pp, "own_pages": int(held.max()), "scale": 1.0 / math.sqrt(c["dim"]),
          "out": torch.empty((S * n, c["q_heads"], c["dim"]), dtype=torch.float16, device="cuda"),
          "slab": torch.empty(SLAB_BYTES, dtype=torch.uint8, device="cuda")}
    return s


def _append_case(c, seed):
    r = np.random.default_rng([seed, 4])
    page, S, n, D = c["page"], c["seqs"], c["n_new"], c["dim"]
    lens = r.integers(0, c["max_pos"], S)
    stride = -(-(c["max_pos"] + n) // page)
    first, last = lens // page, (lens + n - 1) // page   # the pages that the step writes, the others elsewhere
    pages = S * (1 + (n + page - 2) // page) + 3
    ids = r.permutation(pages)
    table, at = np.full((S, stride), -1), 0
    for s in range(S):
        k = last[s] - first[s] + 1
        table[s, first[s]:last[s] + 1] = ids[at:at + k]
        at += k
    refs = np.zeros(pages)
    refs[ids[:at]] = 1
    s = _cache(_pool(1, pages, c["kv_heads"], page, D, seed), refs, table, lens)
    s |= {"case": c, "qkv": _normal((S * n, (c["q_heads"] + 2 * c["kv_heads"]) * D), seed, 2),
          "q": torch.empty((S * n, c["q_heads"], D), dtype=torch.float16, device="cuda")}
    return s


def _branch_case(c, seed):
    r = np.random.default_rng([seed, 5])
    held = -(-c["length"] // c["page"])
    stride = held + -(-c["room"] // c["page"]) + 2
    ids = r.permutation(c["pages"])
    slots = c["forks"] + 2
    table = np.full((slots, stride), -1)
    table[0, :held] = ids[:held]
    other = min(7, stride)                         # another request, which is left alone
    table[1, :other] = ids[held:held + other]
    refs = np.zeros(c["pages"])
    refs[ids[:held + other]] = 1
    lens = np.full(slots, -1)
    lens[0], lens[1] = c["length"], 5 * c["page"] if other >= 7 else c["page"] // 2
    s = _cache(_pool(c["layers"], c["pages"], c["kv_heads"], c["page"], c["dim"], seed), refs, table, lens)
    s |= {"case": c, "parents": _ints(np.zeros(c["forks"])),
          "children": _ints(2 + r.permutation(c["forks"])), "status": _ints([0])}
    return s


def _compact_case(c, seed):
    r = np.random.default_rng([seed, 6])
    page, S = c["page"], c["seqs"]
    lens = r.integers(1, c["length"] + 1, S)
    held, stride = -(-lens // page), -(-c["length"] // page) + 1
    shared = int(min(held[0], 2))                   # the first slots share a prompt's pages
    ids = r.permutation(c["pages"])
    table, at = np.full((S, stride), -1), shared
    most = c["pages"] * 7 // 10
    for s in range(S):
        k = min(shared, held[s])
        h = int(min(held[s] - k, max(0, most - at)))
        table[s, :k] = ids[:k]
        table[s, k:k + h] = ids[at:at + h]
        lens[s] = min(lens[s], (k + h) * page)
        at += h
    refs = np.zeros(c["pages"])
    np.add.at(refs, table[table >= 0], 1)
    s = _cache(_pool(c["layers"], c["pages"], c["kv_heads"], page, c["dim"], seed), refs, table, lens)
    s |= {"case": c, "refs_out": torch.empty_like(s["refs"]), "table_out": torch.empty_like(s["table"]),
          "live": _ints([0]), "moved": int((refs[int((refs > 0).sum()):] > 0).sum()),
          "slab": torch.empty(SLAB_BYTES, dtype=torch.uint8, device="cuda")}
    return s


def _logits(shape, seed, salt):
    """Logits as a language model's head gives them: a wide body and a few likely tokens."""
    x = torch.randn(shape, generator=_gen(seed, salt), device="cuda")
    return x * 2.0 + 6.0 * (torch.rand(shape, generator=_gen(seed, salt + 1), device="cuda") > 0.9995)


def _softmax_case(c, seed):
    r = np.random.default_rng([seed, 7])
    rows, V = c["reqs"] * c["rows"], c["vocab"]
    x = _logits((rows, V), seed, 10)
    x[:, r.integers(0, V, 1 + V // 1000)] = -math.inf        # tokens that may not be taken
    temp = r.uniform(0.3, 1.5, c["reqs"])
    if c["reqs"] > 2:
        temp[r.integers(0, c["reqs"])] = 0.0                 # a request that takes the likeliest token
    return {"case": c, "x": x.to(torch.float32 if c["f32"] else torch.float16),
            "temp": torch.tensor(temp, dtype=torch.float32, device="cuda"),
            "y": torch.empty((rows, V), dtype=torch.float32, device="cuda"),
            "slab": torch.empty(SLAB_BYTES, dtype=torch.uint8, device="cuda")}


def _verify_case(c, seed):
    S, K, V = c["seqs"], c["drafts"], c["vocab"]
    p = torch.empty((S, K + 1, V), device="cuda")
    q = None if c["greedy"] else torch.empty((S, K, V), device="cuda")
    drafts = torch.zeros((S, K), dtype=torch.int32, device="cuda")
    for j in range(K + 1):                                   # a row at a time: p and q are large
        x = _logits((S, V), seed, 20 + 4 * j)
        p[:, j] = torch.softmax(x, 1)
        if j < K:
            d = torch.softmax(x + 0.7 * torch.randn((S, V), generator=_gen(seed, 22 + 4 * j), device="cuda"), 1)
            if q is not None:
                q[:, j] = d
                cut = torch.rand((S, 1), generator=_gen(seed, 23 + 4 * j), device="cuda")
                drafts[:, j] = (d.double().cumsum(1) <= cut.double()).sum(1).clamp(max=V - 1)
            else:
                drafts[:, j] = d.argmax(1)
    counts = torch.full((S,), K, dtype=torch.int32, device="cuda")
    if K:
        counts[::3] = torch.randint(0, K + 1, counts[::3].shape, generator=_gen(seed, 18), device="cuda").int()
    return {"case": c, "p": p, "q": q, "drafts": drafts, "counts": counts,
            "u": torch.rand((S, K + 1), generator=_gen(seed, 19), device="cuda"),
            "accepted": torch.empty(S, dtype=torch.int32, device="cuda"),
            "tokens": torch.empty((S, K + 1), dtype=torch.int32, device="cuda"),
            "slab": torch.empty(SLAB_BYTES, dtype=torch.uint8, device="cuda")}


def prepare(case, seed):
    return {"attn": _attn_case, "append": _append_case, "branch": _branch_case, "compact": _compact_case,
            "softmax": _softmax_case, "verify": _verify_case}[case["op"]](case, seed)


# -------------------------------------------------------------- plain forms

def _plain_attn(s):
    c = s["case"]
    S, n, H, D, page = c["seqs"], c["n_new"], c["kv_heads"], c["dim"], c["page"]
    g, P, M = c["q_heads"] // H, c["prefix"], s["own_pages"] * page
    q = s["q"].float().view(S, n, H, g, D).permute(2, 0, 1, 3, 4).contiguous()      # [H, S, n, g, D]
    at = s["lens"].view(S, 1) + torch.arange(n, device="cuda")                       # [S, n] positions
    low = (at - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(at)
    # the pages that every slot holds
    ids = s["table"][0, :s["prefix_pages"]].long()
    kp = s["pool"][0][ids].float().permute(1, 0, 2, 3).reshape(H, P, D)
    vp = s["pool"][1][ids].float().permute(1, 0, 2, 3).reshape(H, P, D)
    where = torch.arange(P, device="cuda")
    seen = (where <= at[..., None]) & (where >= low[..., None])                      # [S, n, P]
    sp = torch.matmul(q.view(H, S * n * g, D), kp.transpose(1, 2).contiguous()).mul_(s["scale"]).view(H, S, n, g, P)
    sp.masked_fill_(~seen[None, :, :, None, :], -math.inf)
    # each slot's own
    ids = s["table"][:, s["prefix_pages"]:s["prefix_pages"] + s["own_pages"]].clamp(min=0).long()
    where = P + torch.arange(M, device="cuda")
    live = (where < (s["lens"] + n)[:, None]).view(S, 1, M, 1)
    ko = s["pool"][0][ids].float().permute(0, 2, 1, 3, 4).reshape(S, H, M, D).masked_fill(~live, 0.0)
    vo = s["pool"][1][ids].float().permute(0, 2, 1, 3, 4).reshape(S, H, M, D).masked_fill(~live, 0.0)
    seen = (where <= at[..., None]) & (where >= low[..., None])
    qs = q.permute(1, 0, 2, 3, 4).reshape(S, H, n * g, D)
    so = torch.matmul(qs, ko.transpose(2, 3).contiguous()).mul_(s["scale"]).view(S, H, n, g, M)
    so.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = so.amax(-1, keepdim=True)
    if P:
        m = torch.maximum(m, sp.amax(-1, keepdim=True).transpose(0, 1))
    eo = torch.exp(so - m)
    den = eo.sum(-1, keepdim=True)
    num = torch.matmul(eo.view(S, H, n * g, M), vo).view(S, H, n, g, D)
    if P:
        ep = sp.sub_(m.transpose(0, 1)).exp_()
        den = den + ep.sum(-1, keepdim=True).transpose(0, 1)
        num = num + torch.matmul(ep.view(H, S * n * g, P), vp).view(H, S, n, g, D).transpose(0, 1)
    o = (num / den).permute(0, 2, 1, 3, 4)
    s["out"].copy_(o.reshape(S * n, c["q_heads"], D))
    return s["out"]


def _plain_append(s):
    c = s["case"]
    S, n, H, D, page = c["seqs"], c["n_new"], c["kv_heads"], c["dim"], c["page"]
    at = s["lens"].view(S, 1) + torch.arange(n, device="cuda")
    freq = THETA ** (-2.0 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
    angle = at.reshape(-1, 1, 1).double() * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    x = s["qkv"].view(S * n, -1, D)
    r = x[:, :c["q_heads"] + H].float()
    a, b = r[..., :D // 2], r[..., D // 2:]
    r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1).half()
    s["q"].copy_(r[:, :c["q_heads"]])
    ids = s["table"].gather(1, (at // page).long()).view(-1).long()
    row = (at % page).view(-1).long()
    s["pool"][0][ids, :, row] = r[:, c["q_heads"]:]
    s["pool"][1][ids, :, row] = x[:, c["q_heads"] + H:]
    return {"q": s["q"], "pool": s["pool"]}


def _plain_free(s, slots):
    rows = s["table"][slots]
    s["refs"].index_add_(0, rows.clamp(min=0).view(-1).long(), -(rows >= 0).view(-1).int())
    s["table"][slots] = -1
    s["lens"][slots] = -1


def _lowest_free(refs, k):
    """The k lowest pages that nobody holds."""
    rank = (refs == 0).cumsum(0)
    return torch.searchsorted(rank, torch.arange(1, k + 1, device="cuda", dtype=rank.dtype))


def _plain_branch(s):
    c = s["case"]
    page, n, stride = c["page"], c["forks"], s["table"].shape[1]
    parents, children = s["parents"].long(), s["children"].long()
    _plain_free(s, children)
    # fork: whole pages are shared, what follows them is copied
    length = s["lens"][parents]
    full, rest = length // page, length % page
    col = torch.arange(stride, device="cuda")
    rows = s["table"][parents]
    shared = col < full[:, None]
    s["refs"].index_add_(0, rows.clamp(min=0).view(-1).long(), shared.view(-1).int())
    got = _lowest_free(s["refs"], n)
    part = rest > 0
    rank = part.cumsum(0) - 1
    new = torch.where(part, got[rank.clamp(min=0)], -1)
    s["table"][children] = torch.where(shared, rows, torch.where((col == full[:, None]) & part[:, None],
                                                                  new[:, None].int(), -1)).int()
    s["lens"][children] = length
    s["refs"].index_add_(0, new.clamp(min=0), part.int())
    src = rows.gather(1, full.long().clamp(max=stride - 1)[:, None])[:, 0].clamp(min=0).long()
    dst = new.clamp(min=0)
    keep = ((torch.arange(page, device="cuda") < rest[:, None]) & part[:, None]).view(1, n, 1, page, 1)
    s["pool"][:, dst] = torch.where(keep, s["pool"][:, src], s["pool"][:, dst])
    # room for the step's tokens, the slots in order
    end = torch.where(s["lens"] >= 0, (s["lens"] + c["room"] + page - 1) // page, 0)
    want = (s["table"] < 0) & (col < end[:, None]) & (col >= (s["lens"] // page)[:, None])
    rank = want.view(-1).cumsum(0).view_as(want)
    free = (s["refs"] == 0).cumsum(0)
    enough = rank[-1, -1] <= free[-1]
    want &= enough
    new = torch.searchsorted(free, rank.to(free.dtype).clamp(min=1)).clamp(max=c["pages"] - 1)
    s["table"].copy_(torch.where(want, new.int(), s["table"]))
    s["refs"].index_add_(0, new.view(-1), want.view(-1).int())
    s["status"].copy_(torch.where(enough, 0, rank[-1, -1] - free[-1]))
    return {k: s[k] for k in ("table", "refs", "lens", "status", "pool")}


def _plain_compact(s):
    live = s["refs"] > 0
    n_live = live.sum()
    ids = torch.arange(live.numel(), device="cuda")
    # the k-th live page behind the first n_live takes the k-th hole in them
    src, hole = live & (ids >= n_live), ~live & (ids < n_live)
    n = s["moved"]
    k = torch.arange(1, n + 1, device="cuda")
    a = torch.searchsorted(src.cumsum(0), k)
    b = torch.searchsorted(hole.cumsum(0), k)
    remap = ids.clone()
    remap[a] = b
    s["refs_out"].copy_(torch.where(ids < n_live, s["refs"], 0))
    s["refs_out"][b] = s["refs"][a]
    t = s["table"]
    s["table_out"].copy_(torch.where(t >= 0, remap[t.clamp(min=0).long()], -1))
    s["live"].copy_(n_live)
    s["pool"][:, b] = s["pool"][:, a]
    return {k: s[k] for k in ("table_out", "refs_out", "live", "pool")}


def _plain_softmax(s):
    c = s["case"]
    x = s["x"].float()
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    t = s["temp"].repeat_interleave(c["rows"])[:, None]
    m = x.amax(1, keepdim=True)
    e = torch.exp((x - m) / torch.where(t > 0, t, 1.0))
    e = e / e.sum(1, keepdim=True)
    top = torch.arange(c["vocab"], device="cuda") == x.argmax(1, keepdim=True)
    s["y"].copy_(torch.where(t > 0, e, top.float()))
    return s["y"]


def _plain_verify(s):
    c = s["case"]
    S, K, V = c["seqs"], c["drafts"], c["vocab"]
    p, q, u = s["p"], s["q"], s["u"].double()
    d = s["drafts"].long()[..., None]
    pd = p[:, :K].gather(2, d)[..., 0].double()
    qd = q.gather(2, d)[..., 0].double() if q is not None else torch.ones_like(pd)
    ok = (u[:, :K] * qd < pd) & (torch.arange(K, device="cuda") < s["counts"][:, None])
    a = ok.int().cumprod(1).sum(1)
    row = torch.arange(S, device="cuda")
    last = p[row, a]
    refused = (a < s["counts"])[:, None]
    if K:
        k = a.clamp(max=K - 1)
        other = q[row, k] if q is not None else (torch.arange(V, device="cuda") == d[row, k]).float()
        r = torch.where(refused, (last - other).clamp(min=0), last)
        if q is None:
            r = torch.where(refused & (other > 0), 0.0, last)
    else:
        r = last
    r = torch.where((r.sum(1, keepdim=True) > 0), r, last)
    cs = r.double().cumsum(1)
    t = (cs <= (u[:, K] * cs[:, -1])[:, None]).sum(1).clamp(max=V - 1)
    col = torch.arange(K + 1, device="cuda")
    drafted = torch.cat([s["drafts"], s["drafts"].new_zeros((S, 1))], 1)
    s["tokens"].copy_(torch.where(col < a[:, None], drafted, torch.where(col == a[:, None], t[:, None].int(), -1)))
    s["accepted"].copy_(a)
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


# -------------------------------------------------------------------- a pass

def _own_run(s):
    h, c = _hip(), s["case"]
    op = c["op"]
    if op == "attn":
        h.attn_paged(s["kv"], 0, s["q"], s["out"], c["seqs"], c["n_new"], c["q_heads"], s["scale"], s["slab"],
                     prefix_pages=s["prefix_pages"], prefix_slot=0, window=c["window"])
        return s["out"]
    if op == "append":
        h.rope_append_paged(s["kv"], 0, s["qkv"], s["q"], c["seqs"], c["n_new"], c["q_heads"], THETA)
        return {"q": s["q"], "pool": s["pool"]}
    if op == "branch":
        h.kv_pages_free(s["kv"], s["children"], c["forks"])
        h.kv_pages_fork(s["kv"], s["parents"], s["children"], c["forks"], s["status"])
        h.kv_pages_reserve(s["kv"], c["forks"] + 2, c["room"], s["status"])
        return {k: s[k] for k in ("table", "refs", "lens", "status", "pool")}
    if op == "compact":
        h.kv_pages_compact(s["kv"], s["refs_out"], s["table_out"], s["live"], s["slab"])
        return {k: s[k] for k in ("table_out", "refs_out", "live", "pool")}
    if op == "softmax":
        h.softmax_rows(s["x"], s["y"], c["reqs"] * c["rows"], c["vocab"], s["temp"], c["rows"], c["cap"], s["slab"])
        return s["y"]
    h.verify_drafts(s["p"], s["q"], s["drafts"], s["counts"], s["u"], s["accepted"], s["tokens"], None, c["seqs"],
                    c["drafts"], c["vocab"], s["slab"])
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


def run(state):
    if own:
        return _own_run(state)
    return {"attn": _plain_attn, "append": _plain_append, "branch": _plain_branch, "compact": _plain_compact,
            "softmax": _plain_softmax, "verify": _plain_verify}[state["case"]["op"]](state)


# ---------------------------------------------------------------------- work

def work(case):
    """What a pass cannot do without.  Lengths that depend on the seed count with their mean."""
    c, op = case, case["op"]
    if op == "attn":
        rows = c["seqs"] * c["n_new"]
        mean = c["own_max"] / 2 + c["n_new"] / 2
        seen = c["prefix"] + mean
        pre, mine = c["prefix"], mean
        if c["window"]:
            seen = min(seen, c["window"])
            pre = max(0.0, min(c["prefix"], c["window"] + c["n_new"]))
            mine = min(mean, c["window"] + c["n_new"])
        token = c["kv_heads"] * c["dim"] * 4
        return {"bytes": (pre + c["seqs"] * mine) * token + 4 * rows * c["q_heads"] * c["dim"],
                "flops": 4.0 * rows * c["q_heads"] * c["dim"] * seen}
    if op == "append":
        rows, heads = c["seqs"] * c["n_new"], c["q_heads"] + 2 * c["kv_heads"]
        return {"bytes": 4.0 * rows * heads * c["dim"], "flops": 3.0 * rows * (c["q_heads"] + c["kv_heads"]) * c["dim"]}
    if op == "branch":
        token = c["layers"] * c["kv_heads"] * c["dim"] * 4
        held = -(-c["length"] // c["page"])
        # the copied rows read once for all children and written for each; rows of the table; the counts
        rest = c["length"] % c["page"]
        return {"bytes": rest * token * (1 + c["forks"]) + 8.0 * c["forks"] * held + 8.0 * c["pages"], "flops": 0}
    if op == "compact":
        page = 2 * c["layers"] * c["kv_heads"] * c["page"] * c["dim"] * 2
        held = min(c["pages"] * 7 // 10, c["seqs"] * (c["length"] / 2 / c["page"] + 0.5))
        moved = held * (1 - held / c["pages"])
        return {"bytes": 2.0 * moved * page + 8.0 * c["pages"], "flops": 0}
    if op == "softmax":
        n = c["reqs"] * c["rows"] * c["vocab"]
        return {"bytes": n * (4.0 + (4 if c["f32"] else 2)), "flops": 4.0 * n}
    rows = 1 if c["greedy"] or not c["drafts"] else 2
    return {"bytes": 4.0 * c["seqs"] * (rows * c["vocab"] + 5 * c["drafts"] + 3), "flops": 2.0 * c["seqs"] * c["vocab"]}


# ---------------------------------------------------------------- in 64 bits

def _exact_attn(c, seed):
    s = _attn_case(c, seed)
    S, n, H, D, page = c["seqs"], c["n_new"], c["kv_heads"], c["dim"], c["page"]
    g = c["q_heads"] // H
    out = torch.zeros((S, n, c["q_heads"], D), dtype=torch.float64, device="cuda")
    q = s["q"].double().view(S, n, H, g, D)
    lens, table = s["lens"].tolist(), s["table"].long()
    for b in range(S):
        total = lens[b] + n
        ids = table[b, :-(-total // page)]
        for h in range(H):
            k = s["pool"][0, ids, h].reshape(-1, D)[:total].double()
            v = s["pool"][1, ids, h].reshape(-1, D)[:total].double()
            for j in range(n):
                lo = max(0, lens[b] + j + 1 - c["window"]) if c["window"] else 0
                hi = lens[b] + j + 1
                w = torch.softmax((q[b, j, h] @ k[lo:hi].t().contiguous()) * s["scale"], -1)
                out[b, j, h * g:(h + 1) * g] = w @ v[lo:hi]
    return out.view(S * n, c["q_heads"], D)


def _exact_append(c, seed):
    s = _append_case(c, seed)
    n, H, Q, D, page = c["n_new"], c["kv_heads"], c["q_heads"], c["dim"], c["page"]
    x = s["qkv"].double().view(c["seqs"], n, -1, D).cpu().numpy()
    lens, table = s["lens"].tolist(), s["table"].cpu().numpy()
    pool = s["pool"].double()
    q = np.empty((c["seqs"], n, Q, D))
    freq = np.power(THETA, -np.arange(0, D, 2) / D)
    for b, length in enumerate(lens):
        for j in range(n):
            pos = length + j
            z = (x[b, j, :Q + H, :D // 2] + 1j * x[b, j, :Q + H, D // 2:]) * np.exp(1j * pos * freq)
            r = np.concatenate([z.real, z.imag], -1)
            q[b, j] = r[:Q]
            where = table[b, pos // page]
            pool[0, where, :, pos % page] = torch.from_numpy(r[Q:]).cuda()
            pool[1, where, :, pos % page] = torch.from_numpy(x[b, j, Q + H:]).cuda()
    return {"q": q.reshape(-1, Q, D), "pool": pool}


def _exact_softmax(c, seed):
    s = _softmax_case(c, seed)
    y = torch.empty((c["reqs"] * c["rows"], c["vocab"]), dtype=torch.float64, device="cuda")
    temp = s["temp"].double().tolist()
    for i in range(y.shape[0]):
        x, t = s["x"][i].double(), temp[i // c["rows"]]
        if c["cap"]:
            x = c["cap"] * torch.tanh(x / c["cap"])
        if t > 0:
            y[i] = torch.softmax(x / t, 0)
        else:
            y[i] = 0.0
            y[i, int((x == x.max()).nonzero()[0, 0])] = 1.0
    return y


def _exact_verify(c, seed):
    s = _verify_case(c, seed)
    S, K = c["seqs"], c["drafts"]
    u, counts, drafts = s["u"].cpu().double().numpy(), s["counts"].tolist(), s["drafts"].tolist()
    tokens, accepted = np.full((S, K + 1), -1, np.int32), np.zeros(S, np.int32)
    for b in range(S):
        a = 0
        while a < counts[b]:
            d = drafts[b][a]
            if not u[b, a] * (1.0 if s["q"] is None else float(s["q"][b, a, d])) < float(s["p"][b, a, d]):
                break
            tokens[b, a] = d
            a += 1
        r = s["p"][b, a].cpu().numpy()
        if a < counts[b]:
            other = np.zeros_like(r)
            if s["q"] is not None:
                other = s["q"][b, a].cpu().numpy()
            left = np.maximum(r - other, np.float32(0))
            if s["q"] is None:
                left[drafts[b][a]] = 0
            r = left if left.any() else r
        total = np.cumsum(r.astype(np.float64))
        tokens[b, a] = int(np.searchsorted(total, u[b, K] * total[-1], side="right"))
        accepted[b] = a
    return {"tokens": torch.from_numpy(tokens), "accepted": torch.from_numpy(accepted)}


def exact(case, seed):
    """None for the pages' operators: they move values and compute none."""
    f = {"attn": _exact_attn, "append": _exact_append, "softmax": _exact_softmax, "verify": _exact_verify}
    return f[case["op"]](case, seed) if case["op"] in f else None
