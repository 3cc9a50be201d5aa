"""The operators that serve a batch from a paged cache of 4- and 8-bit elements, and
report the tokens' log probabilities, as they are timed: their inputs, a plain form of
each, and the same in 64 bits.

The cache's pages hold groups of 32 elements of a head's row in GGUF's formats Q4_1
(codes 0 to 15, f16 scale and minimum: c * d + m) and Q8_0 (codes -127 to 127, f16
scale: c * d); the value of an element is that number rounded to f16.  A page of a head
is its rows' codes, then its rows' scales.  A step of the batch is

* ``append``: rotary embedding of the step's queries and keys, the new keys and values
  quantised as they are written to their pages, and the rows read back;
* ``attn``: attention of the step's queries over the pages, those that all slots share
  read once for all;
* ``read``: positions of some slots taken out of the pages as f16 caches;
* ``logprobs``: of the tokens taken, with the rows' entropies and likeliest alternatives.

Shapes are those of the repository's decoder configurations (Qwen2.5-0.5B heads
14 / 2 of 64, vocabulary 151936; Llama-3-8B heads 32 / 8 of 128, vocabulary 128256) and
generic ones between them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

SLAB_BYTES = 64 << 20   # scratch that a serving program keeps for its calls
THETA = 1e6
FORMATS = {4: 3, 8: 8}  # bits -> ggml type: Q4_1, Q8_0
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

def _attn(name, bits, seqs, n_new, q_heads, kv_heads, dim, page, prefix, own_max, window=0):
    c = {"op": "attn", "bits": bits, "seqs": seqs, "n_new": n_new, "q_heads": q_heads, "kv_heads": kv_heads,
         "dim": dim, "page": page, "prefix": prefix, "own_max": own_max, "window": window}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few answers by the small model: what a step costs in latency
        _attn("attn few", 4, 4, 1, 14, 2, 64, 16, 512, 61),
        # a batch of requests of their own, as long as memory lets them be
        _attn("attn batch", 4, 64, 1, 32, 8, 128, 64, 0, 12000),
        # a full batch over a very long document
        _attn("attn long", 4, 128, 1, 32, 8, 128, 128, 65536, 500),
        # drafted tokens checked in one step, with a sliding window that ends inside the prefix, 8-bit elements
        _attn("attn drafts", 8, 24, 5, 14, 2, 64, 32, 4096, 700, 4000),
        # requests of middling length with 8-bit elements
        _attn("attn fine", 8, 40, 1, 28, 4, 128, 64, 0, 6001),
        # rotary embedding and cache write of one token of a few slots, and of drafts of a large batch
        {"name": "append few", "op": "append", "bits": 4, "seqs": 4, "n_new": 1, "q_heads": 14, "kv_heads": 2,
         "dim": 64, "page": 16, "max_pos": 4000},
        {"name": "append drafts", "op": "append", "bits": 4, "seqs": 256, "n_new": 8, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "max_pos": 120000},
        # one request handed to the single-sequence decoder, and a batch taken out of the pages
        {"name": "read one", "op": "read", "bits": 8, "slots": 1, "kv_heads": 2, "dim": 64, "page": 16,
         "length": 4003, "room": 4096},
        {"name": "read batch", "op": "read", "bits": 4, "slots": 24, "kv_heads": 8, "dim": 128, "page": 64,
         "length": 5000, "room": 5000},
        # one token reported, every row of a batch with its alternatives, and a long prompt scored
        {"name": "logprobs one", "op": "logprobs", "reqs": 1, "rows": 1, "vocab": 151936, "f32": False, "cap": 0.0,
         "top": 5},
        {"name": "logprobs batch", "op": "logprobs", "reqs": 64, "rows": 6, "vocab": 128256, "f32": False, "cap": 0.0,
         "top": 20},
        {"name": "logprobs prompt", "op": "logprobs", "reqs": 1, "rows": 777, "vocab": 151936, "f32": False,
         "cap": 0.0, "top": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "read", "logprobs", "logprobs"])
    heads = rng.choice([(14, 2, 64), (32, 8, 128), (28, 4, 128), (12, 12, 64), (16, 1, 128), (24, 8, 64)])
    page = rng.choice([16, 32, 64, 128, 256])
    bits = rng.choice([4, 4, 8])
    if op == "attn":
        seqs, n_new = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 3, 5, 8])
        prefix = _log(rng, 16, 65536) if rng.random() < 0.5 else 0
        while seqs * n_new * heads[0] * heads[2] * prefix > 128 * 32 * 128 * 65536:  # no dearer than the largest
            prefix = prefix * 3 // 4
        own_max = _log(rng, 2, 12000)
        while seqs * own_max * heads[1] * heads[2] * bits > 64 * 12000 * 8 * 128 * 4:
            own_max = own_max * 3 // 4
        window = _log(rng, 30, 2 * (prefix + 500)) if rng.random() < 0.25 else 0
        return _attn(None, bits, seqs, n_new, *heads, page, prefix // page * page, max(own_max, 2), window)
    if op == "append":
        return {"op": "append", "bits": bits, "seqs": _log(rng, 1, 256), "n_new": rng.randint(1, 8),
                "q_heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "page": page,
                "max_pos": _log(rng, 1000, 120000)}
    if op == "read":
        slots = _log(rng, 1, 24)
        length = _log(rng, 1, 5000)
        return {"op": "read", "bits": bits, "slots": slots, "kv_heads": min(heads[1], 8), "dim": heads[2],
                "page": page, "length": length, "room": length + rng.choice([0, 0, 1, 100])}
    rows = rng.randint(1, 6)
    return {"op": "logprobs", "reqs": _log(rng, 1, 64), "rows": rows, "vocab": _log(rng, 500, 128256),
            "f32": rng.random() < 0.3, "cap": 30.0 if rng.random() < 0.3 else 0.0,
            "top": rng.choice([0, 1, 5, 8, 20, 32])}


# ------------------------------------------------------------------- inputs

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt * 7919) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(shape, seed, salt, dtype=torch.float16):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda", dtype=torch.float32).to(dtype)


def _ints(v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


def _head_bytes(c):
    """Bytes of a page of one head: codes, then scales."""
    return c["page"] * c["dim"] * (20 if c["bits"] == 4 else 34) // 32


def _pack(codes, scales, bits):
    """Codes uint8 [.., page, D] and scales f16 [.., page, D / 32, 2 or 1] as a head's page."""
    if bits == 4:
        e = codes.unflatten(-1, (-1, 8))           # the eight elements of a 32-bit word, even ones in its low half
        codes = torch.stack([e[..., 0] | e[..., 2] << 4, e[..., 4] | e[..., 6] << 4, e[..., 1] | e[..., 3] << 4,
                             e[..., 5] | e[..., 7] << 4], -1).flatten(-2)
    return torch.cat([codes.flatten(-2), scales.contiguous().view(torch.uint8).flatten(-3)], -1)


def _pool(c, planes, pages, seed):
    """Planes of keys and values, as a running cache holds them, made some pages at a time."""
    t = torch.empty((planes, pages, c["kv_heads"], _head_bytes(c)), dtype=torch.uint8, device="cuda")
    g = _gen(seed, 1)
    step = max(1, (64 << 20) // (c["kv_heads"] * c["page"] * c["dim"]))
    for plane in t:
        for a in range(0, pages, step):
            n = min(step, pages - a)
            x = torch.randn((n, c["kv_heads"], c["page"], c["dim"] // 32, 32), generator=g, device="cuda")
            if c["bits"] == 4:
                m = x.amin(-1, keepdim=True).half()
                d = ((x.amax(-1, keepdim=True) - m) / 15).half()
                codes = ((x - m) / d).round_().clamp_(0, 15)
                scales = torch.cat([d, m], -1)
            else:
                scales = (x.abs().amax(-1, keepdim=True) / 127).half()
                codes = (x / scales).round_().clamp_(-127, 127) + 128
            plane[a:a + n] = _pack(codes.to(torch.uint8).flatten(-2), scales, c["bits"])
    return t


def _cache(c, pool, refs, table, lens):
    """The tensors of a paged cache, and the framework's handle on them."""
    s = {"pool": pool, "refs": _ints(refs), "table": _ints(table), "lens": _ints(lens)}
    if own:
        from cima_amd.paged import PagedKV

        s["kv"] = PagedKV(s["pool"], s["refs"], s["table"], s["lens"], ggml_type=FORMATS[c["bits"]], page=c["page"],
                          head_dim=c["dim"])
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
    s = _cache(c, _pool(c, 2, pages, seed), refs, table, lens)
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
    s = _cache(c, _pool(c, 2, pages, seed), refs, table, lens)
    s |= {"case": c, "qkv": _normal((S * n, (c["q_heads"] + 2 * c["kv_heads"]) * D), seed, 2),
          "q": torch.empty((S * n, c["q_heads"], D), dtype=torch.float16, device="cuda"),
          "k": torch.empty((S, c["kv_heads"], n, D), dtype=torch.float16, device="cuda"),
          "v": torch.empty((S, c["kv_heads"], n, D), dtype=torch.float16, device="cuda")}
    return s


def _read_case(c, seed):
    r = np.random.default_rng([seed, 5])
    page, S, n = c["page"], c["slots"], c["length"]
    held = -(-n // page)
    pages = S * held + 4
    slots = S + 2                                 # others are left in the batch
    order = r.permutation(slots)[:S]
    table = np.full((slots, held + 1), -1)
    table[order, :held] = r.permutation(pages)[:S * held].reshape(S, held)
    refs = np.zeros(pages)
    refs[table[table >= 0]] = 1
    lens = np.full(slots, -1)
    lens[order] = n
    s = _cache(c, _pool(c, 2, pages, seed), refs, table, lens)
    out = dict(dtype=torch.float16, device="cuda")
    s |= {"case": c, "slots": _ints(order), "k": torch.zeros((S, c["kv_heads"], c["room"], c["dim"]), **out),
          "v": torch.zeros((S, c["kv_heads"], c["room"], c["dim"]), **out)}
    return s


def _logprobs_case(c, seed):
    r = np.random.default_rng([seed, 7])
    rows, V = c["reqs"] * c["rows"], c["vocab"]
    # logits as a language model's head gives them: a wide body and a few likely tokens
    x = torch.randn((rows, V), generator=_gen(seed, 10), device="cuda") * 2.0
    x += 6.0 * (torch.rand((rows, V), generator=_gen(seed, 11), device="cuda") > 0.9995)
    x[:, r.integers(0, V, 1 + V // 1000)] = -math.inf        # tokens that may not be taken
    tokens = x.argmax(1)
    some = torch.rand(rows, generator=_gen(seed, 12), device="cuda") < 0.5
    other = torch.randint(0, V, (rows,), generator=_gen(seed, 13), device="cuda")
    tokens = torch.where(some & (x.gather(1, other[:, None])[:, 0] > -math.inf), other, tokens)
    temp = r.uniform(0.3, 1.5, c["reqs"])
    f32 = dict(dtype=torch.float32, device="cuda")
    return {"case": c, "x": x.to(torch.float32 if c["f32"] else torch.float16), "tokens": tokens.int(),
            "temp": torch.tensor(temp, **f32), "logprob": torch.empty(rows, **f32), "entropy": torch.empty(rows, **f32),
            "top_ids": torch.empty((rows, c["top"]), dtype=torch.int32, device="cuda") if c["top"] else None,
            "top_logprobs": torch.empty((rows, c["top"]), **f32) if c["top"] else None,
            "slab": torch.empty(SLAB_BYTES, dtype=torch.uint8, device="cuda")}


def prepare(case, seed):
    return {"attn": _attn_case, "append": _append_case, "read": _read_case,
            "logprobs": _logprobs_case}[case["op"]](case, seed)


# -------------------------------------------------------------- plain forms

def _values(pages, c):
    """The f16 values of heads' pages, uint8 [.., head bytes], as float [.., page, D]."""
    page, D = c["page"], c["dim"]
    if c["bits"] == 4:
        w = pages[..., :page * D // 2].unflatten(-1, (page, D // 8, 4))
        low, high = w & 15, w >> 4
        codes = torch.stack([low[..., 0], low[..., 2], high[..., 0], high[..., 2], low[..., 1], low[..., 3],
                             high[..., 1], high[..., 3]], -1).flatten(-2)
        s = pages[..., page * D // 2:].contiguous().view(torch.float16).unflatten(-1, (page, D // 32, 2))
        x = codes.unflatten(-1, (D // 32, 32)) * s[..., :1].float() + s[..., 1:].float()
    else:
        codes = pages[..., :page * D].unflatten(-1, (page, D // 32, 32)).float() - 128
        s = pages[..., page * D:].contiguous().view(torch.float16).unflatten(-1, (page, D // 32, 1))
        x = codes * s.float()
    return x.half().float().flatten(-2)


def _plain_attn(s):
    c = s["case"]
    S, n, H, D, page = c["seqs"], c["n_new"], c["kv_heads"], c["dim"], c["page"]
    g, P, M = c["q_heads"] // H, c["prefix"], s["own_pages"] * page
    q = s["q"].float().view(S, n, H, g, D).permute(2, 0, 1, 3, 4).contiguous()      # [H, S, n, g, D]
    at = s["lens"].view(S, 1) + torch.arange(n, device="cuda")                       # [S, n] positions
    low = (at - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(at)
    # the pages that every slot holds
    ids = s["table"][0, :s["prefix_pages"]].long()
    kp = _values(s["pool"][0][ids], c).permute(1, 0, 2, 3).reshape(H, P, D)
    vp = _values(s["pool"][1][ids], c).permute(1, 0, 2, 3).reshape(H, P, D)
    where = torch.arange(P, device="cuda")
    seen = (where <= at[..., None]) & (where >= low[..., None])                      # [S, n, P]
    sp = torch.matmul(q.view(H, S * n * g, D), kp.transpose(1, 2).contiguous()).mul_(s["scale"]).view(H, S, n, g, P)
    sp.masked_fill_(~seen[None, :, :, None, :], -math.inf)
    # each slot's own
    ids = s["table"][:, s["prefix_pages"]:s["prefix_pages"] + s["own_pages"]].clamp(min=0).long()
    where = P + torch.arange(M, device="cuda")
    live = (where < (s["lens"] + n)[:, None]).view(S, 1, M, 1)
    ko = _values(s["pool"][0][ids], c).permute(0, 2, 1, 3, 4).reshape(S, H, M, D).masked_fill_(~live, 0.0)
    vo = _values(s["pool"][1][ids], c).permute(0, 2, 1, 3, 4).reshape(S, H, M, D).masked_fill_(~live, 0.0)
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


def _up(q):
    """The least f16 that is not below q >= 0 (float64)."""
    t = q.half()
    return torch.where(t.double() < q, (t.view(torch.int16) + 1).view(torch.float16), t)


def _half(x):
    """float64 to float16, rounded once: an inexact float32 on the way is made odd, which no tie is."""
    f = x.float()
    b = f.view(torch.int32) - (f.double().abs() > x.abs()).int()
    return (b | (f.double() != x).int()).view(torch.float32).half()


def _quantised(x, bits):
    """Rows of f16 values [.., D] as a head's page keeps them: codes and scales.  In 64 bits:
    a quotient next to a border of two codes has to fall on the right side."""
    x = x.double().unflatten(-1, (-1, 32))
    if bits == 4:
        m = x.amin(-1, keepdim=True)
        d = _up((x.amax(-1, keepdim=True) - m) / 15)
        codes, scales = x - m, torch.cat([d, m.half()], -1)
    else:
        d = _up(x.abs().amax(-1, keepdim=True) / 127)
        codes, scales = x, d
    codes = torch.where(d > 0, codes / d.double(), 0.0).round() + (0 if bits == 4 else 128)
    return codes.to(torch.uint8).flatten(-2), scales


def _plain_append(s):
    c = s["case"]
    S, n, H, D, page, bits = c["seqs"], c["n_new"], c["kv_heads"], c["dim"], c["page"], c["bits"]
    at = s["lens"].view(S, 1) + torch.arange(n, device="cuda")
    freq = THETA ** (-2.0 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
    angle = at.reshape(-1, 1, 1).double() * freq
    cos, sin = angle.cos(), angle.sin()
    x = s["qkv"].view(S * n, -1, D)
    r = x[:, :c["q_heads"] + H].double()
    a, b = r[..., :D // 2], r[..., D // 2:]
    r = _half(torch.cat([a * cos - b * sin, a * sin + b * cos], -1))
    s["q"].copy_(r[:, :c["q_heads"]])
    ids = s["table"].gather(1, (at // page).long()).view(-1).long()
    row = (at % page).view(-1).long()
    one = dict(c, page=1)                                                            # a row as a page of its own
    for plane, y, out in ((0, r[:, c["q_heads"]:], s["k"]), (1, x[:, c["q_heads"] + H:], s["v"])):
        codes, scales = _quantised(y, bits)
        packed = _pack(codes.unsqueeze(-2), scales.unsqueeze(-3), bits)              # [S n, H, bytes]
        w = D * bits // 8
        pool = s["pool"][plane]
        pool[..., :page * w].unflatten(-1, (page, w))[ids, :, row] = packed[..., :w]
        pool[..., page * w:].unflatten(-1, (page, -1))[ids, :, row] = packed[..., w:]
        out.copy_(_values(packed, one).view(S, n, H, D).transpose(1, 2))
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _plain_read(s):
    c = s["case"]
    n, H, D, page = c["length"], c["kv_heads"], c["dim"], c["page"]
    ids = s["table"][s["slots"].long(), :-(-n // page)].long()
    for plane, out in ((0, s["k"]), (1, s["v"])):
        x = _values(s["pool"][plane][ids], c).transpose(1, 2).reshape(c["slots"], H, -1, D)
        out[:, :, :n] = x[:, :, :n].half()
    return {"k": s["k"], "v": s["v"]}


def _plain_logprobs(s):
    c = s["case"]
    x = s["x"].float()
    if c["cap"]:
        x = torch.where(x.isinf(), x, c["cap"] * torch.tanh(x / c["cap"]))
    z = x / s["temp"].repeat_interleave(c["rows"])[:, None]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    z = z - torch.log(total)
    s["logprob"].copy_(z.gather(1, s["tokens"].long()[:, None])[:, 0])
    s["entropy"].copy_(-(e / total * torch.where(e > 0, z, 0.0)).sum(1))
    out = {"logprob": s["logprob"], "entropy": s["entropy"]}
    if c["top"]:
        # equal logits in the order of their ids: as whole numbers, the lower id the larger
        k = (s["x"].float() + 0.0).view(torch.int32).long()
        k = (torch.where(k < 0, ~k | -0x80000000, k) << 32) - torch.arange(c["vocab"], device="cuda")
        ids = k.topk(c["top"], 1).indices
        s["top_ids"].copy_(ids)
        s["top_logprobs"].copy_(z.gather(1, ids))
        out |= {"top_ids": s["top_ids"], "top_logprobs": s["top_logprobs"]}
    return out


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
        h.kv_pages_read(s["kv"], 0, s["k"], s["v"], c["seqs"], c["n_new"], first=s["lens"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if op == "read":
        h.kv_pages_read(s["kv"], 0, s["k"], s["v"], c["slots"], c["length"], slots=s["slots"], max_seq=c["room"])
        return {"k": s["k"], "v": s["v"]}
    h.logprobs_rows(s["x"], c["reqs"] * c["rows"], c["vocab"], s["tokens"], s["logprob"], s["entropy"], c["top"],
                    s["top_ids"], s["top_logprobs"], s["temp"], c["rows"], c["cap"], s["slab"])
    out = {"logprob": s["logprob"], "entropy": s["entropy"]}
    return out | ({"top_ids": s["top_ids"], "top_logprobs": s["top_logprobs"]} if c["top"] else {})


def run(state):
    if own:
        return _own_run(state)
    return {"attn": _plain_attn, "append": _plain_append, "read": _plain_read,
            "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# ---------------------------------------------------------------------- work

def work(case):
    """What a pass cannot do without.  Lengths that depend on the seed count with their mean."""
    c, op = case, case["op"]
    if op == "logprobs":
        rows = c["reqs"] * c["rows"]
        return {"bytes": rows * (c["vocab"] * (4.0 if c["f32"] else 2.0) + 12 + 8 * c["top"]),
                "flops": 6.0 * rows * c["vocab"]}
    token = 2 * c["kv_heads"] * c["dim"] * (20 if c["bits"] == 4 else 34) / 32     # of keys and values
    if op == "attn":
        rows = c["seqs"] * c["n_new"]
        mean = c["own_max"] / 2 + c["n_new"] / 2
        seen = c["prefix"] + mean
        pre, mine = c["prefix"], mean
        if c["window"]:
            seen = min(seen, c["window"])
            pre = max(0.0, min(c["prefix"], c["window"] + c["n_new"]))
            mine = min(mean, c["window"] + c["n_new"])
        return {"bytes": (pre + c["seqs"] * mine) * token + 4 * rows * c["q_heads"] * c["dim"],
                "flops": 4.0 * rows * c["q_heads"] * c["dim"] * seen}
    if op == "append":
        rows = c["seqs"] * c["n_new"]
        # the step's rows read, the queries written, keys and values written to the pages and, read back, as f16
        return {"bytes": rows * (2.0 * (c["q_heads"] + 2 * c["kv_heads"]) * c["dim"] + 2 * c["q_heads"] * c["dim"]
                                 + token + 4 * c["kv_heads"] * c["dim"]),
                "flops": 3.0 * rows * (c["q_heads"] + c["kv_heads"]) * c["dim"]}
    return {"bytes": c["slots"] * c["length"] * (token + 4.0 * c["kv_heads"] * c["dim"]),
            "flops": 4.0 * c["slots"] * c["length"] * c["kv_heads"] * c["dim"]}


# ---------------------------------------------------------------- in 64 bits

def _exact_values(pool, c):
    """A plane's values by its definition: bytes [pages, heads, bytes] -> [pages, heads, page, D] float16."""
    page, D = c["page"], c["dim"]
    e = torch.arange(D, device="cuda")
    out = torch.empty((*pool.shape[:2], page, D), dtype=torch.float16, device="cuda")
    for h in range(pool.shape[1]):
        b = pool[:, h]
        if c["bits"] == 4:
            j = e % 8
            nibble = j // 2 + 4 * (j % 2)
            byte = torch.arange(page, device="cuda")[:, None] * (D // 2) + e // 8 * 4 + nibble // 2
            codes = (b[:, byte].int() >> (4 * (nibble % 2))) & 15
            s = b[:, page * D // 2:].contiguous().view(torch.float16).view(-1, page, D // 32, 2)[:, :, e // 32].double()
            out[:, h] = (codes.double() * s[..., 0] + s[..., 1]).half()
        else:
            s = b[:, page * D:].contiguous().view(torch.float16).view(-1, page, D // 32)[:, :, e // 32].double()
            out[:, h] = ((b[:, :page * D].view(-1, page, D).double() - 128) * s).half()
    return out


def _exact_attn(c, seed):
    s = _attn_case(c, seed)
    S, n, H, D, page = c["seqs"], c["n_new"], c["kv_heads"], c["dim"], c["page"]
    g = c["q_heads"] // H
    keys, values = _exact_values(s["pool"][0], c), _exact_values(s["pool"][1], c)
    out = torch.zeros((S, n, c["q_heads"], D), dtype=torch.float64, device="cuda")
    q = s["q"].double().view(S, n, H, g, D)
    lens, table = s["lens"].tolist(), s["table"].long()
    for b in range(S):
        total = lens[b] + n
        ids = table[b, :-(-total // page)]
        for h in range(H):
            k = keys[ids, h].reshape(-1, D)[:total].double()
            v = values[ids, h].reshape(-1, D)[:total].double()
            for j in range(n):
                lo = max(0, lens[b] + j + 1 - c["window"]) if c["window"] else 0
                hi = lens[b] + j + 1
                w = torch.softmax((q[b, j, h] @ k[lo:hi].t().contiguous()) * s["scale"], -1)
                out[b, j, h * g:(h + 1) * g] = w @ v[lo:hi]
    return out.view(S * n, c["q_heads"], D)


def _exact_rows(x, bits):
    """What rows of f16 values (numpy float64 [.., D]) read back as."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    least = g.min(-1, keepdims=True) if bits == 4 else np.zeros((*g.shape[:-1], 1))
    steps = 15 if bits == 4 else 127
    width = g.max(-1, keepdims=True) - least if bits == 4 else np.abs(g).max(-1, keepdims=True)
    d = (width / steps).astype(np.float16)
    d = np.where(d.astype(np.float64) * steps < width, np.nextafter(d, np.float16(np.inf)), d).astype(np.float64)
    code = np.rint(np.divide(g - least, d, out=np.zeros_like(g), where=d > 0))
    return (code * d + least).reshape(x.shape)


def _exact_append(c, seed):
    s = _append_case(c, seed)
    n, H, Q, D = c["n_new"], c["kv_heads"], c["q_heads"], c["dim"]
    x = s["qkv"].double().view(c["seqs"], n, -1, D).cpu().numpy()
    pos = s["lens"].cpu().numpy()[:, None] + np.arange(n)
    turn = np.exp(1j * pos[..., None, None] * np.power(THETA, -np.arange(0, D, 2) / D))
    z = (x[:, :, :Q + H, :D // 2] + 1j * x[:, :, :Q + H, D // 2:]) * turn
    r = np.concatenate([z.real, z.imag], -1)
    k = _exact_rows(r[:, :, Q:].astype(np.float16).astype(np.float64), c["bits"])   # keys are f16 before they are stored
    v = _exact_rows(x[:, :, Q + H:], c["bits"])
    return {"q": r[:, :, :Q].reshape(-1, Q, D), "k": k.transpose(0, 2, 1, 3), "v": v.transpose(0, 2, 1, 3)}


def _exact_read(c, seed):
    s = _read_case(c, seed)
    out = {}
    table = s["table"].long()
    for plane, name in ((0, "k"), (1, "v")):
        x = _exact_values(s["pool"][plane], c)
        y = torch.zeros_like(s[name], dtype=torch.float64)
        for i, slot in enumerate(s["slots"].tolist()):
            for p in range(0, c["length"], c["page"]):
                m = min(c["page"], c["length"] - p)
                y[i, :, p:p + m] = x[table[slot, p // c["page"]], :, :m].double()
        out[name] = y
    return out


def _exact_logprobs(c, seed):
    s = _logprobs_case(c, seed)
    temp, tokens = s["temp"].double().tolist(), s["tokens"].tolist()
    rows = len(tokens)
    f64 = dict(dtype=torch.float64, device="cuda")
    lp, ent = torch.empty(rows, **f64), torch.empty(rows, **f64)
    ids, alt = torch.empty((rows, c["top"]), dtype=torch.int32, device="cuda"), torch.empty((rows, c["top"]), **f64)
    for i in range(rows):
        x = s["x"][i].double()
        if c["cap"]:
            x = torch.where(x.isinf(), x, c["cap"] * torch.tanh(x / c["cap"]))
        y = torch.log_softmax(x / temp[i // c["rows"]], 0)
        lp[i] = y[tokens[i]]
        ent[i] = -(y.exp() * torch.where(y.isinf(), 0.0, y)).sum()
        if c["top"]:
            ids[i] = torch.sort(s["x"][i].float(), descending=True, stable=True).indices[:c["top"]]
            alt[i] = y[ids[i].long()]
    out = {"logprob": lp, "entropy": ent}
    return out | ({"top_ids": ids, "top_logprobs": alt} if c["top"] else {})


def exact(case, seed):
    f = {"attn": _exact_attn, "append": _exact_append, "read": _exact_read, "logprobs": _exact_logprobs}
    return f[case["op"]](case, seed)
