"""The operators of a batch that is served from quantised pages, run together as a
server runs them: prompts, continuations and drafts, what was written read back, the
tokens' log probabilities; captured and replayed, and on two streams.

Tolerances.  Codes, scales and values read back are equal.  The attention's error over
the values that the pages stand for is bounded as in test_gpu_paged.py (2^-11 relative to
the largest value twice for the weights and once for the result, and as much again where
q is rounded once more); log probabilities as in test_gpu_logprobs.py.
"""
import numpy as np
import pytest
from test_gpu_logprobs import _near, _want
from test_gpu_paged import EPS16, THETA, Batch, _attend, _check, _i32
from test_gpu_paged_quant import TYPES, QBatch, quantise, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _rotate(x, pos):
    D = x.shape[-1]
    z = (x[..., :D // 2] + 1j * x[..., D // 2:]) * np.exp(1j * pos * THETA ** (-np.arange(0, D, 2) / D))
    return np.concatenate([z.real, z.imag], -1)


def _cache(t, n_pages, page, slots, max_len, H, D, layers, seed):
    """An empty cache whose pages hold any bytes."""
    from cima_amd.paged import PagedKV

    kv = PagedKV.empty(layers, n_pages, H, page, D, slots, max_len, ggml_type=t)
    kv.pool.copy_(torch.from_numpy(np.random.default_rng(seed).integers(0, 256, tuple(kv.pool.shape), dtype=np.uint8)))
    return kv


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128)], ids=str)
def test_a_batch_of_continuations_step_by_step(hip, t, heads):
    """A prompt forked into four continuations that take steps of one to three tokens, one
    freed and its pages used again, the pool compacted in between: every step's attention
    and log probabilities against the host's own history, and the caches read back at
    the end."""
    Q, H, D = heads
    page, layers, V = 16, 2, 33001
    kv = _cache(t, 64, page, 6, 400, H, D, layers, 40)
    r = np.random.default_rng(41)
    status, live = _i32([1]), _i32([0])
    slab = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
    history = {}

    def step(seqs, n, prefix_pages, slot):
        hip.kv_pages_reserve(kv, seqs, n, status)
        assert int(status.item()) == 0
        lens, rows = kv.lens.cpu().numpy(), seqs * n
        for layer in range(layers):
            qkv = r.standard_normal((rows, Q + 2 * H, D)).astype(np.float16)
            q = torch.zeros((rows, Q, D), dtype=torch.float16, device="cuda")
            out = torch.empty_like(q)
            hip.rope_append_paged(kv, layer, torch.from_numpy(qkv).cuda(), q, seqs, n, Q, THETA)
            hip.attn_paged(kv, layer, q, out, seqs, n, Q, 1 / np.sqrt(D), slab, prefix_pages, slot)
            torch.cuda.synchronize()
            got = out.cpu().numpy().astype(np.float64)
            for s in range(seqs):
                for j in range(n):
                    if lens[s] < 0:
                        assert not got[s * n + j].any()
                        continue
                    x, pos = qkv[s * n + j], lens[s] + j
                    k, v = history[s][layer]
                    k.append(values(*quantise(_rotate(x[Q:Q + H].astype(np.float64), pos).astype(np.float16), t), t))
                    v.append(values(*quantise(x[Q + H:], t), t))
                    K, W = np.array(k, np.float64), np.array(v, np.float64)
                    qq = _rotate(x[:Q].astype(np.float64), pos).astype(np.float16).astype(np.float64)
                    for h in range(Q):
                        z = K[:, h // (Q // H)] @ qq[h] / np.sqrt(D)
                        w = np.exp(z - z.max())
                        want = w @ W[:, h // (Q // H)] / w.sum()
                        tol = 4 * EPS16 * np.abs(W).max() + EPS16 * np.abs(want)
                        assert (np.abs(got[s * n + j, h] - want) <= tol).all()
        logits = (r.standard_normal((rows, V)) * 3).astype(np.float16)
        tokens = r.integers(-1, V, rows)
        temp = r.uniform(0.5, 1.5, seqs).astype(np.float32)
        lp, ent, alt = (torch.zeros((rows, m), device="cuda") for m in (1, 1, 4))
        ids = torch.zeros((rows, 4), dtype=torch.int32, device="cuda")
        hip.logprobs_rows(torch.from_numpy(logits).cuda(), rows, V, _i32(tokens), lp, ent, 4, ids, alt,
                          torch.from_numpy(temp).cuda(), n, 0.0, slab)
        torch.cuda.synchronize()
        want = _want(logits, temp.repeat(n), 0.0, tokens, 4)
        assert np.array_equal(ids.cpu().numpy(), want[2])
        for g, w in ((lp[:, 0], want[0]), (ent[:, 0], want[1]), (alt, want[3])):
            _near(g.cpu().numpy(), *w)
        kv.lens.add_((kv.lens >= 0).int() * n)

    kv.lens[0] = 0
    history[0] = [([], []) for _ in range(layers)]
    step(1, 37, 0, 0)
    hip.kv_pages_fork(kv, _i32([0, 0, 0]), _i32([3, 1, 2]), 3, status)
    assert int(status.item()) == 0
    for c in (3, 1, 2):
        history[c] = [(list(k), list(v)) for k, v in history[0]]
    step(4, 1, 2, 0)
    step(4, 3, 2, 3)
    hip.kv_pages_free(kv, _i32([1]), 1)
    step(4, 2, 2, 0)
    hip.kv_pages_compact(kv, kv.refs, kv.table, live, slab)
    assert int(live.item()) == int((kv.refs > 0).sum())
    hip.kv_pages_fork(kv, _i32([2]), _i32([1]), 1, status)
    assert int(status.item()) == 0
    history[1] = [(list(k), list(v)) for k, v in history[2]]
    for n in (1, 2, 1):
        step(5, n, 2, 2)
    room = 64
    k, v = (torch.full((4, H, room, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    for layer in range(layers):
        hip.kv_pages_read(kv, layer, k, v, 4, room, slots=_i32([3, 1, 0, 2]), max_seq=room)
        torch.cuda.synchronize()
        for i, s in enumerate((3, 1, 0, 2)):
            for got, rows in zip((k, v), history[s][layer]):
                assert len(rows) == int(kv.lens[s])
                assert np.array_equal(got[i, :, :len(rows)].cpu().numpy(), np.array(rows).transpose(1, 0, 2))
    hip.kv_pages_free(kv, _i32([0, 1, 2, 3]), 4)
    torch.cuda.synchronize()
    assert not kv.refs.any() and (kv.table == -1).all() and (kv.lens == -1).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_a_captured_step_replays_as_the_batch_grows(hip, t):
    """Reserve, append, attention, read back, softmax, verification and the taken tokens'
    log probabilities recorded once and replayed while lengths, pages and slots change;
    an eager twin gives the same bits after every step, and the log probabilities are
    the host's."""
    Q, H, D, page, layers, S, n, V, top = 14, 2, 64, 16, 2, 4, 3, 40000, 3
    r = np.random.default_rng(70)
    twins = [_cache(t, 96, page, S, 900, H, D, layers, 71) for _ in range(2)]
    f32, i32, f16 = (dict(device="cuda", dtype=d) for d in (torch.float32, torch.int32, torch.float16))
    qkv = torch.zeros((layers, S * n, (Q + 2 * H) * D), **f16)
    logits = torch.zeros((S * n, V), **f16)
    drafts, u = torch.zeros((S, n - 1), **i32), torch.zeros((S, n), **f32)
    temp = torch.tensor([0.7, 0.0, 1.2, 1.0], **f32)
    slots = _i32([2, 0])
    bufs = [dict(q=torch.zeros((S * n, Q, D), **f16), out=torch.zeros((layers, S * n, Q, D), **f16),
                 p=torch.zeros((S * n, V), **f32), acc=torch.zeros(S, **i32), tok=torch.zeros((S, n), **i32),
                 k=torch.zeros((2, H, 128, D), **f16), v=torch.zeros((2, H, 128, D), **f16),
                 lp=torch.zeros(S * n, **f32), ent=torch.zeros(S * n, **f32), ids=torch.zeros((S * n, top), **i32),
                 alt=torch.zeros((S * n, top), **f32), status=torch.zeros(1, **i32),
                 slab=torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")) for _ in twins]

    def step(kv, b):
        hip.kv_pages_reserve(kv, S, n, b["status"])
        for layer in range(layers):
            hip.rope_append_paged(kv, layer, qkv[layer], b["q"], S, n, Q, THETA)
            hip.attn_paged(kv, layer, b["q"], b["out"][layer], S, n, Q, 0.125, b["slab"], prefix_pages=2, window=200)
        hip.kv_pages_read(kv, 1, b["k"], b["v"], 2, 100, slots=slots, max_seq=128)
        hip.softmax_rows(logits, b["p"], S * n, V, temp, n, 0.0, b["slab"])
        hip.verify_drafts(b["p"], None, drafts, None, u, b["acc"], b["tok"], kv.lens, S, n - 1, V, b["slab"])
        hip.logprobs_rows(logits, S * n, V, b["tok"], b["lp"], b["ent"], top, b["ids"], b["alt"], temp, n, 0.0, b["slab"])

    for kv, b in zip(twins, bufs):
        kv.lens[0] = 0
        hip.kv_pages_reserve(kv, 1, 37, b["status"])
        for layer in range(layers):
            x = torch.from_numpy(np.random.default_rng(layer).standard_normal((37, (Q + 2 * H) * D)).astype(np.float16))
            hip.rope_append_paged(kv, layer, x.cuda(), torch.zeros((37, Q * D), **f16), 1, 37, Q, THETA)
        kv.lens[0] = 37
        hip.kv_pages_fork(kv, _i32([0, 0]), _i32([1, 2]), 2, b["status"])
        torch.cuda.synchronize()
        assert b["status"].item() == 0
    st = torch.cuda.Stream()
    hip.set_stream(st)
    try:
        hip.capture_begin()
        try:
            step(twins[0], bufs[0])
        finally:
            g = hip.capture_end()
    finally:
        hip.use_torch_stream()
    for i in range(8):
        qkv.copy_(torch.from_numpy(r.standard_normal(qkv.shape).astype(np.float16)))
        logits.copy_(torch.from_numpy((r.standard_normal(logits.shape) * 3).astype(np.float16)))
        drafts.copy_(logits.view(S, n, V)[:, :n - 1].argmax(-1))
        u.copy_(torch.from_numpy(r.random((S, n)).astype(np.float32)))
        torch.cuda.synchronize()
        before = twins[1].lens.tolist()
        g.launch()
        torch.cuda.synchronize()
        step(twins[1], bufs[1])
        torch.cuda.synchronize()
        for key in bufs[0]:
            if key not in ("slab", "q"):
                one, two = (x[key].view(torch.int16) if key in "kv" else x[key] for x in bufs)  # NaN behind the lengths
                assert torch.equal(one, two), (i, key)
        for key in ("lens", "table", "refs", "pool"):
            assert torch.equal(getattr(twins[0], key), getattr(twins[1], key)), (i, key)
        assert bufs[0]["status"].item() == 0 and torch.isfinite(bufs[0]["out"]).all()
        taken = bufs[0]["acc"].tolist()
        assert twins[0].lens.tolist() == [m + a + 1 if m >= 0 else -1 for m, a in zip(before, taken)]
        tokens = bufs[0]["tok"].view(-1).cpu().numpy()
        want = _want(logits.cpu().numpy(), temp.repeat_interleave(n).cpu().numpy(), 0.0, tokens, top)
        assert np.array_equal(bufs[0]["ids"].cpu().numpy(), want[2])
        for key, w in (("lp", want[0]), ("ent", want[1]), ("alt", want[3])):
            _near(bufs[0][key].cpu().numpy(), *w)
        for kv, b in zip(twins, bufs):                  # the batch changes between the steps
            if i == 2:
                hip.kv_pages_fork(kv, _i32([2]), _i32([3]), 1, b["status"])
            if i == 4:
                hip.kv_pages_free(kv, _i32([1]), 1)
            if i == 5:
                hip.kv_pages_compact(kv, kv.refs, kv.table, b["status"], b["slab"])
            if i == 6:
                hip.kv_pages_fork(kv, _i32([3]), _i32([1]), 1, b["status"])
        torch.cuda.synchronize()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_two_streams_at_once(hip, t):
    """Calls that may run together, a slab each: the same bits as alone."""
    n, top = 50000, 8
    a, b = (QBatch(t, [512, 700, 513, 999], 2, (14, 2, 64), 64, 512, seed=s) for s in (21, 22))
    r = np.random.default_rng(23)
    qs = [torch.from_numpy(x.r.standard_normal((x.rows, x.q_heads, x.D)).astype(np.float16)).cuda() for x in (a, b)]
    xs = [torch.from_numpy((r.standard_normal((9, n)) * 3).astype(np.float16)).cuda() for _ in (a, b)]

    def outputs():
        f32 = dict(device="cuda", dtype=torch.float32)
        return [torch.zeros((a.rows, a.q_heads, a.D), dtype=torch.float16, device="cuda"), torch.zeros(9, **f32),
                torch.zeros((9, top), dtype=torch.int32, device="cuda"), torch.zeros((9, top), **f32),
                *(torch.zeros((4, 2, 600, 64), dtype=torch.float16, device="cuda") for _ in range(2))]

    def calls(x, q, logits, o, slab):
        hip.attn_paged(x.kv, 0, q, o[0], 4, 2, 14, 1.0 / np.sqrt(64), slab, prefix_pages=x.pp)
        hip.logprobs_rows(logits, 9, n, entropy=o[1], n_top=top, top_ids=o[2], top_logprobs=o[3], slab=slab)
        hip.kv_pages_read(x.kv, 0, o[4], o[5], 4, 600)
    slabs = [torch.empty(8 << 20, dtype=torch.uint8, device="cuda") for _ in (a, b)]
    alone, outs = [outputs() for _ in (a, b)], [outputs() for _ in (a, b)]
    for x, q, logits, o in zip((a, b), qs, xs, alone):
        calls(x, q, logits, o, slabs[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in (a, b)]
    try:
        for _ in range(10):
            for x, q, logits, o, slab, st in zip((a, b), qs, xs, outs, slabs, streams):
                hip.set_stream(st)
                calls(x, q, logits, o, slab)
    finally:
        hip.use_torch_stream()
    torch.cuda.synchronize()
    for o, want in zip(outs, alone):
        assert all(torch.equal(x, y) for x, y in zip(o, want))


# ------------------------------------------- prefixes of a few tens of rows

@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads,seqs,n_new", [((14, 2, 64), 5, 1), ((14, 2, 64), 9, 1), ((14, 2, 64), 12, 3),
                                              ((14, 2, 64), 37, 1), ((8, 2, 128), 9, 1), ((8, 2, 128), 3, 5),
                                              ((7, 1, 128), 8, 1), ((8, 2, 128), 17, 1)], ids=str)
@pytest.mark.parametrize("page,prefix,window", [(16, 48, 0), (16, 1040, 0), (64, 1984, 700), (256, 4096, 0)])
def test_attention_of_prefix_rows_on_both_sides_of_a_tile(hip, t, heads, seqs, n_new, page, prefix, window):
    """From 33 rows of a head on the prefix is read in tiles of 32 rows, from 65 (of
    heads of 64: 257) in larger ones; the last tile is not full."""
    lens = [prefix + (13 * s) % 77 for s in range(seqs)]
    if seqs > 4:
        lens[1] = -1
    _check(hip, QBatch(t, lens, n_new, heads, page, prefix, seed=seqs, spare=1500 // page), window)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_of_many_slots(hip, t):
    """700 slots, most of them free."""
    r = np.random.default_rng(31)
    lens = np.where(r.random(700) < 0.9, -1, r.integers(0, 300, 700)).tolist()
    b = QBatch(t, lens, 1, (8, 4, 64), 32, seed=32)
    _check(hip, b)
    _check(hip, b, slab_mb=0.05)
    q = b.r.standard_normal((b.rows, b.q_heads, b.D)).astype(np.float16)
    got = _attend(hip, b, q)
    assert not got[np.array(lens) < 0].any()


@pytest.mark.parametrize("t", [0, *TYPES], ids=str)
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)], ids=str)
def test_a_slot_handed_to_the_single_sequence_attention(hip, t, heads):
    """A slot read out of the pages is the contiguous cache of attn_decode: both
    attentions are within their bound of the same 64-bit result."""
    Q, H, D = heads
    lens, room, csz = [40, 333], 512, 128
    b = QBatch(t, lens, 1, heads, 16, seed=33) if t else Batch(lens, 1, heads, 16, seed=33)
    q = b.r.standard_normal((b.rows, Q, D)).astype(np.float16)
    qd = torch.from_numpy(q).cuda()
    k, v = (torch.zeros((1, H, room, D), dtype=torch.float16, device="cuda") for _ in range(2))
    out = torch.empty((Q, D), dtype=torch.float16, device="cuda")
    hip.kv_pages_read(b.kv, 0, k, v, 1, 334, slots=_i32([1]), max_seq=room)
    hip.attn_decode_noalloc(qd[1], k, v, out, Q, H, D, 334, room, csz, -(-room // csz), 1 / np.sqrt(D))
    paged = _attend(hip, b, q)[1]
    want, tol = (x[1] for x in b.want(q, 1 / np.sqrt(D), 0))
    assert (np.abs(paged - want) <= tol).all()
    assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= tol).all()


# --------------------------------------------- slots in the order of their lengths

@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("seqs,n_new,window", [(130, 1, 0), (256, 1, 0), (257, 1, 0), (129, 5, 0), (150, 1, 40)])
def test_attention_of_slots_taken_by_length(hip, t, seqs, n_new, window):
    """Lengths of every kind and number: each slot is served once."""
    r = np.random.default_rng(seqs)
    for lens in (r.integers(-1, 200, seqs), np.full(seqs, 37), np.where(np.arange(seqs) == seqs - 1, 600, -1),
                 np.arange(seqs) * 2, np.zeros(seqs)):
        _check(hip, QBatch(t, [int(n) for n in lens], n_new, (8, 4, 64), 32, seed=34), window)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_lengths_out_of_range_do_no_harm(hip, t):
    """Lengths behind the table and below -1: the other slots' results are what they
    are alone, slots of negative lengths have zeros."""
    b = QBatch(t, [70 + 3 * i for i in range(140)], 1, (8, 4, 64), 32, seed=35)
    q = b.r.standard_normal((b.rows, 8, 64)).astype(np.float16)
    want = _attend(hip, b, q)
    odd = {3: 2 ** 31 - 2, 64: -2 ** 31, 90: -7, 139: 2 ** 30}
    for s, n in odd.items():
        b.kv.lens[s] = n
    got = _attend(hip, b, q)
    rest = [s for s in range(140) if s not in odd]
    assert np.array_equal(got[rest], want[rest])
    assert not got[[64, 90]].any()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_a_captured_batch_of_slots_whose_lengths_change(hip, t):
    """A captured call replayed with lengths that rise, fall and end, against the eager one."""
    b = QBatch(t, [400] * 136, 1, (8, 4, 64), 32, seed=36)
    r = np.random.default_rng(37)
    q = torch.from_numpy(r.standard_normal((136, 8, 64)).astype(np.float16)).cuda()
    out, eager = (torch.zeros((136, 8, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    slabs = [torch.empty(8 << 20, dtype=torch.uint8, device="cuda") for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    hip.set_stream(s)
    try:
        hip.capture_begin()
        try:
            hip.attn_paged(b.kv, 0, q, out, 136, 1, 8, 0.125, slabs[0])
        finally:
            g = hip.capture_end()
    finally:
        hip.use_torch_stream()
    for _ in range(4):
        b.kv.lens.copy_(_i32(r.integers(-1, 400, 136)))
        torch.cuda.synchronize()
        g.launch()
        torch.cuda.synchronize()
        hip.attn_paged(b.kv, 0, q, eager, 136, 1, 8, 0.125, slabs[1])
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.isfinite(out).all()
        b.lens = b.kv.lens.tolist()
        want, tol = b.want(q.cpu().numpy(), 0.125, 0)
        assert (np.abs(out.cpu().numpy() - want) <= tol).all()


# ------------------------------------------------ few slots: a task, a workgroup of eight waves

@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads,n_new", [((14, 2, 64), 1), ((14, 2, 64), 5), ((12, 12, 64), 1), ((32, 8, 128), 1),
                                         ((28, 4, 128), 5), ((16, 1, 128), 1)], ids=str)
@pytest.mark.parametrize("longest", [240, 257, 300, 380, 450, 600, 860, 1500])
def test_attention_of_a_few_slots(hip, t, heads, n_new, longest):
    """Tables around the lengths at which a task has more waves or is split: without a slab
    in one launch, with one as it is planned, behind pages that are shared, in a window."""
    lens = [longest - n_new, 0, 31, -1, longest // 2]
    for prefix, window, slab in ((0, 0, 0), (0, 0, 32), (0, 37, 32), (0, longest // 2, 32), (208, 0, 32)):
        own = [n if n < 0 else max(n, prefix) for n in lens]
        _check(hip, QBatch(t, own, n_new, heads, 16, prefix, seed=longest + n_new), window, slab)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_a_few_slots_without_some_pages(hip, t, dim):
    """Positions that have no page are not seen, whichever wave's they are."""
    b = QBatch(t, [700, 333], 1, (4, 2, dim), 16, seed=40)
    q = b.r.standard_normal((2, 4, dim)).astype(np.float16)
    gone = [(0, 3), (0, 17), (0, 18), (0, 40), (1, 0), (1, 20)]
    for s, e in gone:
        b.kv.table[s, e] = -1 if e % 2 else 10 ** 6
    got = _attend(hip, b, q)
    for s in range(2):
        p = np.array([i for i in range(b.lens[s] + 1) if (s, i // 16) not in gone])
        ids = b.table[s, p // 16]
        for h in range(4):
            k, v = (b.pool[c, ids, h // 2, p % 16].astype(np.float64) for c in range(2))
            z = k @ q[s, h].astype(np.float64) / np.sqrt(dim)
            w = np.exp(z - z.max())
            want = w @ v / w.sum()
            assert (np.abs(got[s, h] - want) <= 2 * EPS16 * np.abs(v).max() + EPS16 * np.abs(want)).all()
