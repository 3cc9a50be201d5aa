"""Page operations at sizes where their loops take more than one round: more
than 16 chunks of 1024 pages, more than 1024 slots and more than 1024 entries of
a slot; and too few pages."""
import numpy as np
import pytest
from test_gpu_paged import Pages, _i32, _some_cache

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _sync_from(kv, host):
    kv.refs.copy_(torch.from_numpy(host.refs))
    kv.table.copy_(torch.from_numpy(host.table))
    kv.lens.copy_(torch.from_numpy(host.lens))


@pytest.mark.parametrize("short", [0, 1, 5])
def test_fork_with_too_few_pages(hip, short):
    """Six children whose parent has begun a page: with enough pages, with one too
    few and with one alone; a shortage changes nothing and the children stay free."""
    kv = _some_cache(60, 16, max_seqs=12, max_len=200)
    host, status = Pages(kv), _i32([99])
    kv.lens[0] = host.lens[0] = 0
    hip.kv_pages_reserve(kv, 1, 40, status)
    assert host.reserve(1, 40) == status.item() == 0
    host.lens[0] = 35                                   # two pages and three rows
    free = np.flatnonzero(host.refs == 0)
    host.refs[free[6 - short:]] = 1
    _sync_from(kv, host)
    kids = [3, 1, 9, 4, 11, 2]
    hip.kv_pages_fork(kv, _i32([0] * 6), _i32(kids), 6, status)
    torch.cuda.synchronize()
    assert status.item() == host.fork([0] * 6, kids) == short
    host.same(kv)
    assert (host.lens[kids] == (-1 if short else 35)).all()


@pytest.mark.parametrize("n_pages", [17 * 1024, 40000, 40 * 1024 + 1])
def test_operations_over_many_chunks(hip, n_pages):
    """Held and free pages mixed over all chunks: reserve, fork and compaction
    take the lowest free ones in order."""
    kv = _some_cache(n_pages, 16, max_seqs=9, max_len=16 * 9000, heads=1, dim=64, layers=1, seed=5)
    host, r, status, live = Pages(kv), np.random.default_rng(n_pages), _i32([5]), _i32([5])
    host.refs[:] = r.random(n_pages) < np.linspace(0.9, 0.3, n_pages)
    host.refs[5000:7100] = 1                            # chunks without a free page
    host.refs[-1024:] = 0
    host.lens[:3] = [0, 40, 7]
    for s, k in ((1, 3), (2, 1)):                       # their tokens' pages, from all over
        at = r.choice(np.flatnonzero(host.refs == 0), k, replace=False)
        host.table[s, :k], host.refs[at] = at, 1
    _sync_from(kv, host)
    n = 16 * (int((host.refs == 0).sum()) // 4)         # three quarters of what is free
    hip.kv_pages_reserve(kv, 9, n, status)
    torch.cuda.synchronize()
    assert status.item() == host.reserve(9, n) == 0
    host.same(kv)
    host.lens[:3] += n - 3
    _sync_from(kv, host)
    kids = [8, 3, 5, 4]
    hip.kv_pages_fork(kv, _i32([1, 2, 0, 1]), _i32(kids), 4, status)
    torch.cuda.synchronize()
    assert status.item() == host.fork([1, 2, 0, 1], kids) == 0
    host.same(kv)
    hip.kv_pages_free(kv, _i32([0, 5]), 2)
    host.free([0, 5])
    host.same(kv)
    # thousands of pages move
    before = host.refs.copy()
    hip.kv_pages_compact(kv, kv.refs, kv.table, live, torch.empty(12 * n_pages + 64, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    assert live.item() == host.compact() == (before != 0).sum()
    assert (before[live.item():] != 0).sum() > 1000
    host.same(kv)
    # one page too few for the five slots, then just enough
    want = 5 * (int((host.refs == 0).sum()) // 5 - 1)
    free = np.flatnonzero(host.refs == 0)
    host.lens[host.lens >= 0] = host.lens[host.lens >= 0] // 16 * 16
    for s in range(9):                                  # their entries from there on are empty
        host.table[s, max(0, host.lens[s]) // 16:] = -1
    for spare, short in ((want - 1, 1), (want, 0)):
        host.refs[free] = np.arange(len(free)) >= spare
        _sync_from(kv, host)
        hip.kv_pages_reserve(kv, 9, 16 * (want // 5), status)
        torch.cuda.synchronize()
        assert status.item() == host.reserve(9, 16 * (want // 5)) == short
        host.same(kv)


def test_operations_on_thousands_of_slots(hip):
    """3000 slots: reserve and fork take them 1024 at a time."""
    slots = 3000
    kv = _some_cache(15000, 16, max_seqs=slots, max_len=96, heads=1, dim=64, layers=1, seed=6)
    host, r, status = Pages(kv), np.random.default_rng(7), _i32([5])
    host.lens[:] = np.where(r.random(slots) < 0.45, 0, -1)
    _sync_from(kv, host)
    hip.kv_pages_reserve(kv, slots, 37, status)
    torch.cuda.synchronize()
    assert status.item() == host.reserve(slots, 37) == 0
    host.same(kv)
    host.lens[host.lens == 0] = r.choice([16, 32, 33, 37], (host.lens == 0).sum())
    _sync_from(kv, host)
    hip.kv_pages_reserve(kv, 2777, 20, status)          # not all of the slots
    torch.cuda.synchronize()
    assert status.item() == host.reserve(2777, 20) == 0
    host.same(kv)
    kids = r.permutation(np.flatnonzero(host.lens < 0))[:1400]
    parents = r.choice(np.flatnonzero(host.lens >= 0), len(kids))
    assert len(kids) == 1400
    keep = host.refs.copy()                             # first with one page too few
    need = int((host.lens[parents] % 16 > 0).sum())
    free = np.flatnonzero(host.refs == 0)
    host.refs[free[need - 1:]] = 1
    _sync_from(kv, host)
    hip.kv_pages_fork(kv, _i32(parents), _i32(kids), 1400, status)
    torch.cuda.synchronize()
    assert status.item() == host.fork(parents.tolist(), kids.tolist()) == 1
    host.same(kv)
    host.refs = keep
    _sync_from(kv, host)
    wrong = kids.copy()                                 # a child named twice, far apart
    wrong[1390] = wrong[3]
    hip.kv_pages_fork(kv, _i32(parents), _i32(wrong), 1400, status)
    torch.cuda.synchronize()
    assert status.item() == host.fork(parents.tolist(), wrong.tolist()) == -1
    host.same(kv)
    hip.kv_pages_fork(kv, _i32(parents), _i32(kids), 1400, status)
    torch.cuda.synchronize()
    assert status.item() == host.fork(parents.tolist(), kids.tolist()) == 0
    host.same(kv)
    out = r.permutation(slots)[:2000]
    hip.kv_pages_free(kv, _i32(out), 2000)
    host.free(out.tolist())
    host.same(kv)


def test_slots_of_thousands_of_entries(hip):
    """2500 entries: freed, and shared by a fork, 1024 or 256 at a time."""
    kv = _some_cache(3000, 16, max_seqs=4, max_len=40000, heads=1, dim=64, layers=1, seed=8)
    host, status = Pages(kv), _i32([5])
    kv.lens[1] = host.lens[1] = 0
    hip.kv_pages_reserve(kv, 2, 16 * 2400 + 5, status)
    assert host.reserve(2, 16 * 2400 + 5) == status.item() == 0
    host.lens[1] = 16 * 2400 + 5
    _sync_from(kv, host)
    hip.kv_pages_fork(kv, _i32([1]), _i32([3]), 1, status)
    torch.cuda.synchronize()
    assert status.item() == host.fork([1], [3]) == 0
    host.same(kv)
    for s in (1, 3):
        hip.kv_pages_free(kv, _i32([s, s]), 2)
        host.free([s])
        host.same(kv)
    assert not host.refs.any()


def test_a_random_history_with_room_and_without(hip):
    """Requests that start, branch, end and are moved together in a pool that is
    often full; every kind of answer comes up."""
    n_pages, slots = 40, 12
    kv = _some_cache(n_pages, 16, max_seqs=slots)
    host, r = Pages(kv), np.random.default_rng(3)
    status, live = _i32([77]), _i32([0])
    slab = torch.empty(12 * n_pages + 64, dtype=torch.uint8, device="cuda")
    seen = set()
    for step in range(200):
        free, used = np.flatnonzero(host.lens < 0), np.flatnonzero(host.lens >= 0)
        op = r.choice(["start", "fork", "fork", "fork", "grow", "grow", "end", "compact"])
        if op in ("start", "grow"):
            if op == "start" and len(free):
                kv.lens[free[0]] = host.lens[free[0]] = 0
            n = int(r.integers(1, 25))
            hip.kv_pages_reserve(kv, slots, n, status)
            got = host.reserve(slots, n)
            assert status.item() == got
            if got == 0:
                host.lens[host.lens >= 0] += n
                kv.lens.copy_(torch.from_numpy(host.lens))
            seen.add(("reserve", got > 0))
        elif op == "fork" and len(free) and len(used):
            kids = r.permutation(free)[:int(r.integers(1, 5))].tolist()
            parents = r.choice(used, len(kids)).tolist()
            hip.kv_pages_fork(kv, _i32(parents), _i32(kids), len(kids), status)
            got = host.fork(parents, kids)
            assert status.item() == got
            seen.add(("fork", got > 0))
        elif op == "end" and len(used):
            out = r.permutation(used)[:int(r.integers(1, 3))].tolist()
            hip.kv_pages_free(kv, _i32(out), len(out))
            host.free(out)
        elif op == "compact":
            held = int((host.refs != 0).sum())
            moves = int((host.refs[held:] != 0).sum())
            hip.kv_pages_compact(kv, kv.refs, kv.table, live, slab)
            assert host.compact() == live.item() == held
            seen.add(("moves", moves > 0))
        host.same(kv)
    assert seen >= {("reserve", False), ("reserve", True), ("fork", False), ("fork", True), ("moves", True)}, seen
