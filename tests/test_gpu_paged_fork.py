"""Forks of slots that are not as they must be."""
import pytest
from test_gpu_paged import Pages, _i32, _some_cache

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_fork_of_a_parent_that_lacks_its_begun_page(hip):
    """The child would get a page of no one's tokens: refused, nothing changed."""
    kv = _some_cache(30, 16, max_seqs=6, max_len=200)
    status = _i32([7])
    kv.lens[:2] = 0
    hip.kv_pages_reserve(kv, 2, 40, status)
    kv.lens[:2] = 37
    torch.cuda.synchronize()
    good = int(kv.table[1, 2].item())
    for bad in (-1, 30, 10 ** 6, -9):
        kv.table[1, 2] = bad
        for parents, children in (([1], [3]), ([0, 1, 0], [4, 2, 5])):
            before = Pages(kv)
            hip.kv_pages_fork(kv, _i32(parents), _i32(children), len(parents), status)
            torch.cuda.synchronize()
            assert status.item() == -1
            before.same(kv)
    # a page that is full and missing is nobody's: the children lack it too
    kv.table[1, 2] = good
    kv.table[1, 0] = -1
    before = Pages(kv)
    hip.kv_pages_fork(kv, _i32([1, 0]), _i32([3, 2]), 2, status)
    torch.cuda.synchronize()
    assert status.item() == 0
    assert kv.table[3].tolist()[:3] == [-1, int(before.table[1, 1]), int(before.lowest(1)[0])]
    assert kv.refs[int(before.table[1, 1])].item() == before.refs[before.table[1, 1]] + 1
