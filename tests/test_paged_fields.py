"""PagedKV's tensors stand behind the descriptor's pointers: they may be written,
not exchanged."""
import pytest

from cima_amd import hip as hipmod

torch = pytest.importorskip("torch")


class _OnDevice(torch.Tensor):
    """Host memory that passes for a device's: nothing here launches a kernel."""
    is_cuda = True

    def get_device(self):
        return 0


def _kv():
    from cima_amd.paged import PagedKV

    i32 = torch.int32
    t = [torch.zeros((4, 6, 2, 16, 64), dtype=torch.float16), torch.zeros(6, dtype=i32),
         torch.full((3, 5), -1, dtype=i32), torch.full((3,), -1, dtype=i32)]
    return PagedKV(*(x.as_subclass(_OnDevice) for x in t))


def test_descriptor_and_fields_agree():
    kv = _kv()
    d = kv.desc
    assert (d.pool, d.refs, d.table, d.lens) == tuple(t.data_ptr() for t in (kv.pool, kv.refs, kv.table, kv.lens))
    assert (d.n_planes, d.n_pages, d.kv_heads, d.page, d.head_dim, d.max_seqs, d.table_stride) == (4, 6, 2, 16, 64, 3, 5)


@pytest.mark.parametrize("name", ["pool", "refs", "table", "lens"])
def test_a_tensor_of_the_cache_is_not_exchanged(name):
    kv = _kv()
    old = getattr(kv, name)
    with pytest.raises(hipmod.EngineError, match=name) as e:
        setattr(kv, name, old.clone())
    assert e.value.code == hipmod.E_INVALID
    assert getattr(kv, name) is old and getattr(kv.desc, name) == old.data_ptr()


def test_a_tensor_of_the_cache_may_be_written():
    kv = _kv()
    kv.lens[0] = 3
    kv.lens += 1                                        # in place: the same tensor
    kv.refs.fill_(2)
    assert kv.lens.tolist() == [4, 0, 0] and kv.desc.lens == kv.lens.data_ptr() and int(kv.refs.sum()) == 12
