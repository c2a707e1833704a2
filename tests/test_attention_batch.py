"""What a PagedBatch hands to the library, on the CPU (its tensors only lend their addresses and strides here)."""
import pytest
import torch

from helios_b200 import _lib
from helios_b200 import attention as A


@pytest.fixture
def batch(monkeypatch):
    monkeypatch.setattr(A, "_int32", lambda t, dims, name: t)
    return A.PagedBatch(*tensors(2, 3), max_q=4, max_kv=40)


def tensors(n, pages):
    return tuple(torch.zeros(s, dtype=torch.int32) for s in ((n + 1,), (n,), (n, pages)))


def held(batch, page_size=16):
    return _lib.G4qPagedBatch.from_address(batch.view(page_size))


def test_assigned_fields_reach_the_next_call(batch):
    c = held(batch)
    assert (c.max_q, c.max_pages, c.n_seqs) == (4, 3, 2)
    assert batch.view(16) == batch.view(16)
    batch.max_q = 9
    assert batch.max_q == 9 and held(batch).max_q == 9
    batch.max_kv = 17
    assert held(batch).max_pages == 2 and held(batch, 32).max_pages == 1
    batch.max_kv = None
    assert held(batch).max_pages == 3
    _, kv, wide = tensors(2, 7)
    batch.block_table = wide
    assert batch.block_table is wide
    c = held(batch)
    assert (c.block_table, c.table_stride, c.max_pages) == (wide.data_ptr(), 7, 7)
    batch.kv_lens = kv
    assert held(batch).kv_lens == kv.data_ptr() and held(batch).block_table == wide.data_ptr()


def test_fields_that_do_not_fit_are_refused_and_change_nothing(batch):
    was = batch.q_offsets, batch.kv_lens, batch.block_table, batch.max_q, batch.max_kv
    off, kv, table = tensors(3, 3)
    for name, bad in (("q_offsets", off), ("kv_lens", kv), ("block_table", table), ("max_q", 0), ("max_q", 2 ** 31), ("max_kv", 0)):
        with pytest.raises(ValueError):
            setattr(batch, name, bad)
    assert (batch.max_q, batch.max_kv) == was[3:]
    assert all(a is b for a, b in zip((batch.q_offsets, batch.kv_lens, batch.block_table), was))
    assert (held(batch).max_q, held(batch).n_seqs) == (4, 2)


def test_a_call_keeps_the_view_that_it_was_given(batch):
    """Another thread may assign a field while the library reads the structure of a call."""
    address, view = batch._held(16)
    batch.max_q = 11
    assert _lib.G4qPagedBatch.from_address(address).max_q == 4 and view.max_q == 4 and held(batch).max_q == 11


class Lent(torch.Tensor):
    """A CPU tensor that passes for a CUDA one, for the addresses and strides."""
    is_cuda = True


def test_a_cache_stays_as_it_was_made():
    k, v, other = (torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16).as_subclass(Lent) for _ in range(3))
    cache = A.PagedKVCache(k, v)
    for name, value in (("k", other), ("v", other), ("page_size", 32), ("n_pages", 8), ("c", None)):
        with pytest.raises(AttributeError, match="make another one"):
            setattr(cache, name, value)
    cache.layer = 3          # a caller's own
    assert cache.k is k and cache.v is v and (cache.page_size, cache.n_pages) == (16, 4)
    assert _lib.G4qPagedCache.from_address(cache.c_addr).k == k.data_ptr()


def test_the_stride_of_a_single_entry_is_not_used():
    """The length of one sequence out of a column, a table of one page out of a wider one."""
    def lent(*shape):
        return torch.zeros(*shape, dtype=torch.int32).as_subclass(Lent)

    off, column, wide = lent(2), lent(5, 3), lent(1, 12)
    batch = A.PagedBatch(off, column[2:3, 1], wide[:, ::12], max_q=1)
    c = held(batch)
    assert c.kv_lens == column.data_ptr() + 7 * 4 and (c.block_table, c.max_pages) == (wide.data_ptr(), 1)
    assert c.table_stride >= c.max_pages
    for bad in ((lent(4)[::2], column[2:3, 1], wide), (off, column[:, 1], lent(5, 3)), (off, column[2:3, 1], wide[:, ::2])):
        with pytest.raises(ValueError, match="contiguous rows"):
            A.PagedBatch(*bad, max_q=1)
