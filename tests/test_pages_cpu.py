"""The page-table calls without a GPU: the C entries' refusals, and the list
oracle's own invariants (every page held, free or pinned, once)."""
import ctypes as ct
import random

import pytest
import torch

import pages_oracle as O
from bmx_amd import _lib, pages

FAKE = 1 << 20   # never dereferenced


def _update(**kw):
    a = _lib.PagesUpdateArgs()
    for i, s in enumerate((getattr(a, "in"), a.out)):
        s.table, s.n_pages, s.refs, s.free, s.n_free = (FAKE * (1 + 5 * i + j) for j in range(5))
    a.rows = a.new_rows = 4
    a.cap, a.n_pool, a.status = 16, 100, FAKE
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(rows=0), "rows"), (dict(rows=20000), "rows"), (dict(new_rows=0), "new_rows"), (dict(cap=0), "cap"),
    (dict(cap=1 << 23), "cap"), (dict(n_pool=0), "n_pool"), (dict(n_pool=1 << 23), "n_pool"), (dict(new_rows=5), "without an index"),
    (dict(status=None), "status"),
])
def test_update_refuses(kw, word):
    a = _update(**kw)
    L = _lib.lib()
    assert L.bmx_pages_update(ct.byref(a), None) == 1 and word in L.bmx_last_error().decode()
    assert L.bmx_pages_update_workspace_bytes(ct.byref(a)) == 0


def test_update_needs_its_workspace_and_buffers_of_its_own():
    L = _lib.lib()
    a = _update()
    need = L.bmx_pages_update_workspace_bytes(ct.byref(a))
    a.workspace, a.workspace_bytes = FAKE, need - 1
    assert need > 0 and L.bmx_pages_update(ct.byref(a), None) == 2
    a.workspace, a.workspace_bytes = FAKE + 4, need
    assert L.bmx_pages_update(ct.byref(a), None) == 2
    a = _update()
    a.out.refs = getattr(a, "in").refs
    assert L.bmx_pages_update(ct.byref(a), None) == 1 and b"buffers of its own" in L.bmx_last_error()
    a = _update()
    a.out.free = None
    assert L.bmx_pages_update(ct.byref(a), None) == 1 and b"non-NULL" in L.bmx_last_error()
    assert L.bmx_pages_update(None, None) == 1


def _compact(**kw):
    a = _lib.PagesCompactArgs()
    for i, s in enumerate((getattr(a, "in"), a.out)):
        s.table, s.n_pages, s.refs, s.free, s.n_free = (FAKE * (1 + 5 * i + j) for j in range(5))
    a.rows, a.cap, a.n_pool, a.n_pools = 4, 16, 100, 1
    a.pools[0], a.page_bytes[0] = FAKE, 12032
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_compact_refuses():
    L = _lib.lib()
    for kw, word in ((dict(n_pools=129), "n_pools"), (dict(n_pools=-1), "n_pools"), (dict(n_pools=2), "non-NULL"),
                     (dict(rows=0), "rows"), (dict(n_pool=0), "n_pool")):
        assert L.bmx_pages_compact(ct.byref(_compact(**kw)), None) == 1 and word in L.bmx_last_error().decode()
    a = _compact()
    a.page_bytes[0] = 40
    assert L.bmx_pages_compact(ct.byref(a), None) == 1 and b"multiple of 16" in L.bmx_last_error()
    a = _compact()
    a.pools[0] = FAKE + 8
    assert L.bmx_pages_compact(ct.byref(a), None) == 1 and b"aligned" in L.bmx_last_error()
    a = _compact()
    need = L.bmx_pages_compact_workspace_bytes(ct.byref(a))
    a.workspace, a.workspace_bytes = FAKE, need - 1
    assert need > 0 and L.bmx_pages_compact(ct.byref(a), None) == 2


def test_wrapper_refuses_cpu_states():
    with pytest.raises(ValueError, match="HIP device"):
        pages.update(pages.PageState.make(2, 4, 8, "cpu"))
    with pytest.raises(ValueError, match="rows"):
        pages.PageState.make(0, 4, 8, "cpu")
    s = pages.PageState.make(2, 4, 8, "cpu")
    assert s.free.tolist() == list(range(7, -1, -1)) and s.n_free.item() == 8
    assert s.like(3).table.shape == (3, 4) and s.like().refs.shape == (8,) and torch.int32 is s.like().table.dtype


def test_oracle_keeps_every_page_accounted_for():
    rng = random.Random(0)
    for _ in range(50):
        rows, cap, pool = rng.randint(1, 6), rng.randint(1, 9), rng.randint(4, 60)
        st = ([[0] * cap for _ in range(rows)], [0] * rows, [0] * pool, list(range(pool - 1, -1, -1)), pool)
        for _ in range(6):
            index = [rng.randint(-1, len(st[0]) - 1) for _ in range(rng.randint(1, 6))]
            *st, status = O.update(*st, cap, index, [rng.randint(0, 3) for _ in index])
            held = [p for r, n in zip(st[0], st[1]) for p in r[:n]]
            assert sorted(set(held) | set(st[3][:st[4]])) == list(range(pool)) and not set(held) & set(st[3][:st[4]])
            assert all(held.count(p) == st[2][p] for p in range(pool))
            *st, moves = O.compact(*st[:3], cap)
            assert all(st[2][p] > 0 for p in range(pool - st[4])) and all(r == 0 for r in st[2][pool - st[4]:])
