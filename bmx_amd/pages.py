"""Page tables of a batch over pools of cache pages, kept on the device: the
torch-facing wrapper of ``bmx_pages_update`` and ``bmx_pages_compact``
(include/bmx_pages.h).

A ``PageState`` holds which pool page is which page of which sequence; the
same ids serve the pools of all layers.  ``update`` forks, reorders and drops
rows by an index (a beam search's step, several samples of one prompt,
finished sequences), frees the pages that no row holds any more and hands out
new ones; ``compact`` moves the live pages of the pools to the lowest ids.
``table`` is the page table that ``k2b.decode``, ``k2b.decode_shared``,
``rtn.decode`` and the append calls' page ids read.  The reference keeps one
sequence's pages in Python lists (src/bmx/cache/packed_streaming.py:116-267).

The calls enqueue on torch's current stream and wait for nothing; a shortage
of pages is reported in the new state's ``status``, on the device.
"""

from __future__ import annotations

import ctypes as ct
from dataclasses import dataclass

import torch

from . import _lib
from .k2b import _need, launch

OK, NO_FREE, NO_ROOM = 0, 1, 2   # BMX_PAGES_*: values of PageState.status
MAX_POOLS = 128


@dataclass
class PageState:
    """int32 device tensors: table (rows, cap), row r's first n_pages[r] entries
    its pages in order; refs (n_pool,), the uses of each page (a table entry is
    one; a holder outside the tables adds its own); free (n_pool,), a stack of
    n_free[0] free ids, the top at its end; status (1,) of the update that made
    the state (compact leaves it; None in a new state of compact's)."""

    table: torch.Tensor
    n_pages: torch.Tensor
    refs: torch.Tensor
    free: torch.Tensor
    n_free: torch.Tensor
    status: torch.Tensor | None = None

    @staticmethod
    def make(rows: int, cap: int, n_pool: int, device) -> "PageState":
        """Empty rows over a pool whose pages are all free, the lowest id on top."""
        _need(1 <= rows and 1 <= cap and 1 <= n_pool, "rows, cap and n_pool must be >= 1")
        z = dict(dtype=torch.int32, device=device)
        return PageState(torch.zeros(rows, cap, **z), torch.zeros(rows, **z), torch.zeros(n_pool, **z),
                         torch.arange(n_pool - 1, -1, -1, **z), torch.full((1,), n_pool, **z), torch.zeros(1, **z))

    def like(self, rows: int | None = None) -> "PageState":
        """Buffers for a state over the same pool with `rows` rows (default: as many)."""
        t = self.table
        rows = t.shape[0] if rows is None else rows
        new, like = t.new_empty, torch.empty_like
        return PageState(new((rows, t.shape[1])), new(rows), like(self.refs), like(self.free), new(1), new(1))


def _check(s: PageState, what: str) -> int:
    """The state's device index."""
    t, l, r, f, n = s.table, s.n_pages, s.refs, s.free, s.n_free
    i32 = torch.int32
    _need(t.dtype is i32 and l.dtype is i32 and r.dtype is i32 and f.dtype is i32 and n.dtype is i32
          and t.is_contiguous() and l.is_contiguous() and r.is_contiguous() and f.is_contiguous(),
          f"{what}: contiguous int32 tensors")
    _need(t.dim() == 2 and l.shape == t.shape[:1] and r.dim() == 1 and f.shape == r.shape and n.numel() == 1,
          f"{what}: table (rows, cap), n_pages (rows,), refs and free (n_pool,), n_free (1,)")
    on = t.get_device()
    _need(on >= 0 and l.get_device() == on and r.get_device() == on and f.get_device() == on and n.get_device() == on,
          f"{what}: on one HIP device")
    return on


def _ptrs(s: PageState) -> tuple:
    return s.table.data_ptr(), s.n_pages.data_ptr(), s.refs.data_ptr(), s.free.data_ptr(), s.n_free.data_ptr()


def _out(state: PageState, out: PageState | None, rows: int, on: int) -> PageState:
    if out is None:
        return state.like(rows)
    _need(_check(out, "out") == on and out.table.shape == (rows, state.table.shape[1])
          and out.refs.shape == state.refs.shape, "out: a state of the new rows over the same pool")
    return out


def update(state: PageState, index: torch.Tensor | None = None, grow: torch.Tensor | None = None, *,
           out: PageState | None = None) -> PageState:
    """The next state: new row i continues old row index[i] (-1: empty; index
    None: every row as it is), pages that lost their last use go onto the free
    stack in ascending order, and row i gets grow[i] new pages off its top, row
    0's first -- all rows, or none and status NO_FREE (the stack is too short)
    or NO_ROOM (a row would pass cap).  Entries past a row's pages are 0, free
    ids past n_free -1.  ``out`` takes the new state in buffers of its own; the
    given one stays as it is."""
    on = _check(state, "state")
    old, cap = state.table.shape
    rows = old
    for x, what in ((index, "index"), (grow, "grow")):
        _need(x is None or (x.dtype is torch.int32 and x.dim() == 1 and x.is_contiguous() and x.get_device() == on),
              f"{what}: a contiguous int32 (rows,) tensor on the state's device")
    if index is not None:
        rows = index.shape[0]
    _need(grow is None or grow.shape[0] == rows, "grow: one count a new row")
    o = _out(state, out, rows, on)
    if o.status is None:
        o.status = o.n_free.new_empty(1)
    st = o.status
    _need(st.dtype is torch.int32 and st.numel() == 1 and st.get_device() == on,
          "out: status, one int32 on the state's device")
    dev = state.table.device
    a = _lib.PagesUpdateArgs(_ptrs(state), _ptrs(o), old, rows, cap, state.refs.shape[0],
                             None if index is None else index.data_ptr(), None if grow is None else grow.data_ptr(),
                             st.data_ptr())
    lib = _lib.lib()
    need = int(lib.bmx_pages_update_workspace_bytes(ct.byref(a)))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    launch(lib.bmx_pages_update, a, dev, "bmx_pages_update")
    return o


def compact(state: PageState, pools, *, out: PageState | None = None) -> PageState:
    """The state with its n live pages (refs > 0) at ids below n: those above
    move, lowest first, to the free ids below, in every pool of ``pools`` (uint8
    (n_pool, page_bytes) tensors, page sizes multiples of 16, changed in place).
    The free stack then hands out the lowest id first.  A holder outside the
    tables is not told its pages' new ids: one that reads them keeps them as a
    row of the table."""
    on = _check(state, "state")
    n_pool, dev = state.refs.shape[0], state.table.device
    pools = list(pools)
    _need(len(pools) <= MAX_POOLS, f"at most {MAX_POOLS} pools")
    for p in pools:
        _need(p.dtype is torch.uint8 and p.dim() == 2 and p.shape[0] == n_pool and p.is_contiguous()
              and p.get_device() == on, "pools: contiguous uint8 (n_pool, page_bytes) on the state's device")
        _need(p.shape[1] % 16 == 0 and p.shape[1] > 0, "pools: page_bytes must be a multiple of 16")
    o = _out(state, out, state.table.shape[0], on)
    if out is None:
        o.status = None
    a = _lib.PagesCompactArgs(_ptrs(state), _ptrs(o), *state.table.shape, n_pool, len(pools))
    for i, p in enumerate(pools):
        a.pools[i], a.page_bytes[i] = p.data_ptr(), p.shape[1]
    lib = _lib.lib()
    need = int(lib.bmx_pages_compact_workspace_bytes(ct.byref(a)))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    launch(lib.bmx_pages_compact, a, dev, "bmx_pages_compact")
    return o
