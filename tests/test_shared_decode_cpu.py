"""The C entry's refusals of the shared-prefix decode, without a GPU: no call
gets past its checks."""
import ctypes as ct

import pytest

from bmx_amd import _lib

FAKE = 1 << 20   # never dereferenced


def _args(**kw):
    a = _lib.DecodeSharedArgs()
    a.geom = _lib.Geom(8, 32, 4)
    a.batch, a.io_dtype = 2, 1
    a.q = a.out = a.pages = a.page_table = a.packed_len = a.basis = a.rope = a.k_tail = a.v_tail = FAKE
    a.n_pool_pages, a.max_pages, a.max_packed_len, a.shared_len, a.rope_pages = 100, 64, 1024, 512, 64
    a.rope_scaling, a.sm_scale = 1.0, 0.1
    a.codebook[:] = (-1.5, -0.5, 0.5, 1.5)
    a.tail_cap, a.tail_len_value = 32, 5
    a.tail_stride_b, a.tail_stride_h, a.tail_stride_t = 8 * 32 * 128, 32 * 128, 128
    for k, v in kw.items():
        if k == "geom":
            a.geom = _lib.Geom(*v)
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(geom=(8, 64, 4)), "recipe's page"), (dict(geom=(8, 32, 4, 64)), "recipe's page"), (dict(geom=(17, 32, 4)), "h_kv"),
    (dict(geom=(0, 32, 4)), "h_kv"), (dict(geom=(8, 32, 17)), "n_q_groups"), (dict(geom=(8, 32, 0)), "n_q_groups"),
    (dict(batch=0), "batch"), (dict(batch=70000), "batch"), (dict(io_dtype=0), "io_dtype"), (dict(io_dtype=3), "io_dtype"),
    (dict(max_packed_len=1000), "max_packed_len"), (dict(max_packed_len=1 << 24), "2\\^24"),
    (dict(shared_len=64), "shared_len"), (dict(shared_len=1152), "shared_len"), (dict(shared_len=-128), "shared_len"),
    (dict(tail_cap=5000), "tail_cap"), (dict(tail_len_value=33), "tail_len_value"), (dict(rope_scaling=0.0), "rope_scaling"),
    (dict(rope_scaling=float("nan")), "rope_scaling"), (dict(q=None), "non-NULL"), (dict(out=FAKE + 2), "aligned"),
    (dict(pages=None), "non-NULL"), (dict(rope=None), "non-NULL"), (dict(basis=FAKE + 8), "aligned"),
    (dict(n_pool_pages=0), "n_pool_pages"), (dict(max_pages=63), "max_pages"), (dict(rope_pages=63), "rope_pages"),
    (dict(k_tail=None), "k_tail"), (dict(tail_stride_t=132), "strides"), (dict(v_tail=FAKE + 2), "aligned"),
])
def test_c_entry_refuses(kw, word):
    import re
    a = _args(**kw)
    assert _lib.lib().bmx_k2b_decode_shared(ct.byref(a), None) != 0
    assert re.search(word, _lib.lib().bmx_last_error().decode()), _lib.lib().bmx_last_error()
    assert _lib.lib().bmx_k2b_decode_shared_workspace_bytes(ct.byref(a)) == 0


def test_codebook_that_does_not_ascend_is_refused():
    a = _args()
    a.codebook[:] = (-1.5, 0.5, 0.5, 1.5)
    assert _lib.lib().bmx_k2b_decode_shared(ct.byref(a), None) != 0
    assert b"codebook" in _lib.lib().bmx_last_error()


def test_workspace_is_asked_for_and_checked():
    a = _args()
    need = _lib.lib().bmx_k2b_decode_shared_workspace_bytes(ct.byref(a))
    rows = 2 * 8 * 4
    assert need > 0 and need % (rows * 132 * 4) == 0     # whole partial slots of every row
    a.workspace, a.workspace_bytes = FAKE, need - 1
    assert _lib.lib().bmx_k2b_decode_shared(ct.byref(a), None) == 2
    a.workspace, a.workspace_bytes = None, need
    assert _lib.lib().bmx_k2b_decode_shared(ct.byref(a), None) == 2
    assert _lib.lib().bmx_k2b_decode_shared(None, None) != 0


def test_rope_table_refuses():
    f = (ct.c_float * 64)()
    for args in ((f, 0, FAKE), (f, 1, None), (f, 1, FAKE + 4), (None, 1, FAKE), (f, (1 << 20) + 1, FAKE)):
        assert _lib.lib().bmx_k2b_rope_table(*args, None) != 0
        assert b"rope_table" in _lib.lib().bmx_last_error()
