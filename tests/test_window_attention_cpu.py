"""The refusals of the windowed attention: the C entry's and the wrapper's
checks, without a GPU (no call gets past them)."""
import ctypes as ct

import pytest
import torch

from bmx_amd import _lib, prefill


def _args(**kw):
    a = _lib.PrefillArgs()
    a.q = a.k = a.v = a.out = 1 << 20   # never dereferenced: every call fails its checks
    a.q_stride_h, a.q_stride_t, a.kv_stride_h, a.kv_stride_t = 128, 128, 128 * 64, 128
    a.h_kv, a.n_q_groups, a.n_q, a.n_kv, a.head_dim = 1, 4, 1, 64, 128
    a.causal, a.sm_scale = 1, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(window=-1), "window"), (dict(sinks=-1, window=8), "sinks"), (dict(sinks=4), "sinks need a window"),
    (dict(window=8, causal=0), "needs causal"), (dict(window=8, n_q=65), "n_q <= n_kv"),
    (dict(window=8, head_dim=64), "head_dim"), (dict(window=8, kv_stride_t=132), "strides"),
])
def test_c_entry_refuses(kw, word):
    a = _args(**kw)
    assert _lib.lib().bmx_prefill(ct.byref(a), None) != 0
    assert word in _lib.lib().bmx_last_error().decode()
    assert _lib.lib().bmx_prefill_workspace_bytes(ct.byref(a)) == 0


@pytest.mark.parametrize("splits", [2, 5, 16])
def test_a_workspace_that_is_missing_or_small_is_refused(splits):
    for n_q in (1, 32):
        a = _args(window=8, sinks=2, n_q=n_q, n_split=splits)
        need = _lib.lib().bmx_prefill_workspace_bytes(ct.byref(a))
        assert need == 4 * n_q * splits * (132 if n_q == 1 else 130) * 4   # fp32 sums, maximum, sum of a row
        a.workspace, a.workspace_bytes = 1 << 20, need - 1
        assert _lib.lib().bmx_prefill(ct.byref(a), None) != 0
        assert "workspace" in _lib.lib().bmx_last_error().decode()


def test_wrapper_refuses_cpu_tensors_and_bad_arguments():
    q, k = torch.zeros(4, 1, 128, dtype=torch.float16), torch.zeros(1, 8, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="HIP device"):
        prefill.attention(q, k, k, 0.1, causal=True, window=4)


@pytest.mark.parametrize("n_q", [1, 32])
def test_an_unaligned_workspace_is_refused_under_a_window(n_q):
    a = _args(window=8, sinks=2, n_q=n_q, n_split=2)
    a.workspace, a.workspace_bytes = (1 << 20) + 8, 1 << 20
    assert _lib.lib().bmx_prefill(ct.byref(a), None) != 0
    assert "16-byte" in _lib.lib().bmx_last_error().decode()
