"""The newer operators where the package calls them itself or registers them:
torch.library forms equal to the direct calls, and the packed cache's prefill
in a layer that slides."""
import pytest
import torch

from bmx_amd import k2b, ops, prefill
from bmx_amd.cache import PackedStreamingCache, PackedStreamingLayer, _is_window_mask
from bmx_amd.specs import spec_pair
from test_gpu_shared_decode import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def test_window_operator_equals_direct_call_and_compiles():
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = (torch.randn(n, t, 128, device=DEV, generator=g).half() for n, t in ((8, 70), (2, 900), (2, 900)))
    for n_q in (70, 1):
        x = q[:, :n_q]
        out = torch.ops.bmx.prefill_attention(x, k, v, SCALE, True, 0, 100, 4)
        assert torch.equal(out, prefill.attention(x, k, v, SCALE, causal=True, window=100, sinks=4))

    def layer(q):
        return torch.ops.bmx.prefill_attention(q * 1.0, k, v, SCALE, True, 0, 100, 4).float().sum(dim=0)

    assert torch.equal(torch.compile(layer, fullgraph=True, backend="aot_eager")(q), layer(q))
    torch.library.opcheck(torch.ops.bmx.prefill_attention.default, (q, k, v, SCALE, True, 0, 100, 4), {},
                          test_utils=("test_schema", "test_faketensor"))


def test_shared_decode_operator_equals_direct_call_and_compiles():
    x = Batch(3, 2, 4, 32, 512, [512, 640, 576], [4, 0, 9], torch.float16)
    args = (x.dq, x.pool, x.table, x.packed_len, x.max_len, x.shared, x.dbasis, x.rope.data)
    kw = dict(sm_scale=x.scale, rank=x.R, k_tail=x.dkt, v_tail=x.dvt, tail_len=x.tail_len, tail_cap=x.dkt.shape[2],
              **ops.consts_args(x.consts))
    assert torch.equal(torch.ops.bmx.k2b_decode_shared(*args, **kw), x.run())

    def layer(q):
        return torch.ops.bmx.k2b_decode_shared(q * 1.0, *args[1:], **kw).float().sum(dim=2)

    assert torch.equal(torch.compile(layer, fullgraph=True, backend="aot_eager")(x.dq), layer(x.dq))
    torch.library.opcheck(torch.ops.bmx.k2b_decode_shared.default, args, kw, test_utils=("test_schema", "test_faketensor"))


class _Config:
    num_attention_heads, num_key_value_heads, head_dim, hidden_size = 8, 2, 128, 1024
    num_hidden_layers, rope_theta, max_position_embeddings = 1, 10000.0, 4096
    rope_parameters = {"rope_type": "default", "rope_theta": 10000.0}
    rope_scaling = None


@pytest.mark.parametrize("window", [40, 300, 5000])
def test_cached_prefill_of_a_sliding_layer(window, monkeypatch):
    """The second block of a prompt in a layer that slides, with HF's mask: on
    the window kernel (no SDPA call), and equal to SDPA with that mask over the
    same dequantized rows."""
    h, G, n1, n2 = 2, 4, 400, 150
    lay = PackedStreamingLayer(*spec_pair("k2b_ph", rank=16), _Config(), recent_window=32)
    g = torch.Generator().manual_seed(1)
    k = torch.randn(h, n1 + n2, 128, generator=g).half().to(DEV)
    v = torch.randn(h, n1 + n2, 128, generator=g).half().to(DEV)
    for lo, hi in ((0, n1), (n1, n1 + n2)):
        lay.stash_pre_rope(k[:, lo:hi].transpose(0, 1).unsqueeze(0))
        lay.update(k[:, lo:hi].unsqueeze(0), v[:, lo:hi].unsqueeze(0))
    q = torch.randn(h * G, n2, 128, generator=g).half().to(DEV)
    gap = torch.arange(n2, device=DEV)[:, None] + n1 - torch.arange(n1 + n2, device=DEV)[None, :]
    mask = ((gap >= 0) & (gap < window))[None, None]
    assert _is_window_mask(mask, n2, n1 + n2, window)
    assert not _is_window_mask(mask, n2, n1 + n2, window - 1) or window > n1 + n2
    assert not _is_window_mask(mask, n2, n1 + n2, None)
    ref = lay.attend(q, SCALE, is_causal=True, attention_mask=mask)                     # no window known: SDPA
    calls = []
    sdpa = torch.nn.functional.scaled_dot_product_attention
    monkeypatch.setattr(torch.nn.functional, "scaled_dot_product_attention", lambda *a, **kw: calls.append(1) or sdpa(*a, **kw))
    out = lay.attend(q, SCALE, is_causal=True, attention_mask=mask, sliding_window=window)
    torch.cuda.synchronize()
    assert not calls
    torch.testing.assert_close(out.float(), ref.float(), atol=2e-3, rtol=2e-3)          # bmx_prefill's bounds against SDPA's
    other = mask.clone()
    other[0, 0, 3, 0] ^= True                                                           # another mask is not taken for it
    lay.attend(q, SCALE, is_causal=True, attention_mask=other, sliding_window=window)
    assert calls


def test_sliding_model_prefill_through_the_cache():
    """A tiny Qwen3 whose layers slide: a cached two-block prefill through the
    packed cache takes the window form in every layer (HF hands over the window
    and the mask), and its logits are those of the SDPA path."""
    from transformers import Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(0)
    cfg = Qwen3Config(vocab_size=128, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=2048, use_sliding_window=True,
                      sliding_window=100, max_window_layers=0, layer_types=["sliding_attention"] * 2)
    model = Qwen3ForCausalLM(cfg).to(DEV).half().eval()
    tokens = torch.randint(0, 128, (1, 500), generator=torch.Generator().manual_seed(1)).to(DEV)
    seen = []
    real = prefill.attention

    def run(use):
        cache = PackedStreamingCache(model.config, *spec_pair("k2b_ph", rank=16), recent_window=32)
        import bmx_amd.cache as C
        old = C._is_window_mask
        C._is_window_mask = old if use else (lambda *a: False)
        C.prefill.attention = lambda *a, **kw: seen.append(kw.get("window", 0)) or real(*a, **kw)
        try:
            with cache.attach(model), torch.no_grad():
                model(tokens[:, :300], past_key_values=cache, use_cache=True)
                return model(tokens[:, 300:], past_key_values=cache, use_cache=True).logits.float()
        finally:
            C._is_window_mask, C.prefill.attention = old, real
    a = run(True)
    assert seen.count(100) == 4, seen      # two layers, two blocks
    b = run(False)
    assert seen.count(100) == 4
    # fp16 layers (2 of attention and MLP, sums and norms, a head): some 20 roundings of 2^-11 on values of
    # up to 2, each of which may fall otherwise where the two attentions differ by less than their bounds
    torch.testing.assert_close(a, b, atol=20 * 2 ** -11 * 2, rtol=20 * 2 ** -11)
