"""Attention with a sliding window and sinks (prefill.attention with window /
sinks) against attention computed in 64 bits from each row's visible keys
alone, in both forms: row tiles on MFMA and few rows.

The bound of every element, with u = eps / 2 of the type, P the exact weights
and A = P |v|:
  * the output's rounding: u |out|;
  * each weight is rounded to 16 bits before it meets v: u A, and in fp16 the
    smallest ones are subnormal: with row tiles (weights below 2^-14 of the
    row's largest) up to 2^-25 a key and unit of v, where the sum of weights
    is at least 1; with few rows (below 2^-29) 2^15 times less;
  * a score is a sum of 128 products in fp32, off by at most 130 2^-24 of the
    sum of their sizes, d; a relative weight is off by 2 d and by the fp32
    exponential, sums and division (8 2^-23 allowed for): (2 d + 2^-20) A."""
import pytest
import torch

from bmx_amd import prefill

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SCALE = 128 ** -0.5
DTYPES = [torch.float16, torch.bfloat16]


def _inputs(h_kv, G, n_q, n_kv, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (1.5 * torch.randn(h_kv * G, n_q, 128, device=DEV, generator=g)).to(dtype)
    k = torch.randn(h_kv, n_kv, 128, device=DEV, generator=g).to(dtype)
    v = torch.randn(h_kv, n_kv, 128, device=DEV, generator=g).to(dtype)
    return q, k, v


def _seen(n_q, n_kv, window, sinks):
    p = torch.arange(n_q, device=DEV)[:, None] + (n_kv - n_q)
    j = torch.arange(n_kv, device=DEV)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks))


def _check(out, q, k, v, window, sinks):
    """Every element of out within its bound; hidden keys take no part in the
    reference (their values are zeroed per row where they are not finite)."""
    hq, n_q, _ = q.shape
    h_kv, n_kv, _ = k.shape
    G, few = hq // h_kv, n_q * (hq // h_kv) <= 16
    u = torch.finfo(q.dtype).eps / 2
    seen = _seen(n_q, n_kv, window, sinks)
    worst = 0.0
    for h in range(hq):
        qd, kd, vd = q[h].double(), k[h // G].double(), v[h // G].double()
        finite = torch.isfinite(kd).all(-1) & torch.isfinite(vd).all(-1)
        assert not (seen & ~finite[None, :]).any()
        kd, vd = torch.where(finite[:, None], kd, 0.0), torch.where(finite[:, None], vd, 0.0)
        s = (qd @ kd.t().contiguous() * SCALE).masked_fill(~seen, float("-inf"))
        d = 130 * 2.0 ** -24 * float((qd.abs() @ kd.abs().t().contiguous() * SCALE).masked_fill(~seen, 0.0).max())
        w = torch.softmax(s, -1)
        ref, A = w @ vd, w @ vd.abs()
        bound = u * ref.abs() + (2 * d + 2.0 ** -20) * A + 1e-30
        bound = bound + u * A
        if q.dtype == torch.float16:   # subnormal weights; outputs below 2^-14 are subnormal too
            bound = bound + 2.0 ** (-40 if few else -25) * seen.sum(-1)[:, None] * vd.abs().max() + 2.0 ** -25
        err = (out[h].double() - ref).abs()
        assert torch.isfinite(out[h].double()).all(), f"head {h}: not finite"
        worst = max(worst, float((err / bound).max()))
    assert worst <= 1.0, f"error {worst:.3f} times its bound"


CASES = [
    # h_kv, G, n_q, n_kv, window, sinks, n_split
    (2, 4, 300, 300, 64, 4, 0),        # square, a window of one tile
    (2, 4, 300, 300, 63, 0, 1),        # odd window, no sinks
    (1, 4, 700, 700, 100, 70, 3),      # sinks past one tile, splits
    (8, 4, 128, 5000, 1000, 4, 0),     # a chunk over a long context
    (1, 3, 50, 1290, 129, 130, 5),     # heads unevenly over the row tiles
    (1, 1, 64, 64, 1, 0, 0),           # a window of the query's own key
    (1, 2, 100, 333, 1, 1, 2),
    (2, 2, 200, 250, 100000, 5, 0),    # a window longer than the keys: none
    (2, 2, 200, 250, 249, 5, 0),
    (1, 8, 9, 40, 16, 300, 0),         # more sinks than keys
    (1, 17, 1, 1000, 200, 4, 16),      # one position, more rows than the few-row form takes
    (1, 16, 1, 1000, 200, 4, 16),
    (2, 4, 4, 6000, 700, 4, 0),
    (1, 5, 3, 400, 90, 33, 3),
    # few rows
    (8, 4, 1, 5000, 1024, 4, 0),
    (2, 7, 1, 700, 256, 1, 0),
    (1, 1, 1, 1, 1, 0, 0),
    (3, 8, 1, 33, 32, 0, 1),
    (1, 1, 8, 2000, 40, 7, 0),         # eight positions of one head
    (2, 2, 3, 999, 130, 64, 7),
    (1, 2, 4, 4, 2, 1, 0),
    (4, 1, 2, 70000, 66000, 4, 0),
    (1, 4, 1, 300, 100000, 2, 0),      # a window longer than the keys
    (1, 4, 2, 300, 50, 299, 0),        # sinks that reach the window
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_window_attention_matches_64_bits(case, dtype):
    h_kv, G, n_q, n_kv, window, sinks, n_split = case
    print(f"window case {case} {dtype}", flush=True)
    q, k, v = _inputs(h_kv, G, n_q, n_kv, dtype, seed=n_q * 7 + n_kv)
    out = prefill.attention(q, k, v, SCALE, causal=True, window=window, sinks=sinks, n_split=n_split)
    torch.cuda.synchronize()
    _check(out, q, k, v, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [
    # several blocks of 16 rows: h_kv, G, n_q, n_kv, window, sinks, n_split
    (2, 4, 5, 6000, 700, 4, 0), (1, 7, 9, 1000, 130, 20, 0), (2, 1, 33, 500, 40, 0, 1), (1, 1, 64, 64, 1, 0, 0),
    (3, 16, 4, 900, 300, 4, 5), (1, 64, 1, 4000, 2000, 1, 0), (1, 3, 21, 21, 8, 2, 16), (1, 5, 13, 300, 50, 4, 0),
    (2, 2, 32, 9000, 100000, 4, 0),
])
def test_blocks_of_rows_match_64_bits(case, dtype):
    h_kv, G, n_q, n_kv, window, sinks, n_split = case
    print(f"row blocks {case} {dtype}", flush=True)
    q, k, v = _inputs(h_kv, G, n_q, n_kv, dtype, seed=n_q * 5 + n_kv)
    out = prefill.attention(q, k, v, SCALE, causal=True, window=window, sinks=sinks, n_split=n_split)
    torch.cuda.synchronize()
    _check(out, q, k, v, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_hidden_infinity_stays_out_of_every_block_of_rows(dtype):
    """48 rows of one head over 3 blocks: a value that only the middle ones see."""
    n_q, n_kv, window = 48, 400, 16
    q, k, v = _inputs(1, 1, n_q, n_kv, dtype, seed=9)
    at = n_kv - n_q + 10
    clean = prefill.attention(q, k, v, SCALE, causal=True, window=window)
    v[0, at, 5] = float("-inf")
    out = prefill.attention(q, k, v, SCALE, causal=True, window=window)
    torch.cuda.synchronize()
    sees = _seen(n_q, n_kv, window, 0)[:, at]
    assert sees.sum() == window
    assert torch.equal(out[0, ~sees], clean[0, ~sees])
    assert not torch.isfinite(out[0, sees][:, 5]).any() and torch.isfinite(out[0, sees][:, 6:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_q,G", [(150, 4), (1, 4), (3, 2)])
def test_strided_operands_and_peaked_scores(n_q, G, dtype):
    """q as a projection's transposed view, K/V rows inside a longer buffer
    with NaN behind them, keys scaled so that few of them weigh."""
    h_kv, n_kv, window, sinks = 2, 1500, 333, 4
    g = torch.Generator(device=DEV).manual_seed(11)
    q = torch.randn(n_q, h_kv * G, 128, device=DEV, generator=g).to(dtype).transpose(0, 1)
    kb = (6.0 * torch.randn(n_kv + 40, h_kv, 136, device=DEV, generator=g)).to(dtype)
    vb = torch.randn(n_kv + 40, h_kv, 136, device=DEV, generator=g).to(dtype)
    kb[n_kv:], vb[n_kv:] = float("nan"), float("nan")
    k, v = kb[:n_kv, :, :128].transpose(0, 1), vb[:n_kv, :, :128].transpose(0, 1)
    out = prefill.attention(q, k, v, SCALE, causal=True, window=window, sinks=sinks)
    torch.cuda.synchronize()
    _check(out, q, k, v, window, sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_q,G,n_split", [(40, 4, 1), (40, 4, 3), (300, 1, 0), (1, 4, 0), (4, 2, 2)])
def test_rows_no_query_sees_may_hold_anything(n_q, G, n_split, dtype):
    """Infinities and NaN in the keys and values between the sinks and the
    first window, which share tiles with both."""
    n_kv, window, sinks = 900, 200, 5
    q, k, v = _inputs(2, G, n_q, n_kv, dtype, seed=3)
    hole = slice(sinks, n_kv - n_q - window + 1)
    clean = prefill.attention(q, k, v, SCALE, causal=True, window=window, sinks=sinks, n_split=n_split)
    for kx, vx in ((float("nan"), float("nan")), (float("inf"), float("-inf"))):
        k[:, hole], v[:, hole] = kx, vx
        out = prefill.attention(q, k, v, SCALE, causal=True, window=window, sinks=sinks, n_split=n_split)
        torch.cuda.synchronize()
        _check(out, q, k, v, window, sinks)
        torch.testing.assert_close(out, clean, atol=2e-2, rtol=2e-2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,n_q", [(1, 200), (2, 4)])
def test_infinite_value_reaches_only_the_rows_that_see_it(G, n_q, dtype):
    """A key that left the window of later rows holds an infinite value: those
    rows are finite and right, the rows that see it are not finite."""
    n_kv, window = n_q + 300, 60
    q, k, v = _inputs(1, G, n_q, n_kv, dtype, seed=5)
    at = n_kv - n_q - window + 1 + n_q // 2      # seen by the first half of the rows
    v[0, at, 3] = float("inf")
    out = prefill.attention(q, k, v, SCALE, causal=True, window=window)
    torch.cuda.synchronize()
    sees = _seen(n_q, n_kv, window, 0)[:, at]
    assert sees.any() and not sees.all()
    assert not torch.isfinite(out[:, sees][..., 3]).any()
    assert torch.isfinite(out[:, ~sees]).all() and torch.isfinite(out[:, sees][..., 4:]).all()
    v2 = v.clone()
    v2[0, at] = 0
    for h in range(G):
        rows = ~sees
        s = (q[h].double() @ k[0].double().t().contiguous() * SCALE).masked_fill(~_seen(n_q, n_kv, window, 0), float("-inf"))
        ref = torch.softmax(s, -1) @ v2[0].double()
        u = torch.finfo(dtype).eps / 2   # the output's rounding, and the weights' (4 sizes of v bound |v| here)
        assert ((out[h][rows].double() - ref[rows]).abs() <= u * (ref[rows].abs() + 5.0) + 1e-4).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [500, 100000])
@pytest.mark.parametrize("G,n_q", [(2, 200), (2, 4)])
def test_window_as_long_as_the_keys_keeps_hidden_values_out(G, n_q, window, dtype):
    """Nothing but the causal mask hides a key: a NaN value reaches the rows from
    its own on, and the rows before are those of the call without it."""
    n_kv = 500
    q, k, v = _inputs(1, G, n_q, n_kv, dtype, seed=8)
    clean = prefill.attention(q, k, v, SCALE, causal=True, window=window)
    row = n_q // 2
    v[0, n_kv - n_q + row, 77] = float("nan")
    out = prefill.attention(q, k, v, SCALE, causal=True, window=window)
    torch.cuda.synchronize()
    assert torch.equal(out[:, :row], clean[:, :row])
    assert torch.isnan(out[:, row:, 77]).all()
    assert torch.isfinite(out[:, row:, :77]).all() and torch.isfinite(out[:, row:, 78:]).all()


def test_repeated_calls_are_equal_bit_for_bit():
    for n_q in (1, 64):
        q, k, v = _inputs(4, 4, n_q, 3000, torch.float16, seed=9)
        outs = [prefill.attention(q, k, v, SCALE, causal=True, window=500, sinks=4) for _ in range(3)]
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_two_streams_and_a_replayed_graph():
    """Calls in flight on two streams, and a captured one replayed between
    eager work, give what the eager call gives."""
    for n_q in (1, 64):
        q, k, v = _inputs(4, 4, n_q, 6000, torch.bfloat16, seed=13)
        q2 = (q.float() * 0.5).bfloat16()
        kw = dict(causal=True, window=2000, sinks=4)
        ref, ref2 = prefill.attention(q, k, v, SCALE, **kw), prefill.attention(q2, k, v, SCALE, **kw)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(5):
            with torch.cuda.stream(side):
                b = prefill.attention(q2, k, v, SCALE, **kw)
            a = prefill.attention(q, k, v, SCALE, **kw)
            torch.cuda.synchronize()
            assert torch.equal(a, ref) and torch.equal(b, ref2)
        g = torch.cuda.CUDAGraph()
        x = q.clone()
        with torch.cuda.graph(g):
            y = prefill.attention(x, k, v, SCALE, **kw)
        for src, want in ((q, ref), (q2, ref2), (q, ref)):
            x.copy_(src)
            g.replay()
            prefill.attention(q2, k, v, SCALE, **kw)
            torch.cuda.synchronize()
            assert torch.equal(y, want)
