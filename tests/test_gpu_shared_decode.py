"""Shared-prefix decode (k2b.decode_shared) against attention in 64 bits over
keys and values rebuilt from the codes the pages were packed of.

The bound of an element, with P the exact weights, V the values, u = eps / 2
of the output's type and h = 2^-11 (fp16's):
  * the output's rounding, u |out|, and in fp16 half a step of its subnormals, 2^-25;
  * a packed token's weight times norm is rounded to fp16, a window row's
    weight to the output's type: h P |V| over packed tokens, u P |V| over window rows;
  * a packed key has two roundings of its own size, its value and the rotation
    it was turned by (each of cos and sin), evenly spread within h: a score's
    error has a standard deviation of
    sd = scale h / sqrt(3) |q (k, k_pre, k_pre')| (k_pre' the pair's other half),
    independent over tokens, and an output's 6 deviations are
    6 |P sd (V - out)|_2;
  * fp32 sums (2^-18 P |V|) and 2^-24 of the largest value where 16-bit weights are
    subnormal."""
import pytest
import torch

from bmx_amd import k2b
from oracle import layout as OL

pytestmark = pytest.mark.gpu

DEV = "cuda"
D = 128
CONSTS = k2b.CodecConsts.make(theta=10000.0)
LEVELS = torch.tensor(CONSTS.codebook, dtype=torch.float64)
SIGNS = torch.tensor([-1.0 if (CONSTS.sign_bits[c // 32] >> (c % 32)) & 1 else 1.0 for c in range(D)], dtype=torch.float64)


def _hadamard():
    H = torch.ones(1, 1, dtype=torch.float64)
    while H.shape[0] < D:
        H = torch.cat([torch.cat([H, H], 1), torch.cat([H, -H], 1)], 0)
    return H


def _codes(g, h, T, R, norm=1.0):
    f = dict(us=(torch.randn(T, R, generator=g)).half(), res=torch.randint(-4, 4, (h * D, T), generator=g),
             scale=(0.1 + 0.2 * torch.rand(h * D, T // 64, generator=g)).half(),
             vidx=torch.randint(0, 4, (T, h * D), generator=g),
             vnorm=(norm * (5 + 10 * torch.rand(T, h, generator=g))).half())
    return f


def _pages(f, h, R):
    return torch.from_numpy(OL.pack_pages(f["us"].numpy(), f["res"].numpy(), f["scale"].numpy(), f["vidx"].numpy(),
                                          f["vnorm"].numpy(), h, R))


def _rows(f, basis, consts, pos0):
    """(keys, pre-rotation keys, values), each (h, T, D) in 64 bits."""
    T = f["us"].shape[0]
    h = f["vnorm"].shape[1]
    k = f["us"].double() @ basis.double().t()
    k = k + (f["res"].double() * f["scale"].double().repeat_interleave(64, 1)).t()
    k = k.view(T, h, D).transpose(0, 1)
    ang = (torch.arange(pos0, pos0 + T, dtype=torch.float32)[:, None] * torch.tensor(consts.inv_freq)[None, :]).double()
    cos, sin = ang.cos() * consts.rope_scaling, ang.sin() * consts.rope_scaling
    a, b = k[..., :64], k[..., 64:]
    kr = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    lv = LEVELS[f["vidx"]].view(T, h, D).transpose(0, 1)
    v = (lv @ _hadamard()) * SIGNS / D * f["vnorm"].double().t()[..., None]
    return kr, k * consts.rope_scaling, v


class Batch:
    """A batch behind a common prefix, with its pages scattered over a pool."""

    def __init__(self, B, h, G, R, shared, lens, tails, dtype, seed=0, consts=CONSTS, edit=None, qscale=1.5):
        g = torch.Generator().manual_seed(seed)
        self.B, self.h, self.G, self.R, self.shared, self.dtype, self.consts = B, h, G, R, shared, dtype, consts
        self.lens, self.tails = lens, tails
        self.prefix = _codes(g, h, shared, R) if shared else None
        self.owns = [_codes(g, h, -(-(n - shared) // 64) * 64, R) if n > shared else None for n in lens]
        if edit:
            edit(self)
        self.basis = torch.linalg.qr(torch.randn(h * D, R, generator=g).double())[0].half().contiguous()
        self.q = (qscale * torch.randn(B, h, G, D, generator=g)).to(dtype)
        cap = max(max(tails), 1)
        self.k_tail = (0.7 * torch.randn(B, h, cap, D, generator=g)).to(dtype)
        self.v_tail = torch.randn(B, h, cap, D, generator=g).to(dtype)
        runs = ([_pages(self.prefix, h, R)] if shared else []) + [_pages(o, h, R) for o in self.owns if o is not None]
        pages = torch.cat(runs) if runs else torch.zeros(1, OL.page_bytes(h, R), dtype=torch.uint8)
        n = pages.shape[0]
        ids = torch.randperm(n + 3, generator=g)[:n]
        pool = torch.zeros(n + 3, pages.shape[1], dtype=torch.uint8)
        pool[ids] = pages
        self.max_len = -(-max(max(lens), shared) // 128) * 128
        width = self.max_len // 16 + 2
        # entries past a row's tokens, and the other rows' shared entries, are never read: anything
        table = torch.randint(-2**31, 2**31 - 1, (B, width), generator=g).to(torch.int32)
        sp = shared // 16
        table[0, :sp] = ids[:sp].int()
        at = sp
        for b, o in enumerate(self.owns):
            if o is not None:
                m = o["us"].shape[0] // 16
                table[b, sp:sp + m] = ids[at:at + m].int()
                at += m
        self.pool, self.table = pool.to(DEV), table.to(DEV)
        self.packed_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.tail_len = torch.tensor(tails, dtype=torch.int32, device=DEV)
        self.rope = k2b.rope_table(consts, max(self.max_len, 1), DEV)
        self.scale = D ** -0.5
        self.dq, self.dkt, self.dvt = self.q.to(DEV), self.k_tail.to(DEV), self.v_tail.to(DEV)
        self.dbasis = self.basis.to(DEV)

    def run(self, **kw):
        a = dict(rank=self.R, rope=self.rope, k_tail=self.dkt, v_tail=self.dvt, tail_len=self.tail_len,
                 tail_cap=self.dkt.shape[2])
        a.update(kw)
        q = a.pop("q", self.dq)
        return k2b.decode_shared(q, self.pool, self.table, self.packed_len, self.max_len, self.shared, self.dbasis,
                                 self.consts, self.scale, **a)

    def reference(self):
        """(out, bound) in 64 bits."""
        u, hh = torch.finfo(self.dtype).eps / 2, 2.0 ** -11
        out = torch.zeros(self.B, self.h, self.G, D, dtype=torch.float64)
        bound = out.clone()
        pre = _rows(self.prefix, self.basis, self.consts, 0) if self.shared else None
        for b in range(self.B):
            n = self.lens[b] // 64 * 64
            parts = []
            if min(n, self.shared):
                parts.append([x[:, :min(n, self.shared)] for x in pre])
            if n > self.shared:
                parts.append([x[:, :n - self.shared] for x in _rows(self.owns[b], self.basis, self.consts, self.shared)])
            k, kp, v = [torch.cat([p[i] for p in parts], 1) if parts else torch.zeros(self.h, 0, D, dtype=torch.float64)
                        for i in range(3)]
            t = self.tails[b]
            kw, vw = self.k_tail[b, :, :t].double(), self.v_tail[b, :, :t].double()
            q = self.q[b].double()
            n = k.shape[1]
            if n + t == 0:
                continue
            P = torch.softmax(torch.cat([q @ k.transpose(1, 2), q @ kw.transpose(1, 2)], -1) * self.scale, -1)
            V = torch.cat([v, vw], 1)
            o = P @ V
            kq = torch.cat([kp[..., 64:], kp[..., :64]], -1)
            sd = self.scale * hh / 3 ** 0.5 * (q.square() @ (k.square() + kp.square() + kq.square()).transpose(1, 2)).sqrt()
            w = (P[..., :n] * sd).square()
            var = w @ v.square() - 2 * o * (w @ v) + o.square() * w.sum(-1, keepdim=True)
            A, Aw = P[..., :n] @ v.abs(), P[..., n:] @ vw.abs()
            big = V.abs().amax((1, 2))[:, None, None]
            out[b] = o
            bound[b] = u * o.abs() + hh * A + u * Aw + 6 * var.clamp(min=0).sqrt() + 2.0 ** -18 * (A + Aw) + 2.0 ** -24 * big
        if self.dtype == torch.float16:
            bound = torch.where(bound > 0, bound + 2.0 ** -25, bound)   # an empty sequence's zeros are exact
        return out, bound

    def check(self, out):
        ref, bound = self.reference()
        err = (out.double().cpu() - ref).abs()
        assert torch.isfinite(out).all()
        worst = (err / (bound + 1e-300)).max().item()
        print(f"error {worst:.3f} of its bound, largest {err.max().item():.2e}", flush=True)
        assert ((err <= bound) | (err == 0)).all(), worst


CASES = [
    # B, h_kv, G, rank, shared, lens, tails
    (2, 8, 4, 32, 512, [512, 512], [7, 33]),                       # nothing but the prefix and a window
    (1, 1, 1, 16, 128, [128], [0]),                                # one row
    (4, 4, 4, 32, 384, [384, 512, 640, 1024], [0, 1, 64, 65]),     # 16 rows, ragged
    (5, 2, 7, 16, 640, [640, 704, 768, 1000, 640], [3, 0, 5, 9, 200]),   # 35 rows; 1000 tokens are 15 groups
    (17, 1, 4, 32, 256, [256] * 16 + [512], [1] * 17),             # 68 rows: a block of 4
    (33, 3, 1, 16, 128, [128 + 64 * (i % 5) for i in range(33)], [i for i in range(33)]),   # h_kv 3: scales over lanes' pages
    (9, 16, 16, 32, 128, [128] * 9, [2] * 9),                      # 144 rows, 16 heads
    (3, 5, 16, 16, 1152, [1152, 1280, 1152], [0, 0, 0]),           # no window
    (4, 8, 4, 32, 1024, [1024, 512, 64, 0], [5, 6, 7, 8]),         # sequences shorter than the prefix
    (4, 2, 4, 32, 1024, [0, 1024, 0, 960], [0, 3, 4, 0]),          # an idle slot, and one with a window alone
    (3, 2, 4, 32, 0, [256, 0, 640], [4, 5, 0]),                    # no prefix
    (2, 4, 4, 32, 0, [0, 0], [40, 0]),                             # windows alone
    (2, 2, 2, 16, 4096, [4096, 8192], [255, 1]),                   # own part longer than the prefix
    (6, 6, 3, 32, 2048, [2048 + 128 * i for i in range(6)], [31] * 6),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_matches_64_bits(case, dtype):
    print(f"shared case {case} {dtype}", flush=True)
    x = Batch(*case, dtype)
    out = x.run()
    torch.cuda.synchronize()
    x.check(out)


def test_rope_scaling_and_host_window_length():
    c = k2b.CodecConsts(CONSTS.codebook, CONSTS.sign_bits, CONSTS.inv_freq, 1.25)
    x = Batch(3, 2, 4, 32, 512, [512, 640, 576], [20, 20, 20], torch.float16, consts=c)
    x.check(x.run(tail_len=20))


def test_strided_window_and_rows_past_its_length():
    """The window as a view of a longer buffer in another order, NaN and
    infinities behind every sequence's rows."""
    x = Batch(3, 2, 4, 16, 256, [256, 384, 256], [9, 0, 70], torch.bfloat16, seed=4)
    big_k = torch.full((x.h, 90, x.B, D + 8), float("nan"), dtype=torch.bfloat16, device=DEV)
    big_v = torch.full_like(big_k, float("inf"))
    for b, t in enumerate(x.tails):
        big_k[:, :t, b, :D] = x.dkt[b, :, :t]
        big_v[:, :t, b, :D] = x.dvt[b, :, :t]
    x.check(x.run(k_tail=big_k[..., :D].permute(2, 0, 1, 3), v_tail=big_v[..., :D].permute(2, 0, 1, 3), tail_cap=80))
    assert torch.isnan(big_k[:, 9:, 0]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm,sink_norm,gap", [
    (1e-4, 1e-4, 0), (1.0, 1.0, 12), (1.0, 1e-4, 12), (1.0, 0.0, 25), (1e-3, 0.0, 90), (1e-3, 200.0, -12), (1.0, 0.0, 250),
])
def test_small_norms_and_sinks(norm, sink_norm, gap, dtype):
    """Values of small norm, and a first token whose score stands `gap` nats
    above (below) the others with a norm of its own, in the prefix and in a
    sequence's own part: the other tokens keep their bits."""
    B, h, G, R = 2, 2, 4, 32
    x = None

    def edit(b):
        for f in [b.prefix, b.owns[1]]:
            f["vnorm"] = (f["vnorm"].float() * norm).half()
            f["us"] = (f["us"].float() * 0.02).half()
            f["scale"] = (f["scale"].float() * 0.05).half()
            f["vnorm"][0] = sink_norm
    c = k2b.CodecConsts(CONSTS.codebook, CONSTS.sign_bits, (0.0,) * 64, 1.0)   # no rotation: the gap is one score
    x = Batch(B, h, G, R, 1024, [1024, 1536], [0, 0], dtype, consts=c, edit=edit, qscale=1.0)
    # the first token's key along every query: |gap| in nats
    for f, page in ((x.prefix, 0), (x.owns[1], 64)):
        target = torch.zeros(h * D, dtype=torch.float64)
        for hh in range(h):
            qm = x.q[:, hh].double().reshape(-1, D)
            want = torch.full((qm.shape[0],), float(gap), dtype=torch.float64) / x.scale
            target[hh * D:(hh + 1) * D] = torch.linalg.pinv(qm) @ want
        coef = torch.linalg.pinv(x.basis.double()) @ target
        f["us"][0] = coef.clamp(-6e4, 6e4).half()
    sp = x.shared // 16
    x.pool[x.table[0, 0].long()] = _pages({k: (v[:64] if k in ("us", "vidx", "vnorm") else v[:, :64] if k == "res" else v[:, :1])
                                           for k, v in x.prefix.items()}, h, R)[0].to(DEV)
    x.pool[x.table[1, sp].long()] = _pages({k: (v[:64] if k in ("us", "vidx", "vnorm") else v[:, :64] if k == "res" else v[:, :1])
                                            for k, v in x.owns[1].items()}, h, R)[0].to(DEV)
    out = x.run(k_tail=None, v_tail=None, tail_len=None, tail_cap=0)
    torch.cuda.synchronize()
    x.check(out)


def test_codes_past_a_sequences_length_may_hold_anything():
    """Norms, scales and coefficients that are not finite in groups that a
    shorter sequence does not see leave it as it was."""
    x = Batch(3, 2, 4, 32, 1024, [512, 448, 64], [3, 3, 3], torch.float16, seed=9)
    clean = x.run()
    f = x.prefix
    f["vnorm"][512:], f["us"][512:] = float("nan"), float("inf")
    f["scale"][:, 8:] = float("nan")
    x.pool[x.table[0, :64].long()] = _pages(f, x.h, x.R).to(DEV)
    out = x.run()
    torch.cuda.synchronize()
    assert torch.equal(out, clean)


def test_queries_of_very_different_sizes():
    """bf16 rows of one batch 2^20 apart, one of them zero: each row as exact as
    it would be alone."""
    x = Batch(4, 1, 4, 32, 512, [512] * 4, [5] * 4, torch.bfloat16, seed=2, qscale=2.0)
    x.q[1] *= 2.0 ** -20
    x.q[2] = 0
    x.q[3] *= 2.0 ** -6
    x.dq = x.q.to(DEV)
    x.check(x.run())


def test_equals_decode_over_the_same_tables():
    """The unshared decode of the same batch, within the two kernels' roundings
    (its tests' 2e-3 and rel 1e-2)."""
    x = Batch(6, 8, 4, 32, 1024, [1024 + 128 * i for i in range(6)], [10 + i for i in range(6)], torch.float16, seed=6)
    x.table[:, :64] = x.table[0, :64]
    n = x.max_len // 16
    tab = x.table[:, :n].clamp(0, x.pool.shape[0] - 1).contiguous()
    ref = k2b.decode(x.dq, x.pool, tab, x.packed_len, x.max_len, x.dbasis, x.consts, x.scale, rank=x.R, k_tail=x.dkt,
                     v_tail=x.dvt, tail_len=x.tail_len, tail_cap=x.dkt.shape[2])
    out = x.run()
    torch.cuda.synchronize()
    torch.testing.assert_close(out.float(), ref.float(), atol=2e-3, rtol=1e-2)


def test_repeated_calls_streams_and_graphs():
    """Equal bit for bit: repeated calls, calls in flight on two streams, and a
    captured call replayed between eager work, with lengths changed between."""
    x = Batch(5, 2, 4, 16, 512, [512, 640, 768, 1024, 512], [4, 0, 30, 9, 1], torch.float16, seed=8)
    q2 = (x.dq.float() * 0.5).half()
    ref, ref2 = x.run(), x.run(q=q2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(side):
            b = x.run(q=q2)
        a = x.run()
        torch.cuda.synchronize()
        assert torch.equal(a, ref) and torch.equal(b, ref2)
    g = torch.cuda.CUDAGraph()
    q = x.dq.clone()
    with torch.cuda.graph(g):
        y = x.run(q=q)
    short = torch.tensor([512, 0, 64, 512, 128], dtype=torch.int32, device=DEV)
    full = x.packed_len.clone()
    for lens, src in ((full, x.dq), (short, q2), (full, q2), (short, x.dq)):
        x.packed_len.copy_(lens)
        q.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        want = x.run(q=src)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_output_is_written_where_asked():
    x = Batch(2, 2, 4, 32, 256, [256, 256], [2, 2], torch.float16)
    out = torch.full((4, 2, 4, D), 7.0, dtype=torch.float16, device=DEV)
    ret = x.run(out=out[1:3])
    torch.cuda.synchronize()
    assert ret.data_ptr() == out[1:3].data_ptr()
    x.check(out[1:3])
    assert (out[0] == 7).all() and (out[3] == 7).all()


@pytest.mark.parametrize("kw,word", [
    (dict(rank=16), "page_bytes"), (dict(tail_cap=9), "tail"), (dict(tail_len=5), "tail_len"),
    (dict(q="f32"), "fp16 or bf16"), (dict(k_tail="bf16"), "q's dtype"), (dict(rope="short"), "fewer positions"),
    (dict(rope="freq"), "other frequencies"), (dict(out="shape"), "out must"),
])
def test_refusals(kw, word):
    x = Batch(2, 2, 4, 32, 256, [256, 256], [2, 2], torch.float16)
    kw = dict(kw)
    if kw.get("q") == "f32":
        kw["q"] = x.dq.float()
    if kw.get("k_tail") == "bf16":
        kw.update(k_tail=x.dkt.bfloat16(), v_tail=x.dvt.bfloat16())
    if kw.get("rope") == "short":
        kw["rope"] = k2b.rope_table(CONSTS, 128, DEV)
    if kw.get("rope") == "freq":
        kw["rope"] = k2b.rope_table(k2b.CodecConsts.make(theta=5e5), 512, DEV)
    if kw.get("out") == "shape":
        kw["out"] = torch.empty(2, 2, 4, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match=word):
        x.run(**kw)
