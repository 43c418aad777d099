"""Operators of a batch that serves many continuations from the packed cache, and of models whose attention slides.

* shared-prefix decode: one token's attention of a batch of sequences over packed k2b pages, where the pages of a
  long common prefix (a system prompt, a document, the prompt of several samples) are read and rebuilt once for all
  sequences, each sequence's own pages and recent window beside them;
* page tables: rows of a batch forked, reordered and dropped by index, pages freed when no row holds them, new pages
  handed out (`update`); and the pool closed up after that, pages moved and tables rewritten (`compact`);
* attention with a sliding window and a few first tokens that stay visible, over dense K/V rows: a prompt, a chunk of
  a prompt, a single token.

With `own` false, `run` computes them from elementary torch operations in 32 bits; with `own` true it calls
bmx_amd's operators.  `exact` computes them in 64 bits, the packed pages from the codes they were built of.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
LEVELS = (-1.5194618701934814, -0.46033763885498047, 0.44421979784965515, 1.5017313957214355)  # 2-bit Lloyd levels
PT = 16    # tokens of a page
D = 128    # head_dim


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # sixteen answers to one 64k document: the cache's headline context and an 8B model's heads, ragged own parts
        dict(name="shared_decode_64k_b16", kind="shared", batch=16, h_kv=8, G=4, shared=65408, own=1024, window=128,
             rank=32, dtype="fp16", theta=500000.0, idle=False),
        # a chat server's batch behind an 8k system prompt and tools, bf16 model, one slot of the batch not in use
        dict(name="shared_decode_8k_b32", kind="shared", batch=32, h_kv=8, G=4, shared=8192, own=512, window=161,
             rank=16, dtype="bf16", theta=1000000.0, idle=True),
        # four samples of a short prompt just after it: all latency; an odd group of query heads
        dict(name="shared_decode_short", kind="shared", batch=4, h_kv=4, G=7, shared=512, own=0, window=60, rank=32,
             dtype="fp16", theta=500000.0, idle=False),
        # a prompt's own attention in a sliding layer
        dict(name="window_prefill_8k", kind="window", h_kv=8, G=4, queries=8192, keys=8192, window=1024, sinks=4,
             dtype="fp16"),
        # a chunk of a long prompt over everything before it, odd sizes
        dict(name="window_prefill_chunk", kind="window", h_kv=8, G=4, queries=509, keys=33001, window=4096, sinks=4,
             dtype="bf16"),
        # one token far into a stream that keeps its first tokens
        dict(name="window_decode_64k", kind="window", h_kv=8, G=4, queries=1, keys=65536, window=4096, sinks=4,
             dtype="bf16"),
        # one token of a model with few heads and a small window
        dict(name="window_decode_short", kind="window", h_kv=2, G=7, queries=1, keys=700, window=256, sinks=1,
             dtype="fp16"),
        # a beam search step: eight beams of 8k tokens reordered, the dropped beams' pages freed, a codec page each
        dict(name="pages_update_beams", kind="update", rows=8, new_rows=8, pages=512, cap=640, pool=8192, shared=480,
             grow=8, drop=0),
        # a large server's step: sequences finished and forked, tables of up to 64k tokens
        dict(name="pages_update_server", kind="update", rows=64, new_rows=64, pages=4088, cap=4096, pool=262144,
             shared=1024, grow=8, drop=7),
        # a small pool of a few layers, a quarter of it live
        dict(name="pages_compact_small", kind="compact", rows=8, pages=32, cap=64, pool=1024, shared=8, layers=4,
             h_kv=8, rank=16),
        # the pools of sixteen layers after a burst of requests, half of the pages live
        dict(name="pages_compact_large", kind="compact", rows=16, pages=160, cap=256, pool=4096, shared=32, layers=16,
             h_kv=8, rank=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "window", "window", "window", "update", "compact"])
    h_kv, G, dtype = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 3, 4, 4, 7, 8]), rng.choice(["fp16", "bf16"])
    if kind == "shared":
        batch = _log_int(rng, 1, 40)
        top = max(1, min(511, 511 * 64 // max(64, batch * G)))
        return dict(kind=kind, batch=batch, h_kv=h_kv, G=G, shared=128 * _log_int(rng, 1, top),
                    own=128 * rng.randint(0, 8), window=rng.randint(0, 255), rank=rng.choice([16, 32]), dtype=dtype,
                    theta=rng.choice([10000.0, 500000.0, 1000000.0]), idle=rng.random() < 0.3)
    if kind == "window":
        form = rng.choice(["token", "few", "chunk", "prompt"])
        if form == "token":
            queries, keys = 1, _log_int(rng, 1, 131072)
        elif form == "few":
            queries = rng.randint(2, 9)
            keys = queries + _log_int(rng, 1, 65536) - 1
        elif form == "chunk":
            queries = _log_int(rng, 2, 1024)
            keys = queries + _log_int(rng, 1, 32768) - 1
        else:
            queries = keys = _log_int(rng, 2, 8192)
        return dict(kind=kind, h_kv=h_kv, G=rng.choice([1, 2, 4, 4, 7]), queries=queries, keys=keys,
                    window=_log_int(rng, 1, 1024 if form == "prompt" else 8192), sinks=rng.choice([0, 1, 4, 4, 5, 64, 130]),
                    dtype=dtype)
    rows = _log_int(rng, 1, 64)
    if kind == "update":
        pages = _log_int(rng, 1, 4096)
        return dict(kind=kind, rows=rows, new_rows=_log_int(rng, 1, 64), pages=pages, cap=pages + rng.randint(0, 40),
                    pool=rows * pages + rng.randint(1, 4096), shared=rng.randint(0, pages), grow=rng.choice([0, 1, 8, 16]),
                    drop=rng.randint(0, rows))
    pages = _log_int(rng, 1, max(2, 2048 // rows))
    return dict(kind="compact", rows=rows, pages=pages, cap=pages + rng.randint(0, 40),
                pool=rows * pages + rng.randint(1, 2048), shared=rng.randint(0, pages), layers=rng.randint(1, 12),
                h_kv=h_kv, rank=rng.choice([16, 32]))


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _inv_freq(theta):
    return 1.0 / (theta ** (torch.arange(0, D, 2, dtype=torch.int64).to(torch.float) / D))


def _signs(n, seed=0):
    """The +-1 signs of the seeded randomized Hadamard."""
    return torch.randint(0, 2, (n,), generator=torch.Generator().manual_seed(seed)) * 2 - 1


def _sign_words():
    words = [0] * 4
    for c, s in enumerate(_signs(D).tolist()):
        words[c // 32] |= (1 << (c % 32)) if s < 0 else 0
    return tuple(words)


def _hadamard(dtype):
    """Sylvester's Hadamard matrix of D points, entries +-1."""
    i = torch.arange(D, device="cuda")
    x = i[:, None] & i[None, :]
    for s in (4, 2, 1):
        x = x ^ (x >> s)
    return (1 - 2 * (x & 1)).to(dtype)


def _fields(g, h, T, R):
    """Codes of T tokens in the distributions the codec makes: low-rank coefficients, 3-bit key residual and scales,
    2-bit value codes and norms."""
    s = torch.arange(1, R + 1, device="cuda", dtype=torch.float32) ** -0.35
    us = (_randn(g, T, R) * (s * math.sqrt(h * D / 2 / float((s * s).sum())))).half()
    res = (_randn(g, h, T, D) / 0.8).round().clamp(-4, 3).to(torch.int32)
    scale = (0.24 * (0.8 + 0.4 * torch.rand(h, T // 64, D, generator=g, device="cuda"))).half()
    mids = torch.tensor([(a + b) / 2 for a, b in zip(LEVELS, LEVELS[1:])], device="cuda")
    vidx = torch.bucketize(_randn(g, h, T, D), mids).to(torch.int32)
    vnorm = (math.sqrt(D) * (0.7 + 0.6 * torch.rand(h, T, generator=g, device="cuda"))).half()
    return dict(us=us, res=res, scale=scale, vidx=vidx, vnorm=vnorm)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _pages(f):
    """The recipe's 16-token pages (include/bmx_k2b.h) of a token run's codes: (T / 16, page bytes) uint8."""
    h, T, _ = f["res"].shape
    P, R = T // PT, f["us"].shape[1]
    us = f["us"].view(P, PT, 4, R // 4).permute(0, 2, 1, 3).reshape(P, -1)
    sc = f["scale"].view(h, T // 64, 2, 64).permute(1, 0, 3, 2).reshape(P, -1)
    c = (f["res"] + 4).view(h, P, PT, 2, 4, 4, 4).permute(1, 0, 5, 2, 3, 4, 6).reshape(P, h, 4, PT, 2, 16)
    lo, hi = c[..., 0, :], c[..., 1, :]
    words = []
    for k in range(3):
        w = (((lo[..., 15] >> k) & 1) << 15) | (((hi[..., 15] >> k) & 1) << 31)
        for p in range(5):
            w = w | (lo[..., 5 * k + p] << (3 * p)) | (hi[..., 5 * k + p] << (16 + 3 * p))
        words.append(w)
    kres = torch.stack(words, -1).to(torch.int32).reshape(P, -1)
    v = f["vidx"].view(h, P, 4, 4, 8, 16).permute(1, 0, 2, 5, 4, 3)                    # P h q m b t
    shift = torch.tensor([0, 2, 4, 6], device="cuda", dtype=torch.int32)
    vcode = (v << shift).sum(-1, dtype=torch.int32).to(torch.uint8).reshape(P, -1)
    parts = [us, f["vnorm"].view(h, P, PT).permute(1, 0, 2).reshape(P, -1), sc, kres, vcode]
    return torch.cat([_bytes(x) for x in parts], 1).contiguous()


def _shared_lengths(case, seed):
    """(committed tokens, window rows) of each sequence: the shared part and up to `own` tokens, a ragged window; an
    idle slot of the batch holds nothing."""
    r = torch.Generator().manual_seed(seed)
    B, own_pages = case["batch"], case["own"] // 128
    lens = [case["shared"] + 128 * int(x) for x in torch.randint(own_pages // 2, own_pages + 1, (B,), generator=r)]
    tails = torch.randint(case["window"] // 2, case["window"] + 1, (B,), generator=r).tolist()
    if case["idle"]:
        lens[B // 2], tails[B // 2] = 0, 0
    return lens, tails


def _shared_data(case, seed):
    g = _gen(seed)
    B, h, G, P = case["batch"], case["h_kv"], case["G"], case["shared"]
    lens, tails = _shared_lengths(case, seed)
    dt = DTYPES[case["dtype"]]
    prefix = _fields(g, h, P, case["rank"])
    owns = [_fields(g, h, n - P, case["rank"]) if n > P else None for n in lens]
    basis = torch.linalg.qr(_randn(g, h * D, case["rank"]).double().cpu())[0].half().cuda().contiguous()
    q = (1.5 * _randn(g, B, h, G, D)).to(dt)
    cap = max(case["window"], 1)
    k_tail, v_tail = (0.7 * _randn(g, B, h, cap, D)).to(dt), _randn(g, B, h, cap, D).to(dt)
    return SimpleNamespace(prefix=prefix, owns=owns, basis=basis, q=q, k_tail=k_tail, v_tail=v_tail, lens=lens,
                           tails=tails, cap=cap)


def _prepare_shared(case, seed):
    d = _shared_data(case, seed)
    B, P = case["batch"], case["shared"]
    runs = [_pages(d.prefix)] + [_pages(o) for o in d.owns if o is not None]
    stacked = torch.cat(runs)
    n_pool = stacked.shape[0] + 5
    r = torch.Generator().manual_seed(seed + 1)
    ids = torch.randperm(n_pool, generator=r)[: stacked.shape[0]].cuda()
    pool = torch.zeros(n_pool, stacked.shape[1], dtype=torch.uint8, device="cuda")
    pool[ids] = stacked
    width = max(max(d.lens), P) // PT
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    at = P // PT
    for b in range(B):
        table[b, : P // PT] = ids[: P // PT]
        n = 0 if d.owns[b] is None else (d.lens[b] - P) // PT
        table[b, P // PT: P // PT + n] = ids[at: at + n]
        at += n
    s = SimpleNamespace(case=case, q=d.q, pool=pool, table=table, basis=d.basis, k_tail=d.k_tail, v_tail=d.v_tail,
                        lens=d.lens, tails=d.tails, cap=d.cap, scale=D ** -0.5, inv_freq=_inv_freq(case["theta"]),
                        packed_len=torch.tensor(d.lens, dtype=torch.int32, device="cuda"),
                        tail_len=torch.tensor(d.tails, dtype=torch.int32, device="cuda"), max_len=width * PT)
    if own:   # what a serving program keeps: the codec's constants and the rotation table of its positions
        from bmx_amd import k2b

        s.consts = k2b.CodecConsts(LEVELS, _sign_words(), tuple(s.inv_freq.tolist()))
        s.rope = k2b.rope_table(s.consts, s.max_len, s.q.device)
    return s


def _window_data(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    h, n, m = case["h_kv"], case["queries"], case["keys"]
    return ((1.5 * _randn(g, h * case["G"], n, D)).to(dt), _randn(g, h, m, D).to(dt), _randn(g, h, m, D).to(dt))


def _page_rows(case, seed):
    """A batch's tables: rows that share their first pages, then pages of their own, ids anywhere in the pool; a few
    pages held by no row; the rest free, in no order.  On the host: (table, lengths, references, free ids)."""
    r = torch.Generator().manual_seed(seed)
    rows, pages, cap, pool = case["rows"], case["pages"], case["cap"], case["pool"]
    shared = min(case["shared"], pages)
    ids = torch.randperm(pool, generator=r)
    lens = torch.randint(max(shared, pages // 2), pages + 1, (rows,), generator=r)
    table = torch.zeros(rows, cap, dtype=torch.int64)
    pos = torch.arange(cap)[None, :].expand(rows, cap)
    held = pos < lens[:, None]
    table[held & (pos < shared)] = ids[:shared].repeat(rows)
    alone = held & (pos >= shared)
    n_alone = int(alone.sum())
    table[alone] = ids[shared: shared + n_alone]
    refs = torch.bincount(table[held], minlength=pool)
    left = ids[shared + n_alone:]
    pinned = left[: len(left) // 16]
    refs[pinned] = 1
    return table, lens, refs, left[len(left) // 16:]


def _prepare_rows(case, seed):
    table, lens, refs, free = _page_rows(case, seed)
    pool = case["pool"]
    stack = torch.full((pool,), -1, dtype=torch.int64)
    stack[: len(free)] = free
    to = dict(dtype=torch.int32, device="cuda")
    s = SimpleNamespace(case=case, table=table.to(**to), n_pages=lens.to(**to), refs=refs.to(**to), free=stack.to(**to),
                        n_free=torch.tensor([len(free)], **to))
    if own:
        from bmx_amd import pages

        s.state = pages.PageState(s.table, s.n_pages, s.refs, s.free, s.n_free)
    return s


def _update_args(case, seed):
    """Which old row each new row continues (-1: none), and the pages each is given, on the host."""
    r = torch.Generator().manual_seed(seed + 2)
    rows, new = case["rows"], case["new_rows"]
    index = torch.randint(0, rows, (new,), generator=r)
    keep = torch.rand(new, generator=r) < 0.6
    index = torch.where(keep, torch.arange(new) % rows, index)
    index[torch.randperm(new, generator=r)[: min(case["drop"], new)]] = -1
    grow = torch.where(torch.rand(new, generator=r) < 0.7, case["grow"], 0)
    return index, grow


def _page_bytes(case):
    return PT * (2 * case["rank"] + 86 * case["h_kv"])


def prepare(case, seed):
    if case["kind"] == "shared":
        return _prepare_shared(case, seed)
    if case["kind"] == "window":
        q, k, v = _window_data(case, seed)
        return SimpleNamespace(case=case, q=q, k=k, v=v, scale=D ** -0.5)
    s = _prepare_rows(case, seed)
    if case["kind"] == "update":
        index, grow = _update_args(case, seed)
        s.index, s.grow = index.to(torch.int32).cuda(), grow.to(torch.int32).cuda()
    else:
        g = _gen(seed)
        s.pools = [torch.randint(0, 256, (case["pool"], _page_bytes(case)), generator=g, device="cuda",
                                 dtype=torch.uint8) for _ in range(case["layers"])]
    return s


# ------------------------------------------------------------------ plain forms


def _plain_rows(pages, h, R, basis, inv_freq, pos0):
    """Keys (rotated) and values of pages in order, each (h, T, D) in 32 bits."""
    P = pages.shape[0]
    T, C = P * PT, h * D
    cut = [0, PT * R * 2, h * PT * 2, C // 2, h * 64 * 12, h * 64 * 8]
    at = [sum(cut[: i + 1]) for i in range(6)]
    part = [pages[:, at[i]: at[i + 1]].contiguous() for i in range(5)]
    us = part[0].view(torch.float16).view(P, 4, PT, R // 4).permute(0, 2, 1, 3).reshape(T, R).float()
    norm = part[1].view(torch.float16).view(P, h, PT).permute(1, 0, 2).reshape(h, T).float()
    scale = part[2].view(torch.float16).reshape(P // 4, h, 64, 2).permute(1, 0, 3, 2).reshape(h, P // 4, D).float()
    w = part[3].view(torch.int32).view(P, h, 4, PT, 3)
    pairs = []
    for p in range(15):
        pairs.append(torch.stack(((w[..., p // 5] >> (3 * (p % 5))) & 7, (w[..., p // 5] >> (16 + 3 * (p % 5))) & 7), -1))
    last = [((w[..., 0] >> s) & 1) | (((w[..., 1] >> s) & 1) << 1) | (((w[..., 2] >> s) & 1) << 2) for s in (15, 31)]
    pairs.append(torch.stack(last, -1))
    codes = torch.stack(pairs, -2).view(P, h, 4, PT, 4, 4, 2)                              # P h q n b i e
    codes = codes.permute(1, 0, 3, 6, 4, 2, 5).reshape(h, T, D) - 4                        # channel 64e + 16b + 4q + i
    k = (us @ basis.float().t()).view(T, h, D).transpose(0, 1) + codes.float() * scale.repeat_interleave(64, 1)
    ang = torch.arange(pos0, pos0 + T, device="cuda", dtype=torch.float32)[:, None] * inv_freq.cuda()[None, :]
    cos, sin = ang.double().cos().float(), ang.double().sin().float()
    a, b = k[..., :64], k[..., 64:]
    k = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    vb = part[4].view(P, h, 4, 16, 8).to(torch.int32)                                      # P h q m b
    vc = torch.stack([(vb >> s) & 3 for s in (0, 2, 4, 6)], -1)                            # ... t
    vc = vc.permute(1, 0, 2, 5, 4, 3).reshape(h, T, D).long()
    lv = torch.tensor(LEVELS, device="cuda")[vc]
    v = (lv @ _hadamard(torch.float32)) * (_signs(D).cuda().float() / D) * norm[..., None]
    return k, v


def _plain_shared(s):
    c = s.case
    B, h, G, P, R = c["batch"], c["h_kv"], c["G"], c["shared"], c["rank"]
    kp, vp = _plain_rows(s.pool[s.table[0, : P // PT].long()], h, R, s.basis, s.inv_freq, 0)
    kp = kp.transpose(1, 2).contiguous()
    out = torch.zeros(B, h, G, D, device="cuda")
    for b in range(B):
        q = s.q[b].float() * s.scale
        ks, vs = [], []
        n = min(s.lens[b], P)
        if n:
            ks.append(q @ kp[:, :, :n])
            vs.append(vp[:, :n])
        if s.lens[b] > P:
            k, v = _plain_rows(s.pool[s.table[b, P // PT: s.lens[b] // PT].long()], h, R, s.basis, s.inv_freq, P)
            ks.append(q @ k.transpose(1, 2).contiguous())
            vs.append(v)
        t = s.tails[b]
        if t:
            ks.append(q @ s.k_tail[b, :, :t].float().transpose(1, 2).contiguous())
            vs.append(s.v_tail[b, :, :t].float())
        if not ks:
            continue
        x = torch.cat(ks, -1)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        out[b] = (p @ torch.cat(vs, 1)) / p.sum(-1, keepdim=True)
    return out.to(s.q.dtype)


def _plain_window(s):
    c = s.case
    G, n, m = c["G"], c["queries"], c["keys"]
    i = torch.arange(n, device="cuda")[:, None] + (m - n)
    j = torch.arange(m, device="cuda")[None, :]
    seen = (j <= i) & ((j > i - c["window"]) | (j < c["sinks"]))
    out = torch.empty_like(s.q)
    for h in range(c["h_kv"]):
        kt, v = s.k[h].float().t().contiguous(), s.v[h].float()
        for g in range(G):
            x = (s.q[h * G + g].float() @ kt * s.scale).masked_fill(~seen, float("-inf"))
            p = torch.exp(x - x.amax(-1, keepdim=True))
            out[h * G + g] = ((p @ v) / p.sum(-1, keepdim=True)).to(out.dtype)
    return out


def _plain_update(s):
    c = s.case
    rows, cap, pool, new = c["rows"], c["cap"], c["pool"], c["new_rows"]
    pos = torch.arange(cap, device="cuda")[None, :]
    src = s.index.long().clamp(min=0)
    lens = torch.where(s.index >= 0, s.n_pages[src], 0)
    table = torch.where(pos < lens[:, None], s.table[src], 0)
    ones = torch.ones(rows * cap, dtype=torch.int32, device="cuda")
    before = torch.zeros(pool + 1, dtype=torch.int32, device="cuda")
    after = before.clone()
    before.scatter_add_(0, torch.where(pos < s.n_pages[:, None], s.table, pool).view(-1).long(), ones)
    after.scatter_add_(0, torch.where(pos < lens[:, None], table, pool).view(-1).long(),
                       torch.ones(new * cap, dtype=torch.int32, device="cuda"))
    refs = s.refs + (after - before)[:pool]
    freed = (s.refs > 0) & (refs <= 0)
    # freed ids in ascending order go on top of the free stack
    n0 = s.n_free.long()
    slot = n0 + torch.cumsum(freed, 0) - 1
    stack = torch.cat((s.free, s.free.new_zeros(1)))
    ids = torch.arange(pool, device="cuda", dtype=torch.int32)
    stack[torch.where(freed, slot, pool)] = ids
    stack = stack[:pool]
    n_free = n0 + freed.sum()
    # new pages off the top, rows in order; all rows or none
    total = s.grow.sum()
    ok = (total <= n_free) & (lens + s.grow <= cap).all()
    grow = torch.where(ok, s.grow, 0).long()
    first = torch.cumsum(grow, 0) - grow
    k = pos - lens[:, None]
    fresh = (k >= 0) & (k < grow[:, None])
    take = n_free - 1 - (first[:, None] + k)
    got = stack[torch.where(fresh, take, 0).clamp(min=0)]
    table = torch.where(fresh, got, table)
    refs = torch.cat((refs, refs.new_zeros(1)))
    refs[torch.where(fresh, got, pool).long()] = 1
    n_free = n_free - grow.sum()
    free = torch.where(ids < n_free, stack, -1)
    status = torch.where(ok, 0, torch.where((lens + s.grow <= cap).all(), 1, 2)).to(torch.int32).view(1)
    return (table.to(torch.int32), (lens + grow).to(torch.int32), refs[:pool].clone(), free.to(torch.int32),
            n_free.to(torch.int32).view(1), status)


def _plain_compact(s):
    pool = s.case["pool"]
    live = s.refs > 0
    n_live = int(live.sum())
    ids = torch.arange(pool, device="cuda")
    src, dst = ids[live & (ids >= n_live)], ids[~live & (ids < n_live)]
    to = ids.clone()
    to[src] = dst
    for p in s.pools:
        p[dst] = p[src]
    held = torch.arange(s.case["cap"], device="cuda")[None, :] < s.n_pages[:, None]
    table = torch.where(held, to[s.table.long()].to(torch.int32), 0)
    refs = s.refs.clone()
    refs[dst] = s.refs[src]
    refs[n_live:] = 0
    free = torch.where(ids < pool - n_live, pool - 1 - ids, -1).to(torch.int32)
    return [table, s.n_pages.clone(), refs, free, torch.tensor([pool - n_live], dtype=torch.int32, device="cuda"),
            *s.pools]


# ------------------------------------------------------------------ one pass


def run(state):
    c = state.case
    if not own:
        return {"shared": _plain_shared, "window": _plain_window, "update": _plain_update,
                "compact": _plain_compact}[c["kind"]](state)
    s = state
    if c["kind"] == "shared":
        from bmx_amd import k2b

        return k2b.decode_shared(s.q, s.pool, s.table, s.packed_len, s.max_len, c["shared"], s.basis, s.consts, s.scale,
                                 rank=c["rank"], rope=s.rope, k_tail=s.k_tail, v_tail=s.v_tail, tail_len=s.tail_len,
                                 tail_cap=s.cap)
    if c["kind"] == "window":
        from bmx_amd import prefill

        return prefill.attention(s.q, s.k, s.v, s.scale, causal=True, window=c["window"], sinks=c["sinks"])
    from bmx_amd import pages

    if c["kind"] == "update":
        o = pages.update(s.state, s.index, s.grow)
        return o.table, o.n_pages, o.refs, o.free, o.n_free, o.status
    o = pages.compact(s.state, s.pools)
    return [o.table, o.n_pages, o.refs, o.free, o.n_free, *s.pools]


# ------------------------------------------------------------------ the work of one pass


def _seen(case):
    """Visible (query, key) pairs of a head, and the keys that some query sees."""
    n, m, w, sinks = case["queries"], case["keys"], case["window"], case["sinks"]
    pairs = 0
    for i in range(m - n, m):
        lo = max(0, i - w + 1)
        pairs += i - lo + 1 + min(sinks, lo)
    lo = max(0, m - n - w + 1)
    return pairs, m - lo + min(sinks, lo)


def work(case):
    if case["kind"] == "shared":
        B, h, G, P = case["batch"], case["h_kv"], case["G"], case["shared"]
        lens, tails = _shared_lengths(case, 0)
        own_tokens, tail_rows = sum(max(n - P, 0) for n in lens), sum(tails)
        packed = P + own_tokens
        pairs = sum(lens) + tail_rows
        return {"bytes": packed * _page_bytes(case) // PT + 4 * tail_rows * h * D + 4 * B * h * G * D
                + 2 * h * D * case["rank"],
                "flops": 4 * G * h * D * pairs + 2 * h * D * case["rank"] * packed}
    if case["kind"] == "window":
        h, G = case["h_kv"], case["G"]
        pairs, keys = _seen(case)
        return {"bytes": 4 * h * keys * D + 4 * h * G * case["queries"] * D, "flops": 4 * h * G * D * pairs}
    rows, cap, pool = case["rows"], case["cap"], case["pool"]
    if case["kind"] == "update":
        return {"bytes": 4 * (rows * case["pages"] + case["new_rows"] * cap + 4 * pool), "flops": 0}
    table, lens, refs, free = _page_rows(case, 0)
    n_live = int((refs > 0).sum())
    moved = int((refs[n_live:] > 0).sum())
    return {"bytes": 2 * moved * case["layers"] * _page_bytes(case) + 4 * (2 * rows * cap + 3 * pool), "flops": 0}


# ------------------------------------------------------------------ exact


def _exact_rows(f, basis, inv_freq, pos0):
    """Keys (rotated) and values (h, T, D) of a token run's codes, in 64 bits."""
    h, T, _ = f["res"].shape
    k = (f["us"].double() @ basis.double().t()).view(T, h, D).permute(1, 0, 2)
    k = k + f["res"].double() * f["scale"].double()[:, torch.arange(T, device="cuda") // 64]
    # the angle is the format's: the 32-bit product of frequency and position
    pos = torch.arange(pos0, pos0 + T, device="cuda").to(torch.float32)
    ang = torch.outer(pos, inv_freq.cuda()).double()
    z = torch.complex(k[..., :64], k[..., 64:]) * torch.polar(torch.ones_like(ang), ang)
    k = torch.cat((z.real, z.imag), -1)
    x = torch.tensor(LEVELS, device="cuda", dtype=torch.float64)[f["vidx"].long()]
    n = 1
    while n < D:   # butterflies
        x = x.view(h, T, D // (2 * n), 2, n)
        x = torch.stack((x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]), -2).reshape(h, T, D)
        n *= 2
    return k, x * _signs(D).cuda().double() * (f["vnorm"].double()[..., None] / D)


def _exact_shared(case, seed):
    d = _shared_data(case, seed)
    B, h, G, P = case["batch"], case["h_kv"], case["G"], case["shared"]
    inv = _inv_freq(case["theta"])
    out = torch.zeros(B, h, G, D, device="cuda", dtype=torch.float64)
    kp, vp = _exact_rows(d.prefix, d.basis, inv, 0)
    for b in range(B):
        ko, vo = _exact_rows(d.owns[b], d.basis, inv, P) if d.owns[b] is not None else (None, None)
        n, t = min(d.lens[b], P), d.tails[b]
        for i in range(h):
            k = [kp[i, :n]] + ([ko[i]] if ko is not None else []) + [d.k_tail[b, i, :t].double()]
            v = [vp[i, :n]] + ([vo[i]] if vo is not None else []) + [d.v_tail[b, i, :t].double()]
            k, v = torch.cat(k), torch.cat(v)
            if k.shape[0] == 0:
                continue
            w = torch.softmax((k @ d.q[b, i].double().t().contiguous()) * D ** -0.5, 0)
            out[b, i] = w.t().contiguous() @ v
    return out


def _exact_window(case, seed):
    q, k, v = _window_data(case, seed)
    G, n, m, w, sinks = case["G"], case["queries"], case["keys"], case["window"], case["sinks"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for i0 in range(0, n, 512):   # queries of a stretch see its band and the first tokens
        i1 = min(i0 + 512, n)
        lo, hi = max(0, i0 + m - n - w + 1), i1 + m - n
        first = min(sinks, lo)
        j = torch.cat((torch.arange(first, device="cuda"), torch.arange(lo, hi, device="cuda")))
        at = torch.arange(i0, i1, device="cuda") + m - n
        gap = at[:, None] - j[None, :]
        hidden = (gap < 0) | ((gap >= w) & (j >= sinks)[None, :])
        for h in range(case["h_kv"]):
            x = q[h * G: (h + 1) * G, i0:i1].double() @ k[h][j].double().t().contiguous()
            x = torch.where(hidden, float("-inf"), x * D ** -0.5)
            out[h * G: (h + 1) * G, i0:i1] = torch.softmax(x, -1) @ v[h][j].double()
    return out


def exact(case, seed):
    """Of the attention operators.  The page operators give whole numbers, which are equal or not."""
    if case["kind"] == "shared":
        return _exact_shared(case, seed)
    if case["kind"] == "window":
        return _exact_window(case, seed)
    return None
