"""bmx_amd.pages against plain Python lists (pages_oracle): every word of the
new state equal; and a run of the calls as a server makes them, with the
appends and the attention that read the tables."""
import random

import pytest
import torch

import pages_oracle as O
from bmx_amd import k2b, pages, synth

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class State:
    def __init__(self, table, n_pages, refs, free, cap):
        pool = len(refs)
        self.table, self.n_pages, self.refs, self.cap = table, n_pages, refs, cap
        self.free, self.n_free = free + [-1] * (pool - len(free)), len(free)

    def dev(self):
        return pages.PageState(_dev(self.table).view(len(self.table), self.cap), _dev(self.n_pages), _dev(self.refs),
                               _dev(self.free), _dev([self.n_free]))


def _random(rng, rows, cap, pool, shared=0, fill=0.7):
    """Rows that share their first pages, then pages of their own; some pages
    held by no row; the rest free, in no order.  Entries past a row's pages are
    anything."""
    ids = list(range(pool))
    rng.shuffle(ids)
    head, ids = ids[:shared], ids[shared:]
    table, n_pages, refs = [], [], [0] * pool
    for _ in range(rows):
        n = min(rng.randint(0, cap), len(head) + int(fill * len(ids)))
        own = max(n - len(head), 0)
        row = head[:n] + ids[:own]
        ids = ids[own:]
        for p in row:
            refs[p] += 1
        table.append(row + [rng.randint(-2**31, 2**31 - 1) for _ in range(cap - len(row))])
        n_pages.append(len(row))
    pinned, ids = ids[: len(ids) // 10], ids[len(ids) // 10:]
    for p in pinned:
        refs[p] = rng.randint(1, 3)
    free = [p for p in ids if refs[p] == 0] + [p for p in head if refs[p] == 0]
    return State(table, n_pages, refs, free, cap)


def _check_update(s, index, grow, state=None):
    want = O.update(s.table, s.n_pages, s.refs, s.free, s.n_free, s.cap, index, grow)
    d = s.dev()
    before = [t.clone() for t in (d.table, d.n_pages, d.refs, d.free, d.n_free)]
    o = pages.update(d, None if index is None else _dev(index), None if grow is None else _dev(grow), out=state)
    torch.cuda.synchronize()
    for name, got, ref in zip(("table", "n_pages", "refs", "free", "n_free", "status"),
                              (o.table, o.n_pages, o.refs, o.free, o.n_free, o.status), want):
        ref = torch.tensor(ref, dtype=torch.int32).view(got.shape)
        assert torch.equal(got.cpu(), ref), name
    for t, b in zip((d.table, d.n_pages, d.refs, d.free, d.n_free), before):
        assert torch.equal(t, b)   # the given state stays as it is
    return want


# rows, cap, pool: the last two are past the one-launch form
SIZES = [(1, 1, 1), (1, 5, 7), (3, 8, 64), (8, 100, 1000), (17, 33, 1025), (64, 16, 2048), (5, 2100, 16384),
         (40, 1500, 9000), (6, 300, 40000)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_update_matches_lists(size, seed):
    rows, cap, pool = size
    rng = random.Random(100 * seed + rows)
    s = _random(rng, rows, cap, pool, shared=rng.choice([0, min(cap, pool) // 2]))
    new = rng.choice([rows, 1, 2 * rows + 3])
    for index in (None, [rng.randint(-1, rows - 1) for _ in range(new)], [0] * new, [-1] * new,
                  [rng.choice([-7, rows, 2**31 - 1, -2**31, 0]) for _ in range(new)], list(range(rows))[::-1]):
        n = rows if index is None else len(index)
        for grow in (None, [rng.randint(0, 3) for _ in range(n)], [0] * n):
            print(f"update {size} seed {seed}", None if index is None else index[:6], flush=True)
            _check_update(s, index, grow)


@pytest.mark.parametrize("pool", [50, 20000])
def test_growth_takes_freed_pages_and_all_or_nothing(pool):
    """Just enough pages, one too few, a row at its end, rows that only drop,
    counts below 0 and past every size."""
    table = [[3, 4, 5, 0], [3, 6, 7, 8], [9, 0, 0, 0]]
    refs = [0] * pool
    for p in (4, 5, 6, 7, 8, 9):
        refs[p] = 1
    refs[3] = 2
    s = State(table, [3, 4, 1], refs, [1, 2], 4)
    assert _check_update(s, [0, -1, 2], [1, 0, 3])[5] == 0          # 2 free, 6 7 8 freed, 4 given
    assert _check_update(s, [0, -1, 2], [1, 2, 3])[5] == 1          # 6 asked of 5
    assert _check_update(s, [0, -1, 2], [1, 1, 3])[5] == 0          # all of them
    assert _check_update(s, [0, 1, 2], [0, 1, 0])[5] == 2           # row 1 is full
    assert _check_update(s, None, [-5, -1, 2])[5] == 0
    assert _check_update(s, None, [2**31 - 1, 0, 0])[5] == 2
    assert _check_update(s, [-1, -1], [4, 4])[5] == 0               # new rows over dropped ones
    assert _check_update(s, [-1], [2**31 - 1])[5] == 2


@pytest.mark.parametrize("pool", [50, 20000])
def test_ids_outside_the_pool_and_lengths_outside_the_row(pool):
    table = [[3, -1, pool, 2**31 - 1], [-2**31, 4, 3, 3]]
    refs = [0] * pool
    refs[3], refs[4] = 3, 1
    s = State(table, [99, 3], refs, [1], 4)
    for index in (None, [1, 1, 0], [-1, 0]):
        _check_update(s, index, None)
    s.n_pages = [-3, 4]
    _check_update(s, [0, 1], [1, 0])
    s.n_free = 10**6   # taken as the whole stack
    s.free = list(range(pool))
    _check_update(s, None, [2, 0])


def test_many_rows_and_a_wide_pool():
    """1,500 rows over 300,000 ids; contended counts of a page that all rows hold."""
    rng = random.Random(5)
    s = _random(rng, 1500, 12, 300000, shared=3)
    _check_update(s, [rng.randint(-1, 1499) for _ in range(2000)], [rng.randint(0, 1) for _ in range(2000)])


def test_state_buffers_are_taken_and_repeats_are_equal():
    rng = random.Random(6)
    for rows, cap, pool in ((4, 20, 200), (6, 300, 40000)):
        s = _random(rng, rows, cap, pool, shared=5)
        index, grow = [0, 0, 1, -1, 2], [1, 0, 2, 1, 0]
        d = s.dev()
        buf = d.like(5)
        for t in (buf.table, buf.n_pages, buf.refs, buf.free, buf.n_free, buf.status):
            t.fill_(-77)
        _check_update(s, index, grow, state=buf)
        a = pages.update(d, _dev(index), _dev(grow))
        b = pages.update(d, _dev(index), _dev(grow))
        for x, y in ((a.table, b.table), (a.refs, b.refs), (a.free, b.free)):
            assert torch.equal(x, y)


def _check_compact(s, sizes, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pools = [torch.randint(0, 256, (len(s.refs), n), generator=g, device=DEV, dtype=torch.uint8) for n in sizes]
    was = [p.clone() for p in pools]
    table, n_pages, refs, free, n_free, moves = O.compact(s.table, s.n_pages, s.refs, s.cap)
    d = s.dev()
    o = pages.compact(d, pools)
    torch.cuda.synchronize()
    for name, got, ref in zip(("table", "n_pages", "refs", "free", "n_free"),
                              (o.table, o.n_pages, o.refs, o.free, o.n_free), (table, n_pages, refs, free, n_free)):
        assert torch.equal(got.cpu(), torch.tensor(ref, dtype=torch.int32).view(got.shape)), name
    for p, w in zip(pools, was):
        if moves:
            w[list(moves.values())] = w[list(moves)]
        assert torch.equal(p, w)   # moved pages at their new ids, all others as they were
    return moves


@pytest.mark.parametrize("size", [(1, 1, 1), (3, 8, 64), (8, 100, 1000), (17, 33, 1025), (5, 200, 5000), (3, 40, 1024)])
@pytest.mark.parametrize("seed", [0, 1])
def test_compact_matches_lists(size, seed):
    rows, cap, pool = size
    rng = random.Random(seed + pool)
    for fill in (0.0, 0.3, 1.0):
        s = _random(rng, rows, cap, pool, shared=min(3, cap), fill=fill)
        print(f"compact {size} {seed} {fill}", flush=True)
        _check_compact(s, rng.choice([[16], [16, 4096, 12032], [16400]]), seed)


def test_compact_edges():
    pool = 2048
    none = State([[0, 0]], [0], [0] * pool, list(range(pool)), 2)
    assert _check_compact(none, [32]) == {}
    full = State([[1, 2]], [2], [1] * pool, [], 2)
    assert _check_compact(full, [32]) == {}
    refs = [0] * pool
    for p in range(1024, 2048):
        refs[p] = 1
    assert len(_check_compact(State([[1024, 2047]], [2], refs, list(range(1024)), 2), [48])) == 1024   # every live page
    o = pages.compact(full.dev(), [])                                                               # tables alone
    torch.cuda.synchronize()
    assert o.n_free.item() == 0


def test_a_pool_listed_twice_and_pools_of_several_sizes():
    rng = random.Random(8)
    s = _random(rng, 4, 30, 400, fill=0.5)
    g = torch.Generator(device=DEV).manual_seed(1)
    a, b = [torch.randint(0, 256, (400, n), generator=g, device=DEV, dtype=torch.uint8) for n in (1600, 48)]
    wa, wb = a.clone(), b.clone()
    moves = O.compact(s.table, s.n_pages, s.refs, s.cap)[5]
    pages.compact(s.dev(), [a, b, a])
    torch.cuda.synchronize()
    wa[list(moves.values())], wb[list(moves.values())] = wa[list(moves)], wb[list(moves)]
    assert torch.equal(a, wa) and torch.equal(b, wb)


@pytest.mark.parametrize("pool", [200, 40000])
def test_under_graph_capture(pool):
    """A captured update, replayed with other indices and states between eager
    calls, and a captured compact."""
    rng = random.Random(9)
    cap, rows = 20, 4
    states = [_random(rng, rows, cap, pool, shared=4, fill=0.01) for _ in range(3)]
    d = states[0].dev()
    index, grow = _dev([0, 1, 2, 3]), _dev([0, 0, 0, 0])
    out = d.like(4)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pages.update(d, index, grow, out=out)
        done = pages.compact(out, [])
    for s, idx, gr in ((states[1], [0, 0, -1, 2], [1, 0, 2, 0]), (states[2], [3, 2, 1, 0], [0, 0, 0, 1]),
                       (states[0], [1, 1, 1, 1], [2, 2, 2, 2])):
        src = s.dev()
        for t, x in ((d.table, src.table), (d.n_pages, src.n_pages), (d.refs, src.refs), (d.free, src.free),
                     (d.n_free, src.n_free), (index, _dev(idx)), (grow, _dev(gr))):
            t.copy_(x)
        g.replay()
        pages.update(src, _dev([0]))
        torch.cuda.synchronize()
        want = O.update(s.table, s.n_pages, s.refs, s.free, s.n_free, cap, idx, gr)
        assert out.table.tolist() == want[0] and out.refs.tolist() == want[2] and out.free.tolist() == want[3]
        w2 = O.compact(want[0], want[1], want[2], cap)
        assert done.table.tolist() == w2[0] and done.refs.tolist() == w2[2] and done.n_free.item() == w2[4]


def test_refusals():
    s = _random(random.Random(1), 3, 8, 64).dev()
    ok = torch.zeros(3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="int32"):
        pages.update(s, ok.long())
    with pytest.raises(ValueError, match="grow"):
        pages.update(s, ok, ok[:2])
    with pytest.raises(ValueError, match="out"):
        pages.update(s, ok, out=s.like(4))
    with pytest.raises(RuntimeError, match="buffers of its own"):
        pages.update(s, None, out=s)
    with pytest.raises(ValueError, match="multiple of 16"):
        pages.compact(s, [torch.zeros(64, 40, dtype=torch.uint8, device=DEV)])
    with pytest.raises(ValueError, match="n_pool"):
        pages.compact(s, [torch.zeros(63, 48, dtype=torch.uint8, device=DEV)])
    with pytest.raises(RuntimeError, match="aligned"):
        pages.compact(s, [torch.zeros(64 * 48 + 1, dtype=torch.uint8, device=DEV)[1:].view(64, 48)])


def test_a_served_batch_from_prompt_to_compaction():
    """A prompt's pages committed into rows of the tables, three samples forked
    off it, each given a codec page of its own and attended with decode_shared
    and decode; one dropped, its pages handed to another; the pools closed up:
    the outputs before and after equal bit for bit."""
    h, G, R, P = 2, 4, 16, 512
    gen = torch.Generator().manual_seed(3)
    consts = k2b.CodecConsts.make()
    k_pre, v = synth.k2b_keys(h, P + 512, R, gen), synth.values(h, P + 512, gen)
    us, basis = synth.first_page_svd(k_pre, R)
    basis32 = basis.to(DEV).contiguous()
    basis16 = basis32.half().contiguous()
    pool = torch.zeros(200, k2b.page_bytes(h, R), dtype=torch.uint8, device=DEV)
    cap = 64

    def commit(ids, at, n, first=None):
        k2b.append(k_pre[:, at:at + n].to(DEV), v[:, at:at + n].to(DEV), basis32, basis16, pool, ids.contiguous(), consts,
                   rank=R, us_first=first)

    s = pages.update(pages.PageState.make(1, cap, 200, DEV), None, _dev([P // 16]))
    commit(s.table[0, : P // 16], 0, P, us.to(DEV).float().contiguous())
    s = pages.update(s, _dev([0, 0, 0]), _dev([8, 8, 8]))
    assert s.status.item() == 0 and s.refs[s.table[0, 0].long()].item() == 3
    for r in range(3):
        commit(s.table[r, P // 16: P // 16 + 8], P + 128 * r, 128)
    rope = k2b.rope_table(consts, cap * 16, DEV)
    q = torch.randn(3, h, G, 128, generator=gen).half().to(DEV)

    def attend(s, rows):
        lens = s.n_pages * 16
        kw = dict(rank=R)
        out = k2b.decode_shared(q[rows], pool, s.table, lens, cap * 16, P, basis16, consts, 128 ** -0.5, rope=rope, **kw)
        ref = k2b.decode(q[rows], pool, s.table, lens, cap * 16, basis16, consts, 128 ** -0.5, **kw)
        torch.cuda.synchronize()
        torch.testing.assert_close(out.float(), ref.float(), atol=2e-3, rtol=1e-2)
        return out
    first = attend(s, [0, 1, 2])
    t = pages.update(s, _dev([2, 0]), _dev([0, 0]))           # the second sample is dropped, the others change places
    assert torch.equal(attend(t, [2, 0]), first[[2, 0]])
    t = pages.update(t, None, _dev([0, 8]))                   # and its pages serve another
    assert t.status.item() == 0 and set(t.table[1, 40:48].tolist()) == set(s.table[1, 32:40].tolist())
    commit(t.table[1, 40:48], P + 384, 128)
    before = attend(t, [2, 0])
    t = pages.compact(pages.update(t, _dev([1]), None), [pool])
    assert t.n_free.item() == 200 - 48 and t.table[0, :48].max().item() == 47
    assert torch.equal(attend(t, [0]), before[1:])


def test_status_belongs_to_updates():
    """compact's new state has no status, buffers given to it keep theirs, and an
    update makes or checks one."""
    s = pages.PageState.make(2, 8, 16, DEV)
    s = pages.update(s, None, _dev([3, 2]))
    c = pages.compact(s, [])
    assert c.status is None
    buf = s.like()
    buf.status.fill_(7)
    pages.compact(s, [], out=buf)
    assert buf.status.item() == 7
    nxt = pages.update(c, _dev([1, 0]), out=c.like())
    assert nxt.status.item() == pages.OK and nxt.n_pages.tolist() == [2, 3]
    bare = c.like()
    bare.status = None
    assert pages.update(c, None, out=bare).status.item() == pages.OK
    bare.status = torch.zeros(1, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="status"):
        pages.update(c, None, out=bare)
