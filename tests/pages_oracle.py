"""Page tables of a batch over plain Python lists: what bmx_amd.pages' calls
give, one page at a time."""


def update(table, n_pages, refs, free, n_free, cap, index, grow):
    """(table, n_pages, refs, free, n_free, status) of the next state; lists."""
    pool = len(refs)
    rows = [table[r][: min(max(n_pages[r], 0), cap)] for r in range(len(table))]
    index = list(range(len(rows))) if index is None else index
    new = [list(rows[i]) if 0 <= i < len(rows) else [] for i in index]
    out_refs = list(refs)
    for sign, part in ((-1, rows), (1, new)):
        for row in part:
            for p in row:
                if 0 <= p < pool:
                    out_refs[p] += sign
    stack = list(free[: min(max(n_free, 0), pool)])
    stack += [p for p in range(pool) if refs[p] > 0 >= out_refs[p]]
    grow = [0] * len(new) if grow is None else [max(g, 0) for g in grow]
    status = 0
    if any(len(r) + g > cap for r, g in zip(new, grow)):
        status = 2
    elif sum(grow) > len(stack):
        status = 1
    if status == 0:
        for r, g in zip(new, grow):
            for _ in range(g):
                p = stack.pop()
                r.append(p)
                out_refs[p] = 1
    return ([r + [0] * (cap - len(r)) for r in new], [len(r) for r in new], out_refs, stack + [-1] * (pool - len(stack)),
            len(stack), status)


def compact(table, n_pages, refs, cap):
    """(table, n_pages, refs, free, n_free, moves) with moves {old id: new id}."""
    pool = len(refs)
    live = [p for p in range(pool) if refs[p] > 0]
    n = len(live)
    moves = dict(zip([p for p in live if p >= n], [p for p in range(n) if refs[p] <= 0]))
    out_refs = [0] * pool
    for p in live:
        out_refs[moves.get(p, p)] = refs[p]
    rows = [[moves.get(p, p) for p in table[r][: min(max(n_pages[r], 0), cap)]] for r in range(len(table))]
    return ([r + [0] * (cap - len(r)) for r in rows], [len(r) for r in rows], out_refs,
            list(range(pool - 1, n - 1, -1)) + [-1] * n, pool - n, moves)
