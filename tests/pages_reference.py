"""Plain Python forms of the tables of shared pages, and random pools for their tests."""


def _held(table, lens, page):
    """(tokens, ids of the pages) of each row: no more than its columns have room for."""
    out = []
    for row, n in zip(table, lens):
        n = min(max(n, 0), len(row) * page)
        out.append((n, row[: -(-n // page)]))
    return out


def fork(table, lens, parents, kept, pinned, free_pages, free_start, page, num_pages):
    """-> new table, lens, copies, free_next, and the free list afterwards."""
    width, old = len(table[0]), _held(table, lens, page)
    real = lambda i: 0 <= i < num_pages  # noqa: E731
    rows = []
    for p, k in zip(parents, kept):
        n, ids = old[p] if 0 <= p < len(old) else (0, [])
        n = min(n, max(k, 0))
        rows.append((n, list(ids[: -(-n // page)])))
    whole = {i for n, ids in rows for i in ids[: n // page] if real(i)} | {i for i in range(num_pages) if pinned[i] > 0}
    copies, keeps, needs = [[-1, -1, 0] for _ in rows], set(), []
    for b, (n, ids) in enumerate(rows):
        if n % page and real(ids[-1]):
            if ids[-1] in whole or ids[-1] in keeps:
                needs.append(b)
            else:
                keeps.add(ids[-1])
    freed = sorted({i for _, ids in old for i in ids if real(i)} - whole - keeps)
    free, at = list(free_pages), free_start - len(freed)
    for k, i in enumerate(freed):
        if 0 <= at + k < len(free):
            free[at + k] = i
    for b in needs:
        n, ids = rows[b]
        got = free[at] if 0 <= at < len(free) else -1
        at += 1
        copies[b] = [ids[-1], got, n % page]
        ids[-1] = got
    return [ids + [-1] * (width - len(ids)) for _, ids in rows], [n for n, _ in rows], copies, at, free


def compact(table, lens, pinned, free_pages, free_start, page, num_pages):
    """-> new table, copies, free list."""
    old, start = _held(table, lens, page), min(max(free_start, 0), len(free_pages))
    real = lambda i: 0 <= i < num_pages  # noqa: E731
    held = {i for _, ids in old for i in ids if real(i)}
    fixed = {i for i in range(num_pages) if pinned[i] > 0}
    low = sorted({i for i in free_pages[start:] if real(i)} - held - fixed)
    high = sorted(held - fixed, reverse=True)
    moves = [(t, f) for t, f in zip(high, low) if f < t]
    to = dict(moves)
    new = [[to.get(i, i) for i in ids] + [-1] * (len(table[0]) - len(ids)) for _, ids in old]
    rest = sorted((set(low) - {f for _, f in moves}) | {t for t, _ in moves})
    free = [-1] * start + rest + [-1] * (len(free_pages) - start - len(rest))
    copies = [[t, f, page] for t, f in moves]
    return new, copies + [[-1, -1, 0]] * (min(len(free_pages), num_pages // 2) - len(moves)), free


def random_pool(rng, rows, width, page, num_pages, shared=0.3, odd=0.0):
    """A table of `rows` requests: pages of their own, prefixes shared with the row above, and (odd) ids that are none;
    its lengths, the free list with its start, pins."""
    order = list(range(num_pages))
    rng.shuffle(order)
    table, lens, k = [], [], 0
    for r in range(rows):
        n = rng.choice([0, 1, page, rng.randint(0, width * page), rng.randint(0, width * page)])
        need = -(-n // page)
        ids = []
        if r and rng.random() < shared:
            whole = min(need, max(lens[-1], 0) // page, width)
            ids = table[-1][: rng.randint(0, whole)]
        while len(ids) < need and k < num_pages:
            ids.append(order[k])
            k += 1
        n = min(n, len(ids) * page)
        ids += [-1] * (width - len(ids))
        if odd and rng.random() < odd:
            ids[rng.randrange(width)] = rng.choice([-1, num_pages, 2 ** 31 - 1, -2 ** 31])
        table.append(ids)
        lens.append(n)
    spare = rng.randint(0, 3)
    free = [-1] * k + order[k:]
    free = free[spare:] if spare <= k else free
    start = k - spare if spare <= k else k
    pinned = [1 if rng.random() < 0.05 else 0 for _ in range(num_pages)]
    return table, lens, free, start, pinned
