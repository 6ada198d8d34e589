"""Forking and compacting pages of a cache, on lists."""


def fork(table, lens, P, num_pages, parents=None, new_lens=None, held=None, width=None):
    """(new table, new lengths, copies [(source, destination, slots)], free pages left)."""
    W = len(table[0]) if table else 0
    width = W if width is None else width
    N = len(table) if parents is None else len(parents)
    held = set() if held is None else {i for i, h in enumerate(held) if h}
    rows, seen = [], set()
    used = set(held)
    for i in range(N):
        p = i if parents is None else parents[i]
        there = 0 <= p < len(table)
        n = min(max(lens[p], 0), min(W, width) * P) if there else 0
        cells = [table[p][j] for j in range(n // P)]
        copy = None
        if n % P:
            last = table[p][n // P]
            if not 0 <= last < num_pages or (p not in seen and last not in held):
                cells.append(last)
            else:
                copy = last
        if there:
            seen.add(p)
        used |= {c for c in cells if 0 <= c < num_pages}
        if copy is not None:
            used.add(copy)   # (its first row has it, or it is held)
        rows.append((n, cells, copy))
    free = [p for p in range(num_pages) if p not in used]
    at, copies, out, out_lens = 0, [], [], []
    for i, (n, cells, copy) in enumerate(rows):
        new = 0 if new_lens is None else max(new_lens[i], 0)
        cells = list(cells)
        want = min(-(-(n + new) // P), width) - len(cells)
        for c in range(want):
            page = free[at] if at < len(free) else -1
            at += 1
            if c == 0 and copy is not None:
                if page >= 0:
                    copies.append((copy, page, n % P))
                else:
                    n -= n % P
            cells.append(page)
        out.append(cells + [-1] * (width - len(cells)))
        out_lens.append(n)
    return out, out_lens, copies, len(free) - at


def compact(table, lens, P, num_pages, held=None):
    """(new table, moves [(source, destination)], pages used)."""
    W = len(table[0]) if table else 0
    held = set() if held is None else {i for i, h in enumerate(held) if h}
    cells = [-(-min(max(n, 0), W * P) // P) for n in lens]
    pages = {row[j] for row, c in zip(table, cells) for j in range(c) if 0 <= row[j] < num_pages}
    live = sorted(pages - held)
    room = [p for p in range(num_pages) if p not in held][:len(live)]
    holes = [p for p in room if p not in pages]
    moves = list(zip([p for p in live if p not in set(room)], holes))
    to = dict(moves)
    new = [[to.get(row[j], row[j]) if j < c else -1 for j in range(W)] for row, c in zip(table, cells)]
    return new, moves, max(room + sorted(held), default=-1) + 1
