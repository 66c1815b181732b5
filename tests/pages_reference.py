"""The page operations one entry after the other, in Python lists, from their definitions."""


def used(rows, page_size, width):
    return min(-(-max(rows, 0) // page_size), width)


def reserve(refs, table, lens, page_size, extra=0):
    missing = 0
    for row, n in zip(table, lens):
        for j in range(used(n + extra, page_size, len(row))):
            if row[j] < 0:
                free = next((p for p, r in enumerate(refs) if r == 0), None)
                if free is None:
                    missing += 1
                else:
                    row[j] = free
                    refs[free] = 1
    return missing


def drop(refs, page):
    if 0 <= page < len(refs) and refs[page] > 0:
        refs[page] -= 1


def free(refs, table, lens=None, page_size=1, extra=0):
    for i, row in enumerate(table):
        for j in range(used(lens[i] + extra, page_size, len(row)) if lens is not None else 0, len(row)):
            drop(refs, row[j])
            row[j] = -1 if row[j] >= 0 else row[j]


def fork(caches, refs, table, lens, parents, page_size, keep_parents=False):
    """caches: lists of pages, each a list of rows (anything)."""
    width = len(table[0]) if table else 0
    new, new_lens, last = [], [], []
    for p in parents:
        ok = 0 <= p < len(table)
        n = max(0, min(lens[p], width * page_size)) if ok else 0
        row = [table[p][j] if j < used(n, page_size, width) and 0 <= table[p][j] < len(refs) else -1 for j in range(width)] if ok else [-1] * width
        for x in row:
            if x >= 0:
                refs[x] += 1
        new.append(row)
        new_lens.append(n)
        last.append(row[n // page_size] if n % page_size else -1)
    if not keep_parents:
        for row in table:
            for x in row:
                drop(refs, x)
    avail = [p for p, r in enumerate(refs) if r == 0]
    missing = 0
    for i, page in enumerate(last):
        if page < 0 or refs[page] <= 1:
            continue
        n = new_lens[i]
        refs[page] -= 1
        if avail:
            to = avail.pop(0)
            refs[to] = 1
            new[i][n // page_size] = to
            for c in caches:
                for r in range(n % page_size):
                    c[to][r] = c[page][r]
        else:
            missing += 1
            new[i][n // page_size] = -1
            new_lens[i] = n - n % page_size
    return new, new_lens, missing
