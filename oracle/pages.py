"""The pages of a cache with lists and loops: what the tests hold the kernels to."""
from __future__ import annotations


def counted(table, n):
    refs = [0] * n
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return refs


def fork(table, lengths, parents):
    W = len(table[0])
    return ([list(table[p]) if p >= 0 else [-1] * W for p in parents], [lengths[p] if p >= 0 else 0 for p in parents])


def reserve(table, lengths, counts, n, page):
    """(table, granted, sources, targets): one sequence after another, from the definition."""
    table = [list(row) for row in table]
    B, W = len(table), len(table[0])
    first, need = [], []
    for b in range(B):
        count = max(0, min(counts[b], W * page - lengths[b]))
        need.append(-(-(lengths[b] + count) // page))
        first.append(lengths[b] // page if count else need[b])
        for i in range(need[b], W):
            table[b][i] = -1
    refs = counted(table, n)
    holders = {}
    writers = {}
    for b in range(B):
        for i in range(W):
            if table[b][i] >= 0:
                holders.setdefault(table[b][i], []).append((b, i))
                if first[b] <= i < need[b]:
                    writers.setdefault(table[b][i], []).append((b, i))
    def keeper(p):
        """Of those that hold a page the one with the most tokens on it, the lowest of several: nobody else's tokens lie where it goes on."""
        return max(holders[p], key=lambda at: (max(0, lengths[at[0]] - at[1] * page), -at[0]))

    free = iter([p for p in range(n) if refs[p] == 0])
    granted, sources, targets = [], [-1] * B, [-1] * B
    for b in range(B):
        count = max(0, min(counts[b], W * page - lengths[b]))
        room = count
        for i in range(first[b], need[b]):
            p = table[b][i]
            if p >= 0 and (len(holders[p]) == 1 or (writers[p] == holders[p] and (b, i) == keeper(p))):
                continue
            new = next(free, None)
            if new is None:
                room = min(room, max(0, i * page - lengths[b]))
                continue
            if p >= 0 and i == lengths[b] // page and lengths[b] % page:
                sources[b], targets[b] = p, new
            table[b][i] = new
        granted.append(room)
    return table, granted, sources, targets


def compact(table, refs):
    used = [p for p, r in enumerate(refs) if r > 0]
    moved = [p for p in used if p >= len(used)]
    holes = [p for p in range(len(used)) if refs[p] == 0]
    to = {p: p for p in used if p < len(used)}
    to.update(zip(moved, holes))
    new = [0] * len(refs)
    for p in used:
        new[to[p]] = refs[p]
    return [[to.get(p, -1) for p in row] for row in table], new, moved, holes
