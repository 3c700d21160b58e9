"""Forking requests and compacting a pool of pages, request by request and page by page on the host."""

from __future__ import annotations


def pages(tokens, page):
    return -(-tokens // page)


def fork(parents, keep, lens, table, ring, head, count, page):
    """Lists in, new ones out: {seq_lens, block_table, state, ring, copies}."""
    B, span, N = len(table), len(table[0]) * page, len(ring)
    inside = lambda p: 0 <= p < N
    lens = [min(max(n, 0), span) for n in lens]
    head, count = head % N, min(max(count, 0), N)
    plan = []
    for p, k in zip(parents, keep):
        ok = 0 <= p < B
        n = min(max(k, 0), lens[p]) if ok else 0
        plan.append((n, list(table[p][:pages(n, page)]) if ok else []))
    whole = {p for n, row in plan for p in row[:n // page] if inside(p)}
    first = {}
    for b, (n, row) in enumerate(plan):
        if n % page:
            first.setdefault(row[-1], b)
    ring, out, copies, after, taken = list(ring), [], [], [], 0
    old_ring = list(ring)
    held = set(whole)
    for b, (n, row) in enumerate(plan):
        pair = [-1, -1]
        if n % page and inside(row[-1]):
            if row[-1] not in whole and first[row[-1]] == b:
                held.add(row[-1])
            elif taken < count:
                pair = [row[-1], old_ring[(head + taken) % N]]
                row[-1] = pair[1]
                taken += 1
            else:
                n, row = n // page * page, row[:-1]
        out.append(row + [0] * (len(table[0]) - len(row)))
        copies.append(pair)
        after.append(n)
    was = {p for row, n in zip(table, lens) for p in row[:pages(n, page)] if inside(p)}
    freed = sorted(was - held)
    for i, p in enumerate(freed):
        if count + i < N:
            ring[(head + count + i) % N] = p
    return {"seq_lens": after, "block_table": out, "copies": copies, "ring": ring,
            "state": [(head + taken) % N, min(N, count - taken + len(freed))]}


def compact(lens, table, ring, head, count, page):
    span, N = len(table[0]) * page, len(ring)
    head, count = head % N, min(max(count, 0), N)
    rows = [row[:pages(min(max(n, 0), span), page)] for row, n in zip(table, lens)]
    used = {p for row in rows for p in row if 0 <= p < N}
    free = {p for p in (ring[(head + i) % N] for i in range(count)) if 0 <= p < N} - used
    order = sorted(used | free)
    low, rest = order[:len(used)], order[len(used):]
    moves = list(zip((p for p in rest if p in used), (p for p in low if p in free)))
    to = dict(moves)
    out = [[to.get(p, p) for p in row] + [0] * (len(table[0]) - len(row)) for row in rows]
    room = max(1, N // 2)
    return {"block_table": out, "ring": rest + [-1] * (N - len(rest)), "state": [0, len(rest)],
            "copies": [list(m) for m in moves] + [[-1, -1]] * (room - len(moves))}


def contents(row, n, page, pool):
    """The tokens that a request sees, by their places: pool maps (page, place) to a token."""
    return [pool[row[i // page], i % page] for i in range(n)]
