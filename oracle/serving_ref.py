"""Definitions of what a server does around a paged cache, in 64 bits and one sequence after the other: the plan of a step, the draw of a token."""
import math

import numpy as np


def whole(v, lo, hi):
    """A number as a whole one in lo .. hi; one that is not a number is the lowest."""
    v = float(v)
    return hi if v >= hi else int(v) if v > lo else lo


def plan(new, lens, table, free, tokens, page, origin=None, shared=None):
    """PAGED_PLAN: what becomes of lens, table, free, starts, positions, slots, last, shared (positions and slots of the new rows only);
    listed: how many entries of the stack mean something."""
    table = np.array(table, np.float64)
    B, W = table.shape
    pages = len(free) - 1
    wish = [-1 if float(n) <= -1 else whole(n, 0, 1 << 24) for n in new]
    lens = [whole(n, 0, W * page) for n in lens]
    held = [whole(s, 0, W * page) for s in (shared if shared is not None else [0] * B)]
    valid = lambda p, n: 0 <= p < n  # noqa: E731  (false for what is not a number)
    stack = np.array(free, np.float64)
    count = whole(stack[0], 0, pages)
    old = table.copy()
    after, borrowed = list(lens), list(held)
    for b in range(B):
        if wish[b] >= 0:
            continue
        for e in range(held[b] // page, -(-lens[b] // page)):
            if valid(old[b, e], pages) and count < pages:
                stack[1 + count] = int(old[b, e])
                count += 1
        table[b], after[b], borrowed[b] = -1, 0, 0
    starts, positions, slots, last = [0], [], [], []
    asked, needed, waits = 0, 0, False
    top = count
    for b in range(B):
        rows = 0
        if wish[b] > 0:
            begin, lender = lens[b], -1
            if begin == 0 and origin is not None and valid(origin[b], B) and int(origin[b]) != b and wish[int(origin[b])] >= 0:
                lender = int(origin[b])
                begin = min(held[b] // page, lens[lender] // page) * page
            if begin + wish[b] <= W * page:
                first, end = -(-begin // page), -(-(begin + wish[b]) // page)
                asked += wish[b]
                needed += end - first
                waits = waits or needed > count or asked > tokens
                if not waits:
                    rows = wish[b]
                    if lender >= 0:
                        table[b, :first] = old[lender, :first]
                    for e in range(first, end):
                        top -= 1
                        table[b, e] = int(stack[1 + top]) if valid(stack[1 + top], pages) else -1
                    if lens[b] == 0:
                        borrowed[b] = begin
                    after[b] = begin + rows
                    for t in range(begin, begin + rows):
                        p = table[b, t // page]
                        positions.append(t)
                        slots.append(int(p) * page + t % page if valid(p, pages) else -1)
        starts.append(starts[-1] + rows)
        last.append(starts[-1] - 1 if rows else -1)
    # what lies behind the number that remains is left as it was
    free = np.concatenate([[top], stack[1:1 + top], np.asarray(free, np.float64)[1 + top:]])
    return dict(lens=after, table=table, free=free, starts=starts, positions=positions, slots=slots, last=last, shared=borrowed, listed=top)


def sample(x, u, temperature=1.0, k=0, p=1.0, m=0.0):
    """SAMPLE_FWD of one row: (id, logarithm of its share, distance of u from the nearest border that decides, as a share of the sum)."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, 0.0, 1.0
    if not temperature > 0:
        return int(np.argmax(x)), 0.0, 1.0
    order = np.argsort(-x, kind="stable")
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / temperature)))
    near = 1.0
    if m > 1:
        order = order[:1]
    else:
        if 1 <= k < len(x):
            order = order[:int(k)]
        if p < 1:
            sums = np.cumsum(w[order])
            target = max(p, 0.0) * math.fsum(w[order])
            n = 1 + int(np.searchsorted(sums, target, side="left"))
            near = min(near, float(np.abs(sums - target)[w[order] > 0].min() / sums[-1])) if target > 0 else near
            order = order[:max(1, n)]
        if m > 0:
            below = w[order][x[order] < top]
            near = min([near] + np.abs(below - m).tolist())
            order = order[w[order] >= m]
    order = np.sort(order)
    order = order[w[order] > 0]
    sums = np.cumsum(w[order])
    target = min(max(u, 0.0), 1.0) * sums[-1] if u == u else 0.0
    at = min(int(np.searchsorted(sums, target, side="right")), len(order) - 1)
    if 0 < u < 1:
        near = min(near, float(np.abs(sums[:-1] - target).min() / sums[-1])) if len(order) > 1 else near
    i = int(order[at])
    log = 0.0 if x[i] == top else (x[i] - top) / temperature
    return i, log - math.log(math.fsum(w[order])), near
