"""Pages that sequences share, verification of drafted tokens and low-rank adapters from their definitions, one thing after the other, in 64 bits
(CPU tensors and lists)."""
import math

import torch

H = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative to the value


# ------------------------------------------------------------------------------------------------ pages
def fork(users, table, lengths, parents, page):
    """New (users, table, lengths) as lists."""
    users, width = list(users), len(table[0]) if table else 0
    new, lens = [], []
    for b, parent in enumerate(parents):
        n = 0 if parent == -1 else lengths[parent]
        pages = -(-n // page)
        new.append([-1] * width if parent == -1 else [max(-1, p) if i < pages else -1 for i, p in enumerate(table[parent])])
        lens.append(n)
    for old, row in zip(table, new):
        for p in old:
            if p >= 0:
                users[p] -= 1
        for p in row:
            if p >= 0:
                users[p] += 1
    return users, new, lens


def grow(users, table, starts, lengths, page):
    """New (users, table, granted, copies) as lists; copies: (from, to, keys)."""
    users, table = list(users), [list(r) for r in table]
    free = [p for p, n in enumerate(users) if n == 0]
    granted, copies, short = [], [], False
    count = {}
    # what each would take if all before it got theirs
    plans, want = [], 0
    for b, row in enumerate(table):
        n = starts[b + 1] - starts[b]
        plan, leans = [], False
        for i in range(lengths[b] // page, -(-(lengths[b] + n) // page) if n else 0):
            p = row[i]
            if p < 0:
                plan.append((i, None))
                continue
            left = users[p] - count.get(p, 0)
            if users[p] > 1:
                leans = leans or count.get(p, 0) > 0
                count[p] = count.get(p, 0) + 1
            if left > 1:
                plan.append((i, p))
        want += len(plan)
        plans.append((n, plan, leans, want))
    for b, (n, plan, leans, want) in enumerate(plans):
        if want > len(free) and (plan or leans):
            granted.append(0)
            short = True
            continue
        for k, (i, old) in enumerate(plan):
            page_ = free[want - len(plan) + k]
            table[b][i] = page_
            users[page_] = 1
            if old is not None:
                users[old] -= 1
                if i == lengths[b] // page and lengths[b] % page:
                    copies.append((old, page_, lengths[b] % page))
        granted.append(n)
    return users, table, granted, copies


def compact(users, table):
    """New (users, table, used, moves)."""
    used = [p for p, n in enumerate(users) if n]
    n = len(used)
    moves = dict(zip([p for p in used if p >= n], [p for p in range(n) if not users[p]]))
    new = [0] * len(users)
    for p in used:
        new[moves.get(p, p)] = users[p]
    return new, [[moves.get(p, p) for p in row] for row in table], n, moves


# ------------------------------------------------------------------------------------------------ drafts
def verify(tokens, parents, starts, target, draft, accept, sample, max_new):
    """(kept, counts, next) as lists; parents None: a chain."""
    def weights(row):
        return [min(x, 3.4028234663852886e38) if x > 0 else 0.0 for x in row.double().tolist()]

    kept, counts, token = [], [], []
    for b in range(len(starts) - 1):
        first, n = starts[b], starts[b + 1] - starts[b]
        if n == 0 or n > max_new:
            kept.append([-1] * max_new)
            counts.append(0)
            token.append(-1)
            continue
        node, path = 0, [0]
        while True:
            p = weights(target[first + node])
            q = None if draft is None else weights(draft[first + node])
            w, mass, chosen = list(p), 1.0, None
            for i in range(1, n):
                up = i - 1 if parents is None else parents[first + i]
                if up != node or up >= i:
                    continue
                x = tokens[first + i]
                if not 0 <= x < len(w):
                    continue
                if w[x] > 0 and accept[first + i] * mass * (1.0 if q is None else q[x]) < w[x]:
                    chosen = i
                    break
                if q is None:
                    mass = max(mass - w[x], 0.0)
                    w[x] = 0.0
                else:
                    w = [max(a - mass * c, 0.0) for a, c in zip(w, q)]
                    mass = math.fsum(w)
            if chosen is None:
                break
            node = chosen
            path.append(node)
        if math.fsum(w) == 0:
            w = p
        whole, run, at = math.fsum(w), 0.0, -1
        for i, x in enumerate(w):
            run += x
            if x > 0:
                at = i
                if run > sample[b] * whole:
                    break
        kept.append(path + [-1] * (max_new - len(path)))
        counts.append(len(path))
        token.append(at)
    return kept, counts, token


# ------------------------------------------------------------------------------------------------ adapters
def adapters(x, a, b, c, starts, which, scales=None):
    """(result, bound on what a kernel may be off by) of the rows that belong to sequences; the others are NaN.

    The bound: 2^-23 for every addition of a sum in 32 bits (tensor cores truncate); the sums between the products as three 16-bit terms of
    half a step each, fp16 terms no finer than 2^-25 where the row's largest is 2^14; the result's own rounding."""
    out = torch.full(c.shape, math.nan, dtype=torch.float64)
    bound = torch.zeros(c.shape, dtype=torch.float64)
    terms = 3
    k, r = x.shape[1], a.shape[1]
    for s, w in enumerate(which):
        rows = slice(starts[s], starts[s + 1])
        base = c[rows].double()
        if not 0 <= w < len(a):
            out[rows] = base
            continue
        scale = 1.0 if scales is None else float(scales[w])
        xs, aw, bw = x[rows].double(), a[w].double(), b[w].double()
        t, far = xs @ aw.T, xs.abs() @ aw.abs().T
        off = far * (k + 72) * 2.0 ** -23 + t.abs() * H[x.dtype] ** terms
        if x.dtype == torch.float16:
            off = off + t.abs().amax(1, keepdim=True) * 2.0 ** -38 * 2
        part, reach = t @ bw.T, t.abs() @ bw.abs().T
        out[rows] = base + scale * part
        off = abs(scale) * (off @ bw.abs().T + reach * (terms * r + 32) * 2.0 ** -23) + (base.abs() + abs(scale) * part.abs()) * 2.0 ** -22
        bound[rows] = off + (out[rows].abs() + off) * H[c.dtype] + 1e-37
        if c.dtype == torch.float16:
            bound[rows] += 2.0 ** -25
    return out, bound
