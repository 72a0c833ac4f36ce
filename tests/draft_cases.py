"""Plain forms of the drafted step's operators for the tests, on the CPU: lists, loops and 64 bits."""

from __future__ import annotations

import torch

from paged_cases import HALF_STEP


def starts_of(sizes, front=0):
    out = [front]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def rows_of(starts, b, total):
    """Rows of request b within the batch, whatever the starts hold."""
    s0 = min(max(0, int(starts[b])), total)
    return s0, max(s0, min(int(starts[b + 1]), total)) - s0


def tree_walk(parents, starts, lengths, max_new):
    """(ancestors: a set of numbers for each row, positions)."""
    sets, positions = [set() for _ in parents], [0] * len(parents)
    for b in range(len(lengths)):
        s0, n = rows_of(starts, b, len(parents))
        first = max(0, int(lengths[b]) - (int(starts[b + 1]) - int(starts[b])))
        for i in range(min(n, max_new)):
            p = int(parents[s0 + i])
            sets[s0 + i] = {i} | (sets[s0 + p] if 0 <= p < i else set())
            positions[s0 + i] = first + len(sets[s0 + i]) - 1
    return sets, positions


def bits_of(sets, words):
    """The sets as ancestors [N, words] int64."""
    out = torch.zeros(len(sets), words, dtype=torch.int64)
    for r, s in enumerate(sets):
        for j in s:
            if j < 64 * words:
                out[r, j // 64] |= (1 << j % 64) - (1 << 64 if j % 64 == 63 else 0)
    return out


def random_tree(rng, n, kind="tree"):
    """Parents of n tokens: a chain, all behind the root, levels of a few tokens, anything before it, or several roots."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "any":
        return [-1] + [rng.randrange(i) for i in range(1, n)]
    if kind == "roots":
        return [rng.choice([-1, i - 1, i, i + 3, -5, rng.randrange(i) if i else -1]) for i in range(n)]
    p, level = [-1], [0]
    while len(p) < n:
        wide = min(n - len(p), rng.randint(1, 6))
        p += [rng.choice(level) for _ in range(wide)]
        level = list(range(len(p) - wide, len(p)))
    return p[:n]


def tree_attention64(q, k_cache, v_cache, block_table, starts, lengths, ancestors, scale=None, gate=None):
    """(out, room) as paged_cases.attention64 gives them: each row over the keys before its request's new tokens and those that its
    bits name."""
    n_rows, heads, dim = q.shape
    pages, page, kv, _ = k_cache.shape
    scale = dim ** -0.5 if scale is None else scale
    out, room = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    half = HALF_STEP[q.dtype]
    words = ancestors.tolist()
    for b in range(block_table.shape[0]):
        s0, n = rows_of(starts, b, n_rows)
        length = int(lengths[b])
        first = length - (int(starts[b + 1]) - int(starts[b]))
        places = [(int(block_table[b, t // page]), t % page) for t in range(min(max(0, length), block_table.shape[1] * page))]
        for j in range(n):
            w = words[s0 + j]
            seen = [p for t, p in enumerate(places)
                    if 0 <= p[0] < pages and (t < first or (t - first < 64 * len(w) and w[(t - first) // 64] >> (t - first) % 64 & 1))]
            if not seen:
                continue
            ip, io = (torch.tensor(x) for x in zip(*seen))
            for h in range(heads):
                k, v = k_cache[ip, io, h * kv // heads].double(), v_cache[ip, io, h * kv // heads].double()
                x = q[s0 + j, h].double()
                p = torch.softmax(scale * (k @ x), 0)
                o, a = p @ v, p @ v.abs()
                # as in attention64: scores off by delta, weights by 4 delta, the sums over the keys, the weights' rounding
                delta = (dim + 8) * 2.0 ** -24 * abs(scale) * float((k.abs() @ x.abs()).max())
                r = a * (4 * delta + (len(seen) + 64) * 2.0 ** -24 + 2.0 ** -20 + (half if q.dtype == torch.bfloat16 else 0.0))
                if gate is not None:
                    sg = torch.sigmoid(gate[s0 + j, h].double())
                    o, r = o * sg, r * sg + 2.0 ** -21 * (o * sg).abs()
                out[s0 + j, h], room[s0 + j, h] = o, r + half * (o.abs() + r)
    return out, room


def clean(x):
    """What is no positive finite number counts as 0, in 64 bits."""
    x = x.double()
    return torch.where((x > 0) & torch.isfinite(x), x, 0.0)


def verify_walk(tokens, target, starts, uniforms, parents, draft, max_new):
    """(tokens, path, kept) as lists, request by request, child by child."""
    vocab, total = target.shape[1], len(tokens)
    outs, paths, kepts = [], [], []
    for b in range(len(starts) - 1):
        s0, real = rows_of(starts, b, total)
        n, way, says, node = min(real, max_new), [0], [], 0
        if not n:
            outs.append([-1] * max_new), paths.append([-1] * max_new), kepts.append(0)
            continue
        up = [(int(parents[s0 + i]) if parents is not None else i - 1) for i in range(n)]
        while True:
            whole = clean(target[s0 + node])
            rest, left, nxt = whole.clone(), 1.0, None
            for c in [i for i in range(node + 1, n) if up[i] == node]:
                x, u = int(tokens[s0 + c]), float(uniforms[s0 + c])
                px = float(rest[x]) if 0 <= x < vocab else 0.0
                bar = max(left, 0.0) if draft is None else (float(clean(draft[s0 + c])[x]) if 0 <= x < vocab else 1.0)
                if px > 0 and u * bar < px:
                    nxt = c
                    break
                if draft is None:
                    left -= px
                    if 0 <= x < vocab:
                        rest[x] = 0.0
                else:
                    rest = (rest - clean(draft[s0 + c])).clamp(min=0.0)
            if nxt is None:
                break
            way.append(nxt), says.append(int(tokens[s0 + nxt]))
            node = nxt
        if not float(rest.sum()) > 0:
            rest = whole
        sums, u = torch.cumsum(rest, 0), float(uniforms[s0])
        over = torch.nonzero(sums > max(0.0, u) * sums[-1])
        some = torch.nonzero(rest > 0)
        says.append(-1 if not len(some) else min(int(over[0]), int(some[-1])) if len(over) else int(some[-1]))
        outs.append((says + [-1] * max_new)[:max_new]), paths.append((way + [-1] * max_new)[:max_new]), kepts.append(len(way))
    return outs, paths, kepts


def compact_walk(caches, table, starts, lengths, path, kept):
    """The moves one after the other, in place; the lengths left."""
    out = []
    for b in range(table.shape[0]):
        n = max(0, int(starts[b + 1]) - int(starts[b]))
        first, count = int(lengths[b]) - n, min(max(0, int(kept[b])), path.shape[1], n)
        out.append(max(0, first + count))
        for j in range(count if first >= 0 else 0):
            f = int(path[b, j])
            if not j < f < n:
                continue
            for pair in caches:
                for c in pair:
                    pages, page = c.shape[:2]
                    to, of = ((int(table[b, t // page]) if t // page < table.shape[1] else -1, t % page) for t in (first + j, first + f))
                    if 0 <= to[0] < pages and 0 <= of[0] < pages:
                        c[to] = c[of].clone()
    return out


def fork_walk(caches, table, lengths, sources, keep, free, taken, shared, page):
    """(table, lengths, free, taken, shared) as lists, the caches' copies in place: every page's holders counted by hand."""
    width, pages = len(table[0]), len(shared)
    count = lambda n: min(width, -(-n // page))  # noqa: E731
    free, shared = list(free), list(shared)
    taken = min(max(0, taken), len(free))
    entries = [p for b, n in enumerate(lengths) for p in table[b][:count(max(0, n))] if 0 <= p < pages]
    holders = {p: shared[p] + 1 for p in entries}
    for p in entries:
        holders[p] -= 1
    new, left, writers = [], [], {}
    for i, b in enumerate(sources):
        on = 0 <= b < len(table)
        k = max(0, lengths[b]) if on else 0
        k = min(k, max(0, keep[i])) if keep is not None else k
        new.append([table[b][j] if j < count(k) else -1 for j in range(width)] if on else [-1] * width)
        left.append(k)
        for p in new[-1][:count(k)]:
            if 0 <= p < pages:
                holders[p] += 1
        if k % page and k // page < width and 0 <= new[-1][k // page] < pages:
            writers.setdefault(new[-1][k // page], []).append(i)
    copies = []
    for i, k in enumerate(left):
        p = new[i][k // page] if k % page and k // page < width else -1
        if 0 <= p < pages and not (holders[p] == len(writers[p]) and writers[p][0] == i):
            copies.append((i, p))
    for _, p in copies:
        holders[p] -= 1
    back = [p for p in dict.fromkeys(entries) if holders[p] == 0]
    for p, n in holders.items():
        shared[p] = max(0, n - 1)
    back = back[:taken]
    at = taken - len(back)
    free[at:taken] = back
    for i, p in copies:
        got = free[at] if at < len(free) else -1
        at += 1
        got = got if 0 <= got < pages else -1
        new[i][left[i] // page] = got
        if got >= 0:
            shared[got] = 0
            for pair in caches:
                for c in pair:
                    c[got, :left[i] % page] = c[p, :left[i] % page].clone()
    return new, left, free, at, shared
