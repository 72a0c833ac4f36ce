"""Measured operators of a served step with drafted tokens over the paged key/value cache: the ancestors and positions of
a tree of drafts, attention for that tree, the drafts' verification against the target's probabilities, the compaction of
the accepted ones, and forking, rolling back and freeing the pages that the requests hold.

``draw`` gives more cases of the ranges that the listed ones stand for: 1 to 256 requests, trees and chains of 1 to 256
tokens (the token that the last step sampled at their root), up to 16384 cached tokens per request, head dims 64, 128
and 256, groups of 1 to 8 query heads per key head, pages of 8 to 128 tokens (ones that end inside a tile among them), bf16
and fp32, vocabularies of 500 to 200000, 1 to 12 layers, 1 to 8 requests made of one. Lengths and trees come from the case
alone (where trees are the operator's values: from the seed); values, tokens and the order of the pages from the seed.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, kind, **kw):
    c = dict(kind=kind, **kw)
    return dict(name=name, **c) if name else c


def _tree(name, requests, nodes, shape, cached=1000):
    return _case(name, "tree", requests=requests, nodes=nodes, shape=shape, cached=cached)


def _attention(name, requests, cached, nodes, shape, page, heads=16, kv_heads=4, dim=256, dtype="bf16", gate=False):
    return _case(name, "attention", requests=requests, cached=cached, nodes=nodes, shape=shape, page=page, heads=heads, kv_heads=kv_heads,
                 dim=dim, dtype=dtype, gate=gate)


def _verify(name, requests, nodes, shape, vocab, dtype="fp32", drawn=False):
    return _case(name, "verify", requests=requests, nodes=nodes, shape=shape, cached=1, vocab=vocab, dtype=dtype, drawn=drawn)


def _compact(name, requests, cached, nodes, layers, page, kv_heads=4, dim=256, dtype="bf16"):
    return _case(name, "compact", requests=requests, cached=cached, nodes=nodes, shape="tree", layers=layers, page=page, kv_heads=kv_heads,
                 dim=dim, dtype=dtype)


def _fork(name, requests, cached, copies, layers, page, kv_heads=4, dim=256, dtype="bf16"):
    return _case(name, "fork", requests=requests, cached=cached, copies=copies, layers=layers, page=page, kv_heads=kv_heads, dim=dim,
                 dtype=dtype)


def listed():
    return [
        # a decode batch's trees, once a step for all layers
        _tree("tree_step", 64, 16, "tree"),
        # many requests with wide trees of very different sizes
        _tree("tree_many", 256, 250, "ragged"),
        # one interactive request's drafted tree: few rows, a cache of some thousand tokens
        _attention("attention_one", 1, 4000, 12, "tree", 16),
        # a full batch of trees over contexts of very different lengths, with the layer's output gate
        _attention("attention_batch", 32, 16384, 24, "ragged", 64, gate=True),
        # wide trees, and pages that end inside a tile
        _attention("attention_wide", 16, 12000, 250, "ragged", 24, heads=32, kv_heads=8, dim=128),
        # a small full-precision run
        _attention("attention_fp32", 3, 1500, 13, "ragged", 16, heads=8, kv_heads=2, dim=64, dtype="fp32"),
        # one request's tree, its tokens chosen (the likeliest ones), a vocabulary of odd size
        _verify("verify_one", 1, 24, "tree", 50257, dtype="bf16"),
        # a batch's chains of tokens drawn from a draft model's probabilities
        _verify("verify_drawn", 64, 6, "chain", 128000, drawn=True),
        # one request's accepted tokens to their places, in the attention layers of a small hybrid decoder
        _compact("compact_one", 1, 300, 16, 6, 16),
        # the same of a large batch with wide trees
        _compact("compact_batch", 128, 100, 60, 8, 64, kv_heads=8, dim=128),
        # after a step's verification: every request gives back the pages that its rejected tokens had, some end
        _fork("fork_rollback", 64, 8192, 1, 0, 16),
        # prompts whose answers are sampled several times each: pages shared, the last ones copied in every layer
        _fork("fork_samples", 24, 5000, 8, 6, 64),
    ]


def _spread(rng, lo, hi):
    """An integer in [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["tree", "attention", "attention", "attention", "attention", "verify", "verify", "compact", "fork", "fork"])
    shape = rng.choice(["tree", "ragged", "ragged", "chain"])
    dtype = "fp32" if rng.random() < 0.2 else "bf16"
    dim = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    requests = _spread(rng, 1, 256)
    if kind == "tree":
        return _tree(None, requests, _spread(rng, 1, min(256, 20000 // requests)), shape, _spread(rng, 1, 16384))
    if kind == "attention":  # up to 500 MB of cache, and as many rows as a large batch of wide trees has
        heads = kv * rng.choice([1, 2, 4, 5, 8])
        requests = _spread(rng, 1, 32)
        nodes = _spread(rng, 1, min(256, 2000 // requests))
        cached = _spread(rng, 1, min(16384, int(5e8 / (kv * dim * (4 if dtype == "bf16" else 8) * requests))))
        cached = min(cached, 1 + int((1e10 if dtype == "fp32" else 6e10) / (4 * requests * nodes * heads * dim)))
        return _attention(None, requests, cached, nodes, shape, page, heads, kv, dim, dtype, rng.random() < 0.5)
    if kind == "verify":
        vocab = _spread(rng, 500, 200000)
        requests = _spread(rng, 1, min(64, 8000000 // vocab))
        drawn = rng.random() < 0.5
        nodes = _spread(rng, 1, min(64, max(1, int(4.5e7 / (requests * vocab)))))
        return _verify(None, requests, nodes, "chain" if drawn else shape, vocab, "fp32" if rng.random() < 0.7 else "bf16", drawn)
    layers = rng.choice([1, 2, 4, 6, 8, 12])
    if kind == "compact":
        requests = _spread(rng, 1, 128)
        return _compact(None, requests, _spread(rng, 1, 100), _spread(rng, 1, 64), min(layers, 8), page, kv, dim, dtype)
    copies = rng.choice([1, 1, 2, 3, 4, 8])
    most = int(1.5e9 / (kv * dim * (4 if dtype == "bf16" else 8) * layers))  # tokens of the cache
    requests = _spread(rng, 1, min(64, max(1, most // (page * copies * 8))))
    return _fork(None, requests, _spread(rng, 1, max(1, min(8192, most // requests - page * copies))), copies, layers, page, kv, dim, dtype)


# --------------------------------------------------------------------------- the case's lengths and trees
def _sizes(case):
    """(cached, new) per request: alike (tree, chain), or ragged, cached lengths and trees of very different sizes."""
    rng = random.Random(f"{case['requests']} {case['cached']} {case['nodes']} {case['shape']}")
    out = []
    for _ in range(case["requests"]):
        c, n = case["cached"], case["nodes"]
        if case["shape"] == "ragged":
            c, n = _spread(rng, max(1, c // 32), c), _spread(rng, max(1, n // 16), n)
        out.append((c, n))
    return out


def _parents(case, seed=0):
    """Every request's parents, numbers within the request: -1 for its first token; a chain, or levels of 1 to 8 tokens, each
    drafted behind one of the level before, a level's parents in order."""
    rng = random.Random(f"{case['requests']} {case['nodes']} {case['shape']} trees {seed}")
    out = []
    for _, n in _sizes(case):
        p, level = [-1], [0]
        while len(p) < n:
            wide = 1 if case["shape"] == "chain" else min(n - len(p), rng.randint(1, 8))
            p += sorted(rng.choice(level) for _ in range(wide))
            level = list(range(len(p) - wide, len(p)))
        out.append(p)
    return out


def _ranks(parents):
    """How many siblings stand before each token."""
    seen, out = {}, []
    for p in parents:
        out.append(seen.get(p, 0))
        seen[p] = out[-1] + 1
    return out


def _chosen(case):
    """The accepted tokens of the compaction's requests: a way down each tree, its first step the likeliest token (which stays in
    its place), no further one a token whose place another accepted one takes."""
    rng = random.Random(f"{case['requests']} {case['nodes']} chosen")
    out = []
    for p in _parents(case):
        way = [0]
        while True:
            below = [i for i, q in enumerate(p) if q == way[-1]]
            if len(way) == 1:
                below = below[:1]
            if not below or rng.random() < 0.15:
                break
            way.append(rng.choice(below))
        while any(j != i < len(way) for j, i in enumerate(way)):
            way.pop()
        out.append(way)
    return out


def _goes_on(case):
    """(lengths, sources, keep) of the forks: with one copy each, the requests go on without a few of their last tokens and every
    sixteenth ends; else each goes on `copies` times, all of it."""
    rng = random.Random(f"{case['requests']} {case['cached']} {case['copies']} forks")
    lens = [_spread(rng, max(1, case["cached"] // 16), case["cached"]) for _ in range(case["requests"])]
    if case["copies"] > 1:
        src = [b for b in range(case["requests"]) for _ in range(case["copies"])]
        return lens, src, [lens[b] for b in src]
    src = [-1 if b % 16 == 7 else b for b in range(case["requests"])]
    return lens, src, [max(0, n - rng.randint(0, 20)) for n in lens]


def _pages(tokens, page):
    return -(-tokens // page)


# --------------------------------------------------------------------------- inputs
def _rn(gen, *shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype) * std


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    s = {"case": dict(case)}
    kind = case["kind"]
    if kind == "fork":
        return _fork_inputs(case, gen, rng, s)
    sizes, parents = _sizes(case), _parents(case)
    if kind == "tree":  # these are its values
        sizes, parents = [(c + int(rng.integers(0, 1000)), n) for c, n in sizes], _parents(case, int(seed))
    s["max_new"] = case["nodes"]
    s["starts"] = _i32(np.concatenate([[0], np.cumsum([n for _, n in sizes])]))
    s["lengths"] = _i32([c + n for c, n in sizes])
    s["parents"] = _i32([p for tree in parents for p in tree])
    if kind == "tree":
        s["trees"], s["cached"] = parents, [c for c, _ in sizes]
        return s
    if kind == "verify":
        return _verify_inputs(case, gen, s, sizes, parents)
    page, dt, hk, d = case["page"], DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    wanted = [_pages(c + n, page) for c, n in sizes]
    pool = sum(wanted) + 5
    order, at = rng.permutation(pool).astype(np.int32), 0
    table = np.full((len(sizes), max(wanted) + 3), -1, np.int32)  # a request may grow further
    for b, n in enumerate(wanted):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"] = torch.from_numpy(table).cuda()
    if kind == "attention":
        s["k_cache"], s["v_cache"] = (_rn(gen, pool, page, hk, d, dtype=dt) for _ in range(2))
        tokens = sum(n for _, n in sizes)
        qg = _rn(gen, tokens, case["heads"], 2 * d, dtype=dt)  # the projection's rows: each head's query beside its gate
        s["q"], s["gate"] = qg[..., :d], qg[..., d:] if case["gate"] else None
        s["ancestors"] = torch.from_numpy(_ancestors(parents, case["nodes"])).cuda()
        s["most_keys"] = max(c + n for c, n in sizes)  # the scheduler's own count
        return s
    s["layers"] = _rn(gen, case["layers"], 2, pool, page, hk, d, dtype=dt)
    s["caches"] = [(x[0], x[1]) for x in s["layers"]]
    chosen = _chosen(case)
    path = np.full((len(sizes), case["nodes"]), -1, np.int32)
    for b, way in enumerate(chosen):
        path[b, :len(way)] = way
    s["path"], s["kept"] = torch.from_numpy(path).cuda(), _i32([len(way) for way in chosen])
    return s


def _ancestors(parents, nodes):
    """Bit j of a token's row: the request's token j is the token or one of its ancestors (64 bits a word)."""
    words = _pages(nodes, 64)
    out = np.zeros((sum(len(t) for t in parents), words), np.uint64)
    at = 0
    for tree in parents:
        for i, p in enumerate(tree):
            if p >= 0:
                out[at + i] = out[at + p]
            out[at + i, i // 64] |= np.uint64(1 << (i % 64))
        at += len(tree)
    return out.view(np.int64)


def _verify_inputs(case, gen, s, sizes, parents):
    """A target sure of some tokens and not of others, and a draft near it."""
    n, v = sum(k for _, k in sizes), case["vocab"]
    at = np.concatenate([np.full(len(t), int(b)) for t, b in zip(parents, np.cumsum([0] + [len(t) for t in parents]))])
    above = torch.from_numpy(np.maximum(0, np.array([p for t in parents for p in t])) + at).cuda()  # the row of each token's parent
    sharp = torch.rand(n, 1, generator=gen, device="cuda") * 3 + 1.5
    logits = _rn(gen, n, v, dtype=torch.float32) * sharp
    s["target_probs"] = torch.softmax(logits, -1).to(DTYPES[case["dtype"]])
    logits = logits[above]
    logits += _rn(gen, n, v, dtype=torch.float32, std=0.7)
    if case["drawn"]:
        q = torch.softmax(logits, -1)
        s["tokens"] = torch.multinomial(q, 1, generator=gen)[:, 0].int()
        s["draft_probs"] = q.to(DTYPES[case["dtype"]])
    else:
        rank = [r for t in parents for r in _ranks(t)]
        top = torch.topk(logits, max(rank) + 1, dim=-1).indices
        s["tokens"] = top.gather(1, torch.tensor(rank, device="cuda")[:, None])[:, 0].int()
        s["draft_probs"] = None
    if case["shape"] == "chain":
        s["parents"] = None
    s["uniforms"] = torch.rand(n, generator=gen, device="cuda")
    return s


def _fork_inputs(case, gen, rng, s):
    page, dt = case["page"], DTYPES[case["dtype"]]
    lens, src, keep = _goes_on(case)
    held = [_pages(n, page) for n in lens]
    pool = sum(held) + len(src) + 7
    order, at = rng.permutation(pool).astype(np.int32), 0
    table = np.full((len(lens), max(held) + 3), -1, np.int32)
    shared = np.zeros(pool, np.int32)
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
        if b % 3 == 2:  # the same system prompt as the request before it
            both = min(lens[b - 1], lens[b]) // (2 * page)
            table[b, :both] = table[b - 1, :both]
            shared[table[b, :both]] += 1
    s["table"], s["shared"] = torch.from_numpy(table).cuda(), torch.from_numpy(shared).cuda()
    gone = np.setdiff1d(order[:at], table)  # pages that sharing left unused stand on the list too
    free = np.concatenate([order[:at][~np.isin(order[:at], gone)], gone, order[at:]])
    s["free"], s["taken"] = torch.from_numpy(free).cuda(), _i32([at - len(gone)])
    s["lengths"], s["sources"], s["keep"] = _i32(lens), _i32(src), _i32(keep)
    s["layers"] = _rn(gen, case["layers"], 2, pool, page, case["kv_heads"], case["dim"], dtype=dt) if case["layers"] else None
    s["caches"] = [(x[0], x[1]) for x in s["layers"]] if case["layers"] else []
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# --------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from tjev_amd import draft_tree, paged_compact, paged_fork, paged_tree_attention, verify_drafts

    case = s["case"]
    if case["kind"] == "tree":
        t = draft_tree(s["parents"], s["starts"], s["lengths"], max_new=s["max_new"])
        return {"ancestors": t.ancestors, "positions": t.positions}
    if case["kind"] == "attention":
        return {"out": paged_tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["lengths"], s["ancestors"],
                                            gate=s["gate"], max_new=s["max_new"])}
    if case["kind"] == "verify":
        v = verify_drafts(s["tokens"], s["target_probs"], s["starts"], s["uniforms"], parents=s["parents"], draft_probs=s["draft_probs"],
                          max_new=s["max_new"])
        return {"tokens": v.tokens, "path": v.path, "kept": v.kept}
    if case["kind"] == "compact":
        lengths = paged_compact(s["caches"], s["table"], s["starts"], s["lengths"], s["path"], s["kept"])
        return {"lengths": lengths, "layers": s["layers"]}
    f = paged_fork(s["caches"], s["table"], s["lengths"], s["sources"], s["keep"], s["free"], s["taken"], s["shared"], page_size=case["page"])
    return {"table": f.block_table, "lengths": f.lengths, "free": f.free_pages, "taken": f.taken, "shared": f.shared,
            **({"layers": s["layers"]} if case["layers"] else {})}


def _run_plain(s):
    return {"tree": _plain_tree, "attention": _plain_attention, "verify": _plain_verify, "compact": _plain_compact, "fork": _plain_fork}[
        s["case"]["kind"]](s)


def _rows(s, n):
    """Of every row of the batch: its request and its number within it."""
    t = torch.arange(n, device=s["starts"].device)
    b = torch.searchsorted(s["starts"][1:].long(), t, right=True).clamp(max=len(s["starts"]) - 2)
    return b, t - s["starts"].long()[b]


def _padded(s, x, most, fill):
    """x [N] as [B, most], one row for each request."""
    b, j = _rows(s, x.shape[0])
    out = torch.full((len(s["starts"]) - 1, most), fill, dtype=x.dtype, device=x.device)
    out[b, j] = x
    return out


def _plain_tree(s):
    most = s["max_new"]
    b, j = _rows(s, s["parents"].shape[0])
    up = _padded(s, s["parents"], most, -1).long()  # [B, most]
    me = torch.arange(most, device=up.device)
    step = (up[..., None] == me).float()  # [B, i, j]: j is i's parent
    seen = torch.eye(most, device=up.device) + step
    for _ in range(max(1, (most - 1).bit_length())):  # all ancestors: twice as many steps up each round
        step = torch.matmul(step, step)
        seen = seen + torch.matmul(seen, step)
    seen = seen[b, j] > 0  # [N, most]
    words = _pages(most, 64)
    bits = torch.nn.functional.pad(seen, (0, 64 * words - most)).view(-1, words, 64)
    one = torch.ones(64, dtype=torch.int64, device=up.device) << torch.arange(64, device=up.device)
    first = (s["lengths"] - s["starts"][1:] + s["starts"][:-1])[b]
    return {"ancestors": torch.where(bits, one, 0).sum(-1), "positions": first + (seen.sum(-1) - 1).int()}


def _plain_attention(s):
    case = s["case"]
    hk, d, most, length = case["kv_heads"], case["dim"], s["max_new"], s["most_keys"]
    g, n = case["heads"] // hk, s["q"].shape[0]
    b, j = _rows(s, n)
    t = torch.arange(length, device=b.device)
    page = s["table"].long()[:, t // case["page"]].clamp(min=0)  # [B, L]
    k, v = (x[page, t % case["page"]].float().permute(0, 2, 1, 3).contiguous() for x in (s["k_cache"], s["v_cache"]))  # [B, Hk, L, D]
    q = torch.zeros(len(page), hk, most, g, d, device=b.device)
    q[b, :, j] = s["q"].float().view(n, hk, g, d)
    w = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).mul_(d ** -0.5).view(len(page), hk, most, g, length)
    first = (s["lengths"] - s["starts"][1:] + s["starts"][:-1]).long()
    bit = t[None] - first[b][:, None]  # [N, L]
    word = s["ancestors"].gather(1, (bit // 64).clamp(0, s["ancestors"].shape[1] - 1))
    seen = (bit < 0) | ((bit < most) & ((word >> (bit % 64)) & 1 > 0) & (t < s["lengths"].long()[b][:, None]))
    mask = torch.zeros(len(page), most, length, dtype=torch.bool, device=b.device)
    mask[b, j] = seen
    w.masked_fill_(~mask[:, None, :, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-1e30))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.flatten(2, 3), v).view(len(page), hk, most, g, d) / torch.where(total > 0, total, 1.0)
    o = o[b, :, j].reshape(n, case["heads"], d)
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    return {"out": o.to(s["q"].dtype)}


def _plain_verify(s):
    most, start, p = s["max_new"], s["starts"].long()[:-1], s["target_probs"]
    rows, vocab = p.shape
    up = s["parents"]
    if up is None:
        up = _rows(s, rows)[1].int() - 1
    token, up, u = (_padded(s, x, most, fill).to(t) for x, fill, t in (
        (s["tokens"], -1, torch.int64), (up, -2, torch.int64), (s["uniforms"], 0.0, torch.float64)))  # [B, most]
    row = start[:, None] + torch.arange(most, device=p.device)
    above = (start[:, None] + up).clamp(0, rows - 1)
    pt = torch.where(up >= 0, p[above, token.clamp(min=0)].double(), 0.0)  # the target's, of each token behind its parent
    alike = (up[:, :, None] == up[:, None]) & (torch.arange(most, device=p.device)[:, None] > torch.arange(most, device=p.device))
    again = (alike & (token[:, :, None] == token[:, None])).any(-1)
    pt = torch.where(again, 0.0, pt)
    if s["draft_probs"] is None:
        left = 1 - torch.where(alike, pt[:, None], 0.0).sum(-1)  # what the siblings before it leave
        good = (pt > 0) & (u * left.clamp(min=0) < pt)
    else:
        good = (pt > 0) & (u * s["draft_probs"][row.clamp(max=rows - 1), token.clamp(min=0)].double() < pt)
    me = torch.arange(most, device=p.device)
    child = good[:, None] & (up[:, None] == me[:, None])  # [B, node, token]
    after = torch.where(child.any(-1), child.int().argmax(-1), -1)  # the first accepted one behind each
    at, path = torch.zeros_like(start), []
    alive = torch.ones_like(start, dtype=torch.bool)
    for _ in range(most):  # a level a time
        path.append(torch.where(alive, at, -1))
        nxt = after.gather(1, at[:, None])[:, 0]
        alive = alive & (nxt >= 0)
        at = torch.where(alive, nxt, at)
    path = torch.stack(path, 1)
    kept = (path >= 0).sum(1)
    full = p[start + at].double()
    below = up == at[:, None]  # rejected ones
    rest = full.clone()
    if s["draft_probs"] is None:
        b, i = torch.where(below & (token >= 0))
        rest[b, token[b, i]] = 0.0
    else:
        last = (start + at + 1).clamp(max=rows - 1)
        rest = torch.where(below.any(1)[:, None], rest - s["draft_probs"][last].double(), rest).clamp(min=0)
    rest = torch.where((rest.sum(-1) > 0)[:, None], rest, full)
    sums = torch.cumsum(rest, -1)
    new = (sums <= u[:, :1] * sums[:, -1:]).sum(-1)
    new = torch.minimum(new, vocab - 1 - (rest > 0).flip(1).int().argmax(-1))
    out = torch.where(path >= 0, token.gather(1, path.clamp(min=0)), -1).roll(-1, 1)
    out[:, -1] = -1
    out.scatter_(1, (kept - 1)[:, None], new[:, None])
    return {"tokens": out.int(), "path": path.int(), "kept": kept.int()}


def _plain_compact(s):
    case = s["case"]
    first = (s["lengths"] - s["starts"][1:] + s["starts"][:-1]).long()
    j = torch.arange(s["path"].shape[1], device=first.device)
    b, j = torch.where((j < s["kept"][:, None]) & (s["path"] > j))
    flat = s["layers"].view(2 * case["layers"], -1, case["kv_heads"], case["dim"])
    slot = lambda t: s["table"][b, t // case["page"]].long() * case["page"] + t % case["page"]  # noqa: E731
    flat[:, slot(first[b] + j)] = flat[:, slot(first[b] + s["path"][b, j])]
    return {"lengths": (first + s["kept"]).int(), "layers": s["layers"]}


def _plain_fork(s):
    case, table, shared = s["case"], s["table"], s["shared"]
    page, width, pages = case["page"], table.shape[1], shared.shape[0]
    held = ((s["lengths"].long() + page - 1) // page)[:, None]
    col = torch.arange(width, device=table.device)
    src = s["sources"].long()
    keep = torch.where(src >= 0, torch.minimum(s["keep"].long(), s["lengths"].long()[src.clamp(min=0)]), 0)
    mine = ((keep + page - 1) // page)[:, None]
    new = torch.where(col < mine, table[src.clamp(min=0)], -1)
    old = table[col < held].long()  # in order
    count = lambda x: torch.zeros(pages, dtype=torch.int64, device=table.device).index_add_(0, x, torch.ones_like(x))  # noqa: E731
    before, after = count(old), count(new[new >= 0].long())
    holders = shared + 1 - before + after
    # a last page with room in it has one holder: the first of them where only such ones are left, else a copy for each
    i = torch.where(keep % page > 0)[0]
    at = keep[i] // page
    last = new[i, at].long()
    lowest = torch.full((pages,), len(src), device=table.device).scatter_reduce_(0, last, i, "amin")
    moves = ~((holders[last] == count(last)[last]) & (lowest[last] == i))
    i, at, last = i[moves], at[moves], last[moves]
    holders = torch.where(before > 0, holders - count(last), -1)
    order = torch.full((pages,), old.shape[0], device=table.device).scatter_reduce_(0, old, torch.arange(old.shape[0], device=table.device), "amin")
    gone = torch.where(holders == 0)[0]
    gone = gone[torch.argsort(order[gone])]
    free, taken = s["free"].clone(), s["taken"].long().clamp(max=len(s["free"]))
    low = taken - len(gone)
    free[low + torch.arange(len(gone), device=table.device)] = gone.int()
    want = low + torch.arange(len(i), device=table.device)
    fresh = torch.where(want < len(free), free[want.clamp(max=len(free) - 1)], -1)
    new[i, at] = fresh
    shared = torch.where(holders > 0, holders - 1, torch.where(holders == 0, 0, shared)).int()
    got = fresh >= 0
    shared[fresh[got].long()] = 0
    out = {"table": new, "lengths": keep.int(), "free": free, "taken": (low + len(i)).int(), "shared": shared}
    if case["layers"]:
        x, place = torch.where(torch.arange(page, device=table.device) < (keep[i] % page)[:, None] * got[:, None])
        s["layers"][:, :, fresh[x].long(), place] = s["layers"][:, :, last[x], place]
        out["layers"] = s["layers"]
    return out


# --------------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "fork":
        lens, src, keep = _goes_on(case)
        row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * (2 if case["dtype"] == "bf16" else 4)
        read, wrote = sum(_pages(n, case["page"]) for n in lens), sum(_pages(k, case["page"]) for b, k in zip(src, keep) if b >= 0)
        seen, copied = set(), 0
        for b, k in zip(src, keep):  # the tokens of last pages that more than one goes on with
            copied += k % case["page"] if b in seen else 0
            seen.add(b)
        return {"bytes": 4 * (read + wrote + 4 * len(src)) + 2 * copied * row, "flops": 0.0}
    sizes = _sizes(case)
    tokens = sum(n for _, n in sizes)
    if kind == "tree":
        return {"bytes": tokens * (4 + 4 + 8 * _pages(case["nodes"], 64)) + 8 * len(sizes), "flops": 0.0}
    e = 2 if case["dtype"] == "bf16" else 4
    if kind == "verify":  # the rows that the last tokens are drawn from, and the drafts' own numbers
        rows = 2 if case["drawn"] else 1
        return {"bytes": len(sizes) * rows * case["vocab"] * e + tokens * (4 + 4 + 4 + rows * e) + len(sizes) * (8 * case["nodes"] + 4),
                "flops": 2.0 * len(sizes) * rows * case["vocab"]}
    hk, d = case["kv_heads"], case["dim"]
    if kind == "compact":
        moved = sum(j != i for way in _chosen(case) for j, i in enumerate(way))
        return {"bytes": 2 * moved * 2 * case["layers"] * hk * d * e + sum(4 * len(way) for way in _chosen(case)) + 12 * len(sizes), "flops": 0.0}
    pairs = sum(n * c for c, n in sizes)
    for tree in _parents(case):
        depth = []
        for p in tree:
            depth.append(1 + (depth[p] if p >= 0 else 0))
        pairs += sum(depth)
    rows = tokens * case["heads"] * d * e
    return {"bytes": 2 * sum(c + n for c, n in sizes) * hk * d * e + rows * (3 if case["gate"] else 2) +
            tokens * 8 * _pages(case["nodes"], 64) + 4 * sum(_pages(c + n, case["page"]) for c, n in sizes), "flops": 4.0 * pairs * case["heads"] * d}


# --------------------------------------------------------------------------- the same from the definitions, in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "fork":
        return _exact_fork(case, s)
    sizes, parents = _sizes(case), _parents(case)
    starts = np.concatenate([[0], np.cumsum([n for _, n in sizes])])
    if case["kind"] == "tree":
        positions = []
        for c, tree in zip(s["cached"], s["trees"]):
            depth = []
            for p in tree:
                depth.append(0 if p < 0 else depth[p] + 1)
            positions += [c + x for x in depth]
        return {"ancestors": torch.from_numpy(_ancestors(s["trees"], case["nodes"])), "positions": torch.tensor(positions, dtype=torch.int32)}
    if case["kind"] == "verify":
        return _exact_verify(case, s, starts, parents)
    if case["kind"] == "compact":
        table, page, layers = s["table"].cpu().numpy(), case["page"], s["layers"].clone()
        for b, way in enumerate(_chosen(case)):
            c = sizes[b][0]
            for j, i in enumerate(way):
                to, of = (divmod(c + x, page) for x in (j, i))
                layers[:, :, int(table[b, to[0]]), to[1]] = layers[:, :, int(table[b, of[0]]), of[1]]
        return {"lengths": torch.tensor([c + len(way) for (c, _), way in zip(sizes, _chosen(case))], dtype=torch.int32), "layers": layers.double()}
    g, d, page = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (c, n) in enumerate(sizes):
        at, where = int(starts[b]), torch.arange(c + n, device="cuda")
        mask = torch.zeros(n, n, dtype=torch.bool)
        for i, p in enumerate(parents[b]):
            if p >= 0:
                mask[i] = mask[p]
            mask[i, i] = True
        mask = torch.cat([torch.ones(n, c, dtype=torch.bool), mask], 1).cuda()
        ids = s["table"][b].long()[where // page]
        for h in range(case["kv_heads"]):
            k, v = (x[ids, where % page, h].double() for x in (s["k_cache"], s["v_cache"]))
            for j in range(h * g, h * g + g):
                w = (s["q"][at:at + n, j].double() / math.sqrt(d)) @ k.t()
                o = torch.softmax(w.masked_fill(~mask, -math.inf), -1) @ v
                out[at:at + n, j] = o / (1 + torch.exp(-s["gate"][at:at + n, j].double())) if case["gate"] else o
    return {"out": out}


def _exact_verify(case, s, starts, parents):
    """Request by request, token by token."""
    most = case["nodes"]
    tokens, u = s["tokens"].cpu().numpy(), s["uniforms"].double().cpu().numpy()
    out, path, kept = np.full((len(parents), most), -1, np.int32), np.full((len(parents), most), -1, np.int32), []
    for b, tree in enumerate(parents):
        at, node, way, says = int(starts[b]), 0, [0], []
        while True:
            p = s["target_probs"][at + node].double().cpu().numpy()
            rest, left, nxt = p.copy(), 1.0, None
            for c in [i for i, up in enumerate(tree) if up == node]:
                x = int(tokens[at + c])
                q = None if s["draft_probs"] is None else s["draft_probs"][at + c].double().cpu().numpy()
                if rest[x] > 0 and u[at + c] * (max(left, 0.0) if q is None else q[x]) < rest[x]:
                    nxt = c
                    break
                if q is None:
                    left -= rest[x]
                    rest[x] = 0.0
                else:
                    rest = np.maximum(rest - q, 0.0)
            if nxt is None:
                break
            says.append(int(tokens[at + nxt]))
            way.append(nxt)
            node = nxt
        rest = rest if rest.sum() > 0 else p
        sums = np.cumsum(rest)
        new = min(int(np.searchsorted(sums, u[at] * sums[-1], side="right")), int(np.nonzero(rest > 0)[0][-1]))
        out[b, :len(way)], path[b, :len(way)] = says + [new], way
        kept.append(len(way))
    return {"tokens": torch.from_numpy(out), "path": torch.from_numpy(path), "kept": torch.tensor(kept, dtype=torch.int32)}


def _exact_fork(case, s):
    """The scheduler's walk with the holders of every page in a list."""
    lens, src, keep = _goes_on(case)
    page, table = case["page"], s["table"].cpu().numpy()
    shared, free = s["shared"].cpu().numpy().copy(), s["free"].cpu().numpy().copy()
    taken, width = int(s["taken"]), table.shape[1]
    holders = {}
    old = [int(p) for b, n in enumerate(lens) for p in table[b, :_pages(n, page)]]
    for p in old:
        holders.setdefault(p, int(shared[p]) + 1)
    for p in old:
        holders[p] -= 1
    new, lengths, open_ = np.full((len(src), width), -1, np.int32), [], {}
    for i, b in enumerate(src):
        k = min(keep[i], lens[b]) if b >= 0 else 0
        lengths.append(k)
        for j in range(_pages(k, page)):
            new[i, j] = table[b, j]
            holders[int(table[b, j])] += 1
        if k % page:
            open_.setdefault(int(table[b, k // page]), []).append(i)
    stays = {p: rows[0] for p, rows in open_.items() if holders[p] == len(rows)}
    copies = []
    for i, k in enumerate(lengths):
        if k % page and stays.get(int(new[i, k // page])) != i:
            copies.append((i, k // page, int(new[i, k // page])))
    for _, _, p in copies:
        holders[p] -= 1
    gone = [p for p in dict.fromkeys(old) if holders[p] == 0]
    for p, n in holders.items():
        shared[p] = max(0, n - 1)
    at = taken - len(gone)
    free[at:taken] = gone
    layers = s["layers"].clone() if case["layers"] else None
    for i, j, p in copies:
        new[i, j] = free[at] if at < len(free) else -1
        if new[i, j] >= 0:
            shared[new[i, j]] = 0
            if layers is not None:
                layers[:, :, int(new[i, j]), :lengths[i] % page] = layers[:, :, p, :lengths[i] % page]
        at += 1
    out = {"table": torch.from_numpy(new), "lengths": torch.tensor(lengths, dtype=torch.int32), "free": torch.from_numpy(free),
           "taken": torch.tensor([at], dtype=torch.int32), "shared": torch.from_numpy(shared)}
    if layers is not None:
        out["layers"] = layers.double()
    return out
