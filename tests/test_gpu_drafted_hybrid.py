"""Steps of drafted trees through a Gated DeltaNet layer and the attention layer behind it: the first a level of the trees at a time, each token
from its parent's state and conv history, the second at once over the paged cache; then verification, compaction and forks, which say whose
state goes on."""

from __future__ import annotations

import random

import pytest
import torch

from draft_cases import random_tree
from gdn_cases import rel
from paged_cases import attention64, compare

pytestmark = pytest.mark.gpu
GDN = dict(key_heads=2, key_dim=32, value_heads=4, value_dim=32)


@pytest.mark.parametrize("seed", [1, 2])
def test_drafted_steps_of_a_hybrid(seed):
    """Every accepted token's GDN output is the recurrence's in 64 bits over its request's own tokens, and its attention row that of the rows before
    it: after accepted tokens anywhere in the trees, requests that go on twice and ones that end."""
    from oracle.gdn_oracle import core_inputs, recurrent_gated_delta_rule
    from tjev_amd import (draft_tree, paged_append, paged_attention, paged_compact, paged_fork, paged_tables, paged_tree_attention, verify_drafts)
    from tjev_amd.serve import gdn_decode_step, gdn_prefill
    from tjev_amd.testing import gdn_inputs

    heads, kv, dim, page, vocab, most, places = 4, 2, 32, 8, 40, 11, 4
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    # the model: token x has row x of these; the attention's q, k, v are a projection of the first layer's output, the target's distribution
    # one of both layers'
    qkv, a, b, a_log, dt_bias, w, _ = (x[0].cuda() if x.dim() == 3 else x.cuda() for x in gdn_inputs(
        batch=1, length=vocab, key_heads=2, value_heads=4, dim=32, seed=seed, style="reference"))
    width, taps = qkv.shape[1], w.shape[0]
    inner = GDN["value_heads"] * GDN["value_dim"]
    project = (torch.randn(inner, (heads + 2 * kv) * dim, generator=gen) * 2).cuda()
    readout = (torch.randn(inner + heads * dim, vocab, generator=gen) * 0.3).cuda()

    def project_rows(y):
        q, k, v = (y.reshape(len(y), inner) @ project).split((heads * dim, kv * dim, kv * dim), -1)
        return q.view(-1, heads, dim), k.view(-1, kv, dim), v.view(-1, kv, dim)

    pages = 60
    kc, vc = (torch.zeros(pages, page, kv, dim, device="cuda") for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, free, taken, shared = i32([[-1] * 12] * places), torch.randperm(pages, generator=gen).int().cuda(), i32([0]), i32([0] * pages)

    # prompts
    texts = [[rng.randrange(vocab) for _ in range(n)] for n in (13, 8, 21, 5)]
    states, convs, rows = [], [], []
    for text in texts:
        x = torch.tensor(text).cuda()
        y, s, c = gdn_prefill(qkv[x][None], a[x][None], b[x][None], a_log, dt_bias, w, torch.ones(1, len(x), dtype=torch.int32, device="cuda"),
                              chunk=16, precision="highest", **GDN)
        states.append(s), convs.append(c), rows.append(project_rows(y[0]))
    state, conv = torch.cat(states), torch.cat(convs)
    sizes = [len(x) for x in texts]
    t = paged_tables(i32([0] * places), i32(sizes), table, free, taken, page_size=page, tokens=sum(sizes))
    q, k, v = (torch.cat(x) for x in zip(*rows))
    paged_append(k, v, kc, vc, t.slots)
    paged_attention(q, kc, vc, t.block_table, t.starts, t.lengths)
    table, lengths, taken = t.block_table, t.lengths, t.taken
    cached = [list(zip(k_.cpu(), v_.cpu())) for _, k_, v_ in rows]  # of each request's tokens, the rows that were written for them
    roots = [3, 4, 5, 6]

    for n, sources in enumerate(([0, 1, 2, 3], [0, 1, 2, 0], [2, 1, -1, 3], [0, 1, 1, 3], [3, 0, 1, 2], [0, 1, 2, 3])):
        print(f"drafted step {n} of a hybrid", flush=True)
        trees = [random_tree(rng, rng.randint(1, most)) if text else [] for text in texts]
        sizes = [len(tree) for tree in trees]
        toks = [[roots[r] if i == 0 else rng.randrange(vocab) for i in range(k)] for r, k in enumerate(sizes)]
        flat, starts = torch.tensor([x for m in toks for x in m]).cuda(), [sum(sizes[:r]) for r in range(places)]
        total = len(flat)
        # the levels: the rows of each, and of their parents
        depth = []
        for tree in trees:
            depth.append([])
            for p in tree:
                depth[-1].append(0 if p < 0 else depth[-1][p] + 1)
        levels = [[(starts[r] + i, starts[r] + trees[r][i] if d else r) for r in range(places) for i, x in enumerate(depth[r]) if x == d]
                  for d in range(1 + max(x for m in depth for x in m))]
        y = torch.empty(total, GDN["value_heads"], GDN["value_dim"], device="cuda")
        after, history = torch.empty(total, *state.shape[1:], device="cuda"), torch.empty(total, taps - 1, width, device="cuda")
        for d, level in enumerate(levels):
            at, above = (torch.tensor(x).cuda() for x in zip(*level))
            x = flat[at]
            y[at], history[at], after[at] = gdn_decode_step(qkv[x], a[x], b[x], a_log, dt_bias, w, (history if d else conv)[above],
                                                            (after if d else state)[above], **GDN)
        # the attention layer, and what the target says
        parents = i32([p for tree in trees for p in tree])
        t = paged_tables(lengths, i32(sizes), table, free, taken, page_size=page, tokens=total)
        d = draft_tree(parents, t.starts, t.lengths, max_new=most)
        q, k, v = project_rows(y)
        paged_append(k, v, kc, vc, t.slots)
        out = paged_tree_attention(q, kc, vc, t.block_table, t.starts, t.lengths, d.ancestors, max_new=most)
        target = torch.softmax(torch.cat([y.flatten(1), out.flatten(1)], 1) @ readout, -1)
        # (drafts of the target's own likely tokens, so that some are accepted: a tree's tokens are known before it runs, so these numbers are 0)
        uniforms = torch.where(torch.rand(total, generator=gen) < 0.5, 0.0, torch.rand(total, generator=gen)).cuda()
        said = verify_drafts(flat, target, t.starts, uniforms, parents=parents, max_new=most)
        left = paged_compact([(kc, vc)], t.block_table, t.starts, t.lengths, said.path, said.kept)
        goes = i32(sources).long().clamp(min=0)
        f = paged_fork([(kc, vc)], t.block_table, t.lengths, i32(sources), left[goes], free, t.taken, shared, page_size=page)
        # whose state goes on: the last kept token's, of the place that the request goes on from
        last = t.starts[:-1].long() + said.path.gather(1, (said.kept.long() - 1).clamp(min=0)[:, None])[:, 0]
        last = torch.where(said.kept > 0, last, 0)
        state, conv = after[last][goes], history[last][goes]
        table, lengths, free, taken, shared = f

        for r, text in enumerate(texts):
            kept = int(said.kept[r])
            assert (kept > 0) == (sizes[r] > 0)
            if not kept:
                continue
            way = [starts[r] + i for i in said.path[r, :kept].tolist()]
            seq = text + flat[way].tolist()
            inputs = [x.cpu().double() for x in (qkv[seq][None], a[seq][None], b[seq][None], a_log, dt_bias, w)]
            want, final = recurrent_gated_delta_rule(*core_inputs(*inputs, torch.ones(1, len(seq), dtype=torch.int32), dtype=torch.float64, **GDN))[:2]
            e_out, e_state = rel(y[way].cpu(), want[0, -kept:]), rel(after[way[-1]].cpu(), final[0])
            print(f"request {r}: {kept} of {sizes[r]} kept, GDN out rel {e_out:.1e}, state rel {e_state:.1e}", flush=True)
            assert e_out <= 1e-5 and e_state <= 1e-5
            assert torch.equal(history[way[-1]], qkv[seq][1 - taps:])
            cached[r] = cached[r] + list(zip(k[way].cpu(), v[way].cpu()))
            keys, values = (torch.stack(x)[:, None] for x in zip(*cached[r]))
            want, room = attention64(q[way].cpu(), keys, values, torch.arange(len(seq), dtype=torch.int32)[None], torch.tensor([0, kept]),
                                     torch.tensor([len(seq)]))
            compare(out[way], want, room)
            texts[r], roots[r] = seq, int(said.tokens[r, kept - 1])
        texts, cached, roots = ([x[s] if s >= 0 else e for s in sources] for x, e in ((texts, []), (cached, []), (roots, 0)))
        assert lengths.tolist() == [len(x) for x in texts]
