"""Drafting as a server does it: several sequences of a paged cache, one of them forked from another, take steps of a drafted tree each — mask, attention, verification, accepted rows —
and end with the tokens and the cache rows that one token at a time gives.  The model is one attention layer whose queries, keys and values are sums of a token's row and a position's,
so that a cache row is the same numbers whichever step writes it."""
import pytest
import torch

from leopard_b200 import ops
from oracle import draft as O

gpu = pytest.mark.gpu
BF16 = torch.bfloat16
H, G, D, V, PAGE, MOST = 4, 2, 64, 12, 16, 220


class Model:
    def __init__(self, device):
        g = torch.Generator().manual_seed(11)
        r = lambda *s: torch.randn(*s, generator=g).to(device)  # noqa: E731
        self.tables = {n: (r(V, h, D) * a, r(MOST, h, D) * a) for n, h, a in (("q", H, 1.4), ("k", G, 0.7), ("v", G, 0.7))}
        self.head = r(H * D, V)

    def rows(self, name, tokens, at):
        token, position = self.tables[name]
        return (token[tokens] + position[at]).to(BF16)

    def logits(self, out):
        return out.flatten(-2).float() @ self.head


def after(model, tokens):
    """the 64-bit logits after a list of tokens, and what roundings of the attention's output may move them by (2^-8 of a weight's product and of the output)"""
    t = torch.tensor(tokens)
    at = torch.arange(len(tokens))
    k, v = (model.rows(n, t, at)[None] for n in ("k", "v"))
    q = model.rows("q", t[-1:], at[-1:])[None]
    out, weight = O.tree_attention(q, k, v, torch.tensor([len(tokens) - 1]), torch.ones(1, 1, 1, dtype=torch.bool))
    head = model.head.double()
    return out.flatten() @ head, ((out.abs() + weight) * (2.0 ** -8 + 2.0 ** -12)).flatten() @ head.abs()


def propose(model, tokens, T, g):
    """a tree behind the last token: at each depth a few wrong guesses beside the likely token, below which the next depth hangs, or hangs below a wrong one"""
    tree, parents, seen, at = [tokens[-1]], [-1], list(tokens), 0
    while len(tree) < T:
        best = int(after(model, seen)[0].argmax())
        guesses = {int(x) for x in torch.randint(0, V, (int(torch.randint(0, 3, (1,), generator=g)),), generator=g)} - {best}
        guesses = sorted(guesses) + [best] if torch.rand((), generator=g) < 0.85 else sorted(guesses) or [(best + 1) % V]
        first = len(tree)
        for x in guesses[:T - first]:
            tree.append(x)
            parents.append(at)
        at = len(tree) - 1
        seen.append(tree[at])
    return tree, parents


def drafted_run(device, steps, T, operators):
    tree_mask, attention, verify, compact, copy_pages = operators
    m, host, g = Model(device), Model("cpu"), torch.Generator().manual_seed(3)
    past = [5, 0, 130]
    seqs = [torch.randint(0, V, (n + 1,), generator=g).tolist() for n in past]
    table = torch.full((4, 14), -1, dtype=torch.int32)
    order = torch.randperm(64, generator=g).int().tolist()
    k, v = (torch.full((64, PAGE, G, D), 9.0, dtype=BF16, device=device) for _ in range(2))
    for b in range(3):
        for j in range(14):
            table[b, j] = order.pop()
        for i, x in enumerate(seqs[b][:-1]):
            k[table[b, i // PAGE], i % PAGE], v[table[b, i // PAGE], i % PAGE] = (m.rows(n, torch.tensor(x), torch.tensor(i)) for n in ("k", "v"))
    # the third is forked: full pages are shared, the begun one and those to come are its own
    own = 130 // PAGE
    table[3, :own] = table[2, :own]
    for j in range(own, 14):
        table[3, j] = order.pop()
    copy_pages([p.view(64, PAGE, G * D) for p in (k, v)], table[2, own:own + 1].to(device), table[3, own:own + 1].to(device))
    seqs.append(seqs[2][:-1] + [(seqs[2][-1] + 5) % V])
    shared = k[table[2, :own].long()].clone()
    pages, counts = table.to(device), []
    lengths = torch.tensor([len(s) - 1 for s in seqs], dtype=torch.int32, device=device)
    for step in range(steps):
        nodes = torch.tensor([T, max(1, T - step), T, 1 + step % T], dtype=torch.int32)
        trees = [propose(host, s, T, g) for s in seqs]
        tokens, parents = (torch.tensor([t[i] for t in trees], dtype=d).to(device) for i, d in ((0, torch.int64), (1, torch.int32)))
        uniform = (torch.rand(4, T, generator=g) * 0.999).to(device)
        nodes = nodes.to(device)
        mask, depth = tree_mask(parents)
        at = lengths[:, None] + depth
        here = lengths[:, None] + torch.arange(T, device=device, dtype=torch.int32)
        live = torch.arange(T, device=device) < nodes[:, None]
        place = (pages.gather(1, (here // PAGE).long()).long()[live], (here % PAGE).long()[live])
        for pool, n in ((k, "k"), (v, "v")):
            pool[place] = m.rows(n, tokens, at)[live]
        out = attention(m.rows("q", tokens, at), k, v, lengths, mask, nodes=nodes, page_table=pages)
        out = torch.where(live[:, :, None, None], out, 0.0)
        target = torch.nn.functional.one_hot(m.logits(out).argmax(-1), V).float()
        path, count, last = verify(target, tokens, parents, uniform, nodes=nodes)
        compact([p.view(64, PAGE, G * D) for p in (k, v)], lengths, path, count, page_table=pages)
        lengths += count
        for b, s in enumerate(seqs):
            n = int(count[b])
            s += [int(tokens[b, int(i)]) for i in path[b, 1:n]] + [int(last[b])]
            counts.append(n)
    for b, s in enumerate(seqs):
        assert int(lengths[b]) == len(s) - 1
        start = past[min(b, 2)] + 1
        for n in range(start, len(s)):                    # each token is the best after those before it, as far as roundings leave one
            want, off = after(host, s[:n])
            assert float(want[s[n]]) >= float((want - off).max() - off[s[n]]), (b, n)
        t, at = torch.tensor(s[:-1]), torch.arange(len(s) - 1)
        rows = (table[b, at // PAGE].long(), at % PAGE)
        assert torch.equal(k[rows].cpu(), host.rows("k", t, at)) and torch.equal(v[rows].cpu(), host.rows("v", t, at))
    assert torch.equal(k[table[2, :own].long()], shared)
    assert max(counts) > 3 and min(counts) == 1           # (whole branches were accepted, and none)
    return seqs


def words(parents):
    sees = O.tree_sees(parents)
    return O.tree_words(sees), (sees.sum(-1) - 1).int()


def bits(mask, T):
    return torch.stack([mask[:, :, j // 64] >> (j % 64) & 1 for j in range(T)], -1).bool()


def in_place(pools, changed):
    for p, c in zip(pools, changed):
        p.copy_(c)


DEFINITIONS = (words, lambda q, k, v, lengths, mask, nodes, page_table: O.tree_attention(q, k, v, lengths, bits(mask, q.shape[1]), nodes, page_table)[0].to(BF16),
               lambda target, tokens, parents, uniform, nodes: O.verify_draft(target, tokens, parents, uniform, None, nodes),
               lambda pools, lengths, path, count, page_table: in_place(pools, [O.cache_compact(p, lengths, path, count, page_table) for p in pools]),
               lambda pools, src, dst: [p.__setitem__(dst.long(), p[src.long()].clone()) for p in pools])


def test_drafted_steps_by_the_definitions():
    drafted_run("cpu", 3, 7, DEFINITIONS)


@gpu
@pytest.mark.parametrize("steps, T", [(9, 7), (4, 21), (2, 40)])
def test_drafted_steps_are_one_token_at_a_time(steps, T):
    drafted_run("cuda", steps, T, (ops.tree_mask, ops.tree_attention, ops.verify_draft, ops.cache_compact, ops.cache_copy_pages))
