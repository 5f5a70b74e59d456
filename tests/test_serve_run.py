"""A run of many continuations of one prompt with the serving operators together: the prompt's rows go to the cache once, requests share its pages, bring a question of their own and then
draw token after token.  The model is small and keeps nothing but what a cache holds: a token's query, key and value are rows of tables, turned by their positions, and its logits are a product with what its attention gives.
Checked at every step: the logits against attention over the request's whole sequence in 64 bits, the token against the definition's draw from those same logits, the cache against the tokens."""
import pytest
import torch

from leopard_b200 import ops
from oracle import serve as O

gpu = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
H, G, D, VOCAB, PAGE = 8, 2, 64, 211, 16


class Model:
    def __init__(self, device, seed):
        g = torch.Generator(device="cpu").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.q, self.k, self.v = ((rnd(VOCAB, n, D) * 1.2).to(BF16).to(device) for n in (H, G, G))
        self.out = rnd(H * D, VOCAB).to(device)
        self.freq = (10000.0 ** (-torch.arange(D // 4, dtype=torch.float64) / (D // 4))).float().to(device)      # half of a head is turned

    def logits_of(self, tokens):
        """after the last of these tokens, in 64 bits, and how far roundings may take them: queries and keys are rounded to bf16 when they are turned (half a step, 2^-8 of their pair's size), weights before the
        second product and the result after it"""
        t = torch.as_tensor(tokens, device=self.q.device)
        pos = torch.arange(len(t), device=self.q.device)
        (q, q_size), (k, k_size) = (O.rotary(x[t], pos, self.freq) for x in (self.q, self.k))
        q, q_size, v = q[-1], q_size[-1], self.v[t].double()
        of = torch.arange(H, device=q.device) // (H // G)
        s = torch.einsum("hd,nhd->hn", q, k[:, of]) * D ** -0.5
        off = (torch.einsum("hd,nhd->hn", q_size, k_size[:, of]) * 2.02 * 2.0 ** -8 * D ** -0.5).amax(-1, keepdim=True)      # of the scores: both factors' half steps
        w = torch.softmax(s, -1)
        o, size = torch.einsum("hn,nhd->hd", w, v[:, of]), torch.einsum("hn,nhd->hd", w, v[:, of].abs())
        move = torch.expm1(2 * off) * size + 2.0 ** -8 * (o.abs() + size) * 1.02 + 2.0 ** -12 * size
        return o.reshape(-1) @ self.out.double(), move.reshape(-1) @ self.out.double().abs() + 1e-6


def serve(device, samples, steps, question, calls):
    tables, append, attend, draw, copy_pages = calls
    m = Model(device, 5)
    g = torch.Generator(device="cpu").manual_seed(samples)
    words = lambda n: torch.randint(0, VOCAB, (n,), generator=g)  # noqa: E731
    prompt = words(150)
    P = len(prompt)
    shared, pages = P // PAGE, 400
    pools = [torch.full((pages, PAGE, G, D), float("nan"), dtype=BF16, device=device) for _ in range(2)]
    free = torch.randperm(pages, generator=g).to(I32).to(device)
    used = torch.zeros(1, dtype=I32, device=device)
    i32 = lambda x: torch.tensor(x, dtype=I32, device=device)  # noqa: E731

    def rows_of(tokens, lengths, new, table, rows):
        """the step's rows into the cache -> queries [rows, H, D], the tables"""
        seq, pos, slots, row0 = tables(lengths, new, table, free, used, PAGE, rows)
        t = torch.zeros(rows, dtype=torch.long, device=device)
        t[:len(tokens)] = torch.as_tensor(tokens, device=device)
        q = append(m.q[t], m.k[t], m.v[t], pos.clamp(min=0), m.freq, *pools, slots)
        return q, seq, pos, row0

    # ---- the prompt: its rows once
    table = torch.full((1, 40), -1, dtype=I32, device=device)
    rows_of(prompt, i32([0]), i32([P]), table, P)
    # ---- the requests hold its whole pages, and a copy each of the last one's rows
    many = table.expand(samples, -1).contiguous()
    own = free[int(used):int(used) + samples].clone()
    used += samples
    copy_pages(pools, table[:, shared].expand(samples).contiguous(), own)
    many[:, shared] = own
    lengths = i32([P] * samples)
    seqs = [prompt.tolist() for _ in range(samples)]
    pending = [words(int(n)).tolist() for n in torch.randint(1, question + 1, (samples,), generator=g)]      # each request's question
    T = question
    for step in range(steps):
        new = i32([0 if step % 3 == 1 and b % 4 == 3 else len(pending[b]) for b in range(samples)])      # now and then some wait
        flat = [t for b in range(samples) if int(new[b]) for t in pending[b]]
        rows = -(-len(flat) // 8) * 8                     # a padded step
        q, seq, pos, row0 = rows_of(flat, lengths, new, many, rows)
        batch = torch.zeros(samples, T, H, D, dtype=BF16, device=device)
        on = seq >= 0
        batch[seq[on].long(), (pos - lengths[seq.clamp(min=0).long()])[on].long()] = q[on]
        out = attend(batch, *pools, lengths, P, new, many)
        last = (new.long() - 1).clamp(min=0)
        logits = out[torch.arange(samples, device=device), last].float().reshape(samples, -1) @ m.out
        u = torch.rand(samples, generator=g).to(device)
        settings = dict(temperature=0.9 * float(logits[new > 0].std()), top_k=60, top_p=0.95)      # (rows of those that wait are unspecified)
        token = draw(logits, u, **settings)
        want = O.sample_tokens(logits, u, **settings)
        for b in range(samples):
            if not int(new[b]):
                continue
            seqs[b] += pending[b]
            exact, off = m.logits_of(seqs[b])
            assert bool(((logits[b].double() - exact).abs() <= off + 2.0 ** -18 * exact.abs().max()).all()), (step, b)
            assert int(token[b]) == want[b]
            pending[b] = [int(token[b])]
        lengths = lengths + new
        T = 1 if step else question
    # ---- the cache holds every request's tokens, the prompt's pages as they were written once
    assert bool((many[:, :shared] == table[0, :shared]).all())
    for b, s in enumerate(seqs):
        t, at = torch.as_tensor(s, device=device), torch.arange(len(s), device=device)
        assert len(s) == int(lengths[b])
        where = (many[b, at // PAGE].long(), at % PAGE)
        turned, size = O.rotary(m.k[t], at, m.freq)
        assert bool(((pools[0][where].double() - turned).abs() <= 2.0 ** -8 * turned.abs() + 2.0 ** -20 * size).all()) and torch.equal(pools[1][where], m.v[t])


def by_definition_tables(lengths, new, table, free, used, size, rows):
    seq, pos, slots, row0, t, n = O.step_tables(lengths, new, table, free, used, size, rows)
    table.copy_(torch.tensor(t))
    used.fill_(n)
    return (*(torch.tensor(x, dtype=I32) for x in (seq, pos)), torch.tensor(slots), torch.tensor(row0, dtype=I32))


def by_definition_append(q, k, v, pos, freq, k_pool, v_pool, slots):
    O.append(k_pool, O.rotary(k, pos, freq)[0].to(BF16), slots)
    O.append(v_pool, v, slots)
    return O.rotary(q, pos, freq)[0].to(BF16)


DEFINITIONS = (by_definition_tables, by_definition_append, lambda q, k, v, lengths, P, new, table: O.prefix_attention(q, k, v, lengths, P, new, table)[0].to(BF16),
               lambda z, u, **kw: torch.tensor(O.sample_tokens(z, u, **kw)), lambda pools, src, dst: [p.__setitem__(dst.long(), p[src.long()].clone()) for p in pools])


def test_a_served_prompt_by_the_definitions():
    serve("cpu", 3, 4, 3, DEFINITIONS)


@gpu
@pytest.mark.parametrize("samples, steps, question", [(1, 12, 5), (4, 12, 1), (24, 9, 4), (70, 5, 12)])
def test_a_served_prompt(samples, steps, question):
    serve("cuda", samples, steps, question, (ops.step_tables, ops.rotary_append, lambda q, k, v, lengths, P, new, table: ops.prefix_attention(q, k, v, lengths, P, new=new, page_table=table),
                                             ops.sample_tokens, lambda pools, src, dst: ops.cache_copy_pages([p.flatten(2) for p in pools], src, dst)))
