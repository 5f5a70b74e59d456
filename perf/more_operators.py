"""What serving many continuations of one prompt adds to the framework, as cases that can be timed and compared: the index tables and cache pages of a step, rotary positions
and the cache rows that they end in, attention of a batch over the prefix that it shares, and the draw of the next tokens.  Sizes are the decoder's (32 query and 8 key heads of 128,
vocabularies of 128256, 32003 and 32000), prompts of the benchmark and longer ones.

A case is a dict of plain values; `prepare` builds what a program holds before the call, `run` makes one pass (the framework's operator where `own`, elementary torch otherwise),
`exact` says in 64 bits what that pass returns."""
import math

import numpy as np
import torch

BF16, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
own = False


# ------------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step of 64 running requests: one token each, a few idle, a page now and then (latency)
        tables(64, 4796, 1, 64, name="tables-decode"),
        # the prompts of 256 requests packed into one step of small pages
        tables(256, 1000, 512, 16, name="tables-prompts"),
        # the queries of the benchmark's prompt: half of each head's dimensions, interleaved, 32 bits
        rotary(4796, 32, 128, 64, pairs="interleaved", bf16=False, grad=False, far=131072, name="rotary-prompt"),
        # gradients of the queries of four training sequences
        rotary(16384, 32, 128, 128, pairs="half", bf16=True, grad=True, far=4096, name="rotary-grad"),
        # the new token of 64 requests: queries turned, keys and values to their cache rows (latency)
        append(64, 32, 8, 128, 128, pairs="half", page=64, far=100003, name="append-decode"),
        # a prompt's rows into the cache
        append(4796, 32, 8, 128, 128, pairs="half", page=64, far=4796, name="append-prompt"),
        # four samples of the benchmark's prompt, a few tokens on
        prefix(4, 1, 4796, 40, page=64, name="prefix-four"),
        # sixty-four samples behind a long document
        prefix(64, 1, 32771, 500, page=64, name="prefix-sixty-four"),
        # sixteen questions of up to 24 tokens about one very long document
        prefix(16, 24, 100003, 24, page=0, name="prefix-questions"),
        # one user, the usual settings, bf16 logits (latency)
        sample(1, 128256, bf16=True, mode="both", name="sample-one"),
        # a batch of 64 whose requests have settings of their own
        sample(64, 128256, bf16=False, mode="mixed", name="sample-mixed"),
        # 256 requests that draw from the whole distribution, rows of an odd length
        sample(256, 32003, bf16=False, mode="plain", name="sample-plain"),
    ]


def tables(batch, length, new, page, name=None):
    return named({"kind": "tables", "batch": batch, "length": length, "new": new, "page": page}, name)


def rotary(rows, heads, dim, turned, pairs, bf16, grad, far, name=None):
    return named({"kind": "rotary", "rows": rows, "heads": heads, "dim": dim, "turned": turned, "pairs": pairs, "bf16": bf16, "grad": grad, "far": far}, name)


def append(rows, heads, kv_heads, dim, turned, pairs, page, far, name=None):
    return named({"kind": "append", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "turned": turned, "pairs": pairs, "page": page, "far": far}, name)


def prefix(batch, new, prefix, length, page, heads=32, kv_heads=8, dim=128, name=None):
    return named({"kind": "prefix", "batch": batch, "new": new, "prefix": prefix, "length": length, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim}, name)


def sample(rows, vocab, bf16, mode, name=None):
    return named({"kind": "sample", "rows": rows, "vocab": vocab, "bf16": bf16, "mode": mode}, name)


def named(case, name):
    return dict(case, name=name) if name else case


def spread(rng, lo, hi):
    """a whole number of [lo, hi], even over its logarithm"""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


HEADS = [(32, 8, 128), (32, 8, 128), (16, 16, 128), (8, 1, 128), (16, 4, 96), (12, 4, 64)]


def draw(rng):
    kind = rng.choice(["tables", "rotary", "append", "prefix", "prefix", "prefix", "sample", "sample"])
    if kind == "tables":
        batch = spread(rng, 1, 1024)
        return tables(batch, spread(rng, 1, 8000), rng.choice([1, 1, spread(rng, 2, max(2, min(512, 130000 // batch)))]), rng.choice([16, 48, 64, 128]))
    if kind == "rotary":
        heads, _, dim = rng.choice(HEADS)
        rows = min(spread(rng, 1, 16384), 16777216 // (heads * dim))
        return rotary(rows, heads, dim, rng.choice([dim, dim, dim // 2, 32]), rng.choice(["half", "interleaved"]), rng.random() < 0.6, rng.random() < 0.4, spread(rng, rows, 1000000))
    if kind == "append":
        heads, kv_heads, dim = rng.choice(HEADS)
        return append(spread(rng, 1, 4796), heads, kv_heads, dim, rng.choice([dim, dim, dim // 2]), rng.choice(["half", "interleaved"]), rng.choice([16, 48, 64]),
                      spread(rng, 4796, 1000000))
    if kind == "prefix":
        heads, kv_heads, dim = rng.choice(HEADS)
        batch, new = spread(rng, 1, 96), rng.choice([1, 1, spread(rng, 2, 32)])
        most = min(100003, 150000000000 // (batch * new * heads * dim))
        return prefix(batch, new, spread(rng, 1, most), spread(rng, 1, 600), rng.choice([0, 16, 48, 64, 128]), heads, kv_heads, dim)
    vocab = rng.choice([32000, 32003, 128256, spread(rng, 100, 128256)])
    return sample(min(spread(rng, 1, 256), 8208384 // vocab), vocab, rng.random() < 0.4, rng.choice(["plain", "top", "nucleus", "both", "least", "mixed"]))


# ------------------------------------------------------------------------------------------------------------------------ inputs
def of_case(case):
    """numbers that only the case fixes: lengths and tokens of the requests, from a generator of their own (`work` needs them too)"""
    return np.random.default_rng([case["batch"], case["new"], case["length"], case["page"]])


def requests_of(case):
    """(cached rows, new tokens) of each request: the first has most of both; of the others a few bring none"""
    r = of_case(case)
    lengths = [case["length"]] + [int(r.integers(0, case["length"] + 1)) for _ in range(case["batch"] - 1)]
    new = [case["new"]] + [int(r.integers(0, case["new"] + 1)) if case["new"] > 1 else int(r.random() < 0.9) for _ in range(case["batch"] - 1)]
    return lengths, new


def rows_of(case):
    """rows that the step has room for: a multiple of 64 (captured steps of a few sizes)"""
    return -(-sum(requests_of(case)[1]) // 64) * 64


def tables_of(needed, r, first=()):
    """a page table [requests, most pages] of pages in random order after the shared ones, and the pages of the pool"""
    order = r.permutation(sum(needed) + len(first) + 3)
    table = np.full((len(needed), len(first) + max(needed)), -1, np.int64)
    table[:, :len(first)] = order[:len(first)]
    at = len(first)
    for b, n in enumerate(needed):
        table[b, len(first):len(first) + n] = order[at:at + n]
        at += n
    return table, len(order)


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    st = {"case": case}
    if case["kind"] == "tables":
        lengths, new = requests_of(case)
        size = case["page"]
        held = [-(-n // size) for n in lengths]
        width = max(-(-(n + t) // size) for n, t in zip(lengths, new))
        order = r.permutation(sum(held) + sum(-(-t // size) + 1 for t in new) + 5)
        table, at = np.full((case["batch"], width), -1, np.int64), 0
        for b, n in enumerate(held):
            table[b, :n] = order[at:at + n]
            at += n
        st["lengths"], st["new"], st["table"], st["free"] = dev(lengths, I32), dev(new, I32), dev(table, I32), dev(order[at:], I32)
        st["used"] = torch.full((1,), 2, dtype=I32, device="cuda")
    elif case["kind"] in ("rotary", "append"):
        n, H, D = case["rows"], case["heads"], case["dim"]
        st["freq"] = dev(500000.0 ** (-np.arange(0, case["turned"], 2) / case["turned"]), F32)
        # the rows of a prompt's chunk, or of many requests
        at = np.arange(n) + case["far"] - n if case["kind"] == "rotary" or n > 512 else r.integers(0, case["far"], n)
        st["pos"] = dev(at, I32)
        if case["kind"] == "rotary":
            st["x"] = rnd(n, H + 2, D).to(BF16 if case["bf16"] else F32)[:, :H]          # the queries of a wider product
        else:
            G, size = case["kv_heads"], case["page"]
            qkv = rnd(n, H + 2 * G, D).to(BF16)
            st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
            pages = -(-n // size) + 3
            st["k_pool"], st["v_pool"] = (rnd(pages, size, G, D).to(BF16) for _ in range(2))
            slots = r.permutation(pages)[:-(-n // size), None] * size + np.arange(size)[None]
            st["slots"] = dev(np.where(r.random(n) < 0.02, -1, slots.reshape(-1)[:n]), I64)      # rows of a padded step go nowhere
    elif case["kind"] == "prefix":
        B, T, H, G, D, P, size = (case[k] for k in ("batch", "new", "heads", "kv_heads", "dim", "prefix", "page"))
        lengths, new = requests_of(case)
        st["q"] = rnd(B, T, H, D).mul_(1.5).to(BF16)
        if size:
            first = P // size                                   # whole pages are shared, the rest of the prefix is each request's own copy
            table, pages = tables_of([-(-(P + n + T) // size) - first for n in lengths], r, range(first))
            st["table"], shape = dev(table, I32), (pages, size, G, D)
            st["k"], st["v"] = (torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=g) for _ in range(2))
            if P % size:
                last = st["table"][:, first].long()
                for x in (st["k"], st["v"]):
                    x[last, :P % size] = x[last[:1], :P % size].clone()
            st["prefix_k"] = st["prefix_v"] = None
        else:
            st["table"] = None
            st["k"], st["v"] = (torch.empty((B, -(-(max(lengths) + T) // 64) * 64, G, D), dtype=BF16, device="cuda").normal_(generator=g) for _ in range(2))
            st["prefix_k"], st["prefix_v"] = (torch.empty((P, G, D), dtype=BF16, device="cuda").normal_(generator=g) for _ in range(2))
        st["lengths"], st["new"] = dev(np.asarray(lengths) + P, I32), dev(new, I32)
        st["out"] = rnd(B, T, H, D).mul_(1e-3).to(BF16)         # rows of tokens that a request does not bring stay as they were
    else:
        R, V, mode = case["rows"], case["vocab"], case["mode"]
        z = rnd(R, V).mul_(2.5)
        z[:, :max(1, V // 1000)] += 3                           # some words are likely everywhere
        st["logits"] = z[:, torch.as_tensor(r.permutation(V)).cuda()].to(BF16 if case["bf16"] else F32)
        st["uniform"] = torch.rand(R, generator=g, device="cuda")
        st.update({"plain": dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), "top": dict(temperature=0.8, top_k=50, top_p=1.0, min_p=0.0),
                   "nucleus": dict(temperature=1.0, top_k=0, top_p=0.9, min_p=0.0), "both": dict(temperature=0.7, top_k=200, top_p=0.95, min_p=0.0),
                   "least": dict(temperature=1.2, top_k=0, top_p=1.0, min_p=0.05)}.get(mode) or
                  dict(temperature=dev(r.choice([0.0, 0.3, 0.7, 1.0, 1.3], R), F32), top_k=dev(r.choice([0, 1, 40, 1000], R), I32),
                       top_p=dev(r.choice([0.5, 0.9, 0.99, 1.0], R), F32), min_p=dev(r.choice([0.0, 0.0, 0.02], R), F32)))
    return st


# ------------------------------------------------------------------------------------------------------------------------ one pass
def run(st):
    return {"tables": run_tables, "rotary": run_rotary, "append": run_append, "prefix": run_prefix, "sample": run_sample}[st["case"]["kind"]](st)


def run_tables(st):
    case, table, used = st["case"], st["table"], st["used"]
    rows, size = rows_of_state(st), case["page"]
    if own:
        from leopard_b200 import ops
        return (*ops.step_tables(st["lengths"], st["new"], table, st["free"], used, size, rows), table, used)
    lengths, new, free = st["lengths"].long(), st["new"].long(), st["free"]
    B, W = table.shape
    row0 = torch.zeros(B + 1, dtype=I64, device="cuda")
    row0[1:] = new.cumsum(0)
    page = torch.arange(W, device="cuda")[None]
    wants = (table < 0) & (page >= (lengths // size)[:, None]) & (page * size < (lengths + new)[:, None]) & (new > 0)[:, None]
    at = used.long() + wants.flatten().cumsum(0).view(B, W) - 1
    given = wants & (at < len(free))
    table.copy_(torch.where(given, free[at.clamp(max=len(free) - 1)], table))
    used.add_(given.sum())
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(row0[1:], row, right=True)
    there = seq < B
    seq = seq.clamp(max=B - 1)
    pos = lengths[seq] + row - row0[seq]
    of = torch.where(pos < W * size, table[seq, (pos // size).clamp(max=W - 1)], -1)
    slots = torch.where(there & (of >= 0), of.long() * size + pos % size, -1)
    return torch.where(there, seq, -1).int(), torch.where(there, pos, -1).int(), slots, row0.int(), table, used


def rows_of_state(st):
    if "rows" not in st:
        st["rows"] = rows_of(st["case"])
    return st["rows"]


def turn(x, pos, freq, pairs, sign):
    """the first dimensions of each head turned by its position's angles, 32 bits out"""
    angle = pos.double()[:, None] * freq.double()[None]
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None] * sign
    n = 2 * freq.numel()
    y = x.float().clone()
    a, b = (y[..., 0:n:2].clone(), y[..., 1:n:2].clone()) if pairs == "interleaved" else (y[..., :n // 2].clone(), y[..., n // 2:n].clone())
    first, second = a * c - b * s, b * c + a * s
    if pairs == "interleaved":
        y[..., 0:n:2], y[..., 1:n:2] = first, second
    else:
        y[..., :n // 2], y[..., n // 2:n] = first, second
    return y


def run_rotary(st):
    case, x = st["case"], st["x"]
    if own:
        from leopard_b200 import ops
        return ops.rotary(x, st["pos"], st["freq"], layout=case["pairs"], inverse=case["grad"])
    return turn(x, st["pos"], st["freq"], case["pairs"], -1.0 if case["grad"] else 1.0).to(x.dtype)


def run_append(st):
    case = st["case"]
    if own:
        from leopard_b200 import ops
        return ops.rotary_append(st["q"], st["k"], st["v"], st["pos"], st["freq"], st["k_pool"], st["v_pool"], st["slots"], layout=case["pairs"]), st["k_pool"], st["v_pool"]
    q, k = (turn(x, st["pos"], st["freq"], case["pairs"], 1.0).to(BF16) for x in (st["q"], st["k"]))
    # rows without a place are written to the place of the pool's last row, which keeps what it has
    to, there = st["slots"].clamp(min=0), (st["slots"] >= 0)[:, None, None]
    for pool, x in ((st["k_pool"], k), (st["v_pool"], st["v"])):
        flat = pool.view(-1, *pool.shape[2:])
        spare = flat.shape[0] - 1
        where = torch.where(st["slots"] >= 0, to, spare)
        kept = flat[spare].clone()
        mine = ((st["slots"] == spare)[:, None, None] * x.float()).sum(0)
        flat[where] = torch.where(there, x, flat[spare][None])
        flat[spare] = torch.where((st["slots"] == spare).any(), mine.to(BF16), kept)
    return q, st["k_pool"], st["v_pool"]


def run_prefix(st):
    case, q, out = st["case"], st["q"], st["out"]
    B, T, H, D = q.shape
    P, size = case["prefix"], case["page"]
    if own:
        from leopard_b200 import ops
        return ops.prefix_attention(q, st["k"], st["v"], st["lengths"], P, new=st["new"], page_table=st["table"], prefix_k=st["prefix_k"], prefix_v=st["prefix_v"], out=out)
    G = st["k"].shape[2]
    behind = st["lengths"].long() - P                           # own rows before the new tokens
    at = torch.arange(case["length"] + T, device="cuda")
    if size:
        table, first = st["table"].long(), torch.arange(P, device="cuda")
        pk, pv = (x[table[0, first // size], first % size] for x in (st["k"], st["v"]))
        page = table[:, ((at + P) // size).clamp(max=table.shape[1] - 1)].clamp(min=0)
        k, v = (x[page, (at + P) % size] for x in (st["k"], st["v"]))
    else:
        pk, pv, k, v = st["prefix_k"], st["prefix_v"], st["k"][:, :len(at)], st["v"][:, :len(at)]
    qf = q.float().view(B, T, G, H // G, D)
    s0 = torch.einsum("btghd,kgd->btghk", qf, pk.float()).mul_(D ** -0.5)
    s1 = torch.einsum("btghd,bkgd->btghk", qf, k.float()).mul_(D ** -0.5)
    sees = at[None, None] <= behind[:, None, None] + torch.arange(T, device="cuda")[None, :, None]
    s1.masked_fill_(~sees[:, :, None, None], float("-inf"))
    top = torch.maximum(s0.amax(-1, keepdim=True), s1.amax(-1, keepdim=True))
    p0, p1 = torch.exp(s0.sub_(top)), torch.exp(s1.sub_(top))
    total = p0.sum(-1) + p1.sum(-1)
    o = (torch.einsum("btghk,kgd->btghd", p0, pv.float()) + torch.einsum("btghk,bkgd->btghd", p1, v.float())) / total[..., None]
    there = torch.arange(T, device="cuda")[None] < st["new"][:, None]
    return out.copy_(torch.where(there[:, :, None, None], o.reshape(B, T, H, D).to(BF16), out))


def run_sample(st):
    z, u = st["logits"], st["uniform"]
    settings = {k: st[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    if own:
        from leopard_b200 import ops
        return ops.sample_tokens(z, u, **settings)
    R, V = z.shape
    t, k, p, least = (torch.as_tensor(x, device="cuda").double().expand(R)[:, None] for x in (settings[n] for n in ("temperature", "top_k", "top_p", "min_p")))
    p, least = p.float().double(), least.float().double()       # settings come in 32 bits
    t = t.float().double()
    # 64 bits: the draw is decided next to a border between two words
    z = z.double()
    top = z.amax(-1, keepdim=True)
    w = torch.exp((z - top) / torch.where(t > 0, t, 1.0))
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(V, device="cuda")[None]
    keep = rank < torch.where(k > 0, k, V)
    mass = torch.where(keep, ws, 0.0).cumsum(-1)
    keep &= ((mass - ws < p * mass[:, -1:]) | (rank == 0)) & (ws >= least)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0)).cumsum_(-1)
    drawn = (kept > u.double()[:, None] * kept[:, -1:]).int().argmax(-1)
    return torch.where(t[:, 0] > 0, drawn, z.argmax(-1))


# ------------------------------------------------------------------------------------------------------------------------ what is needed
def work(case):
    if case["kind"] == "tables":
        lengths, new = requests_of(case)
        pages = sum(-(-(n + t) // case["page"]) - n // case["page"] for n, t in zip(lengths, new) if t)
        return {"bytes": 16 * rows_of(case) + 12 * case["batch"] + 8 * pages, "flops": 0}
    if case["kind"] == "rotary":
        n = case["rows"] * case["heads"]
        return {"bytes": n * case["dim"] * 2 * (2 if case["bf16"] else 4) + 4 * case["rows"], "flops": 3 * n * case["turned"]}
    if case["kind"] == "append":
        n = case["rows"]
        return {"bytes": n * (case["heads"] + 2 * case["kv_heads"]) * case["dim"] * 4 + 12 * n, "flops": 3 * n * (case["heads"] + case["kv_heads"]) * case["turned"]}
    if case["kind"] == "prefix":
        H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
        lengths, new = requests_of(case)
        rows = P + sum(n + t for n, t in zip(lengths, new) if t)
        return {"bytes": 4 * rows * G * D + 4 * sum(new) * H * D, "flops": sum(4 * t * H * D * (P + n + t // 2) for n, t in zip(lengths, new))}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (2 if case["bf16"] else 4) + 12 * case["rows"], "flops": 4 * n}


# ------------------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "tables":
        lengths, new = requests_of(case)
        table, free, used, size = st["table"].tolist(), st["free"].tolist(), 2, case["page"]
        seq, pos, slot, row0 = [], [], [], [0]
        for b, (n, t) in enumerate(zip(lengths, new)):
            for i in range(n, n + t):
                if i // size < len(table[b]) and table[b][i // size] < 0 and used < len(free):
                    table[b][i // size], used = free[used], used + 1
                page = table[b][i // size] if i // size < len(table[b]) else -1
                seq.append(b), pos.append(i), slot.append(page * size + i % size if page >= 0 else -1)
            row0.append(len(seq))
        pad = [-1] * (rows_of(case) - len(seq))
        return tuple(torch.tensor(x, dtype=d, device="cuda") for x, d in ((seq + pad, I32), (pos + pad, I32), (slot + pad, I64), (row0, I32), (table, I32), ([used], I32)))
    if kind in ("rotary", "append"):
        phase = torch.polar(torch.ones((), dtype=F64, device="cuda"), st["pos"].double()[:, None] * st["freq"].double()[None])[:, None]
        n = case["turned"]

        def turned(x, phase):
            y = x.double()
            if case["pairs"] == "half":
                z = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * phase
                return torch.cat([z.real, z.imag, y[..., n:]], -1)
            z = torch.view_as_complex(y[..., :n].reshape(*y.shape[:-1], n // 2, 2).contiguous()) * phase
            return torch.cat([torch.view_as_real(z).flatten(-2), y[..., n:]], -1)
        if kind == "rotary":
            return turned(st["x"], phase.conj() if case["grad"] else phase)
        pools = [st["k_pool"].double(), st["v_pool"].double()]
        on = st["slots"] >= 0
        for pool, x in zip(pools, (turned(st["k"], phase), st["v"].double())):
            pool.view(-1, *pool.shape[2:])[st["slots"][on]] = x[on]
        return (turned(st["q"], phase), *pools)
    if kind == "prefix":
        out = st["out"].double()
        T, H, G, D, P, size = (case[k] for k in ("new", "heads", "kv_heads", "dim", "prefix", "page"))
        for b, (n, t) in enumerate(zip(*requests_of(case))):
            if not t:
                continue
            if size:
                pages = st["table"][b, :-(-(P + n + t) // size)].long()
                k, v = (x[pages].reshape(-1, G, D)[:P + n + t] for x in (st["k"], st["v"]))
            else:
                k, v = (torch.cat([a, x[b, :n + t]]) for a, x in ((st["prefix_k"], st["k"]), (st["prefix_v"], st["v"])))
            hidden = torch.triu(torch.full((t, t), -math.inf, dtype=F64, device="cuda"), 1)
            for h in range(H):
                s = st["q"][b, :t, h].double() @ k[:, h // (H // G)].double().T / math.sqrt(D)
                s[:, P + n:] += hidden
                out[b, :t, h] = torch.softmax(s, -1) @ v[:, h // (H // G)].double()
        return out
    host, u = st["logits"].float().cpu().numpy().astype(np.float64), st["uniform"].cpu().numpy().astype(np.float64)
    t, k, p, least = (np.broadcast_to(np.float32(x.cpu().numpy() if torch.is_tensor(x) else x).astype(np.float64), (case["rows"],))
                      for x in (st[n] for n in ("temperature", "top_k", "top_p", "min_p")))
    tokens = []
    for i, z in enumerate(host):
        best = int(np.argmax(z))
        if t[i] <= 0:
            tokens.append(best)
            continue
        order = np.lexsort((np.arange(len(z)), -z))             # the largest first, equal ones in their order
        w = np.exp((z[order] - z[best]) / t[i])
        w = w[:int(k[i])] if k[i] > 0 else w
        upto = np.concatenate([[0.0], np.cumsum(w)])
        n = max(1, int(np.sum(upto[:-1] < p[i] * upto[-1])))
        n = min(n, int(np.sum(w >= least[i])))
        chosen = np.sort(order[:n])
        c = np.cumsum(np.exp((z[chosen] - z[best]) / t[i]))
        tokens.append(int(chosen[min(n - 1, int(np.searchsorted(c, u[i] * c[-1], side="right")))]))
    return torch.tensor(tokens, device="cuda")
