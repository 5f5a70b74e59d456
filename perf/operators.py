"""What drafting adds to the framework, as cases that can be timed and compared: attention of a tree of drafted tokens over a cache, verification of
the drafts against the target's probabilities, rows and pages of a cache moved in all layers at once, and distillation from a teacher's top logits.
Sizes are the decoder's (32 query and 8 key heads of 128, 32 layers, vocabularies of 128256, 32003 and 32000), prompts of the benchmark and longer ones.

A case is a dict of plain values; `prepare` builds what a program holds before the call, `run` makes one pass (the framework's operator where `own`,
elementary torch otherwise), `exact` says in 64 bits what that pass returns."""
import math

import numpy as np
import torch

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
own = False


# ------------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one user, a short chat, a step without drafts: the smallest call (latency)
        tree(1, 1, 512, page=0, name="tree-one"),
        # a tree of 26 nodes after the headline request's prompt, over the dense cache that decoding fills
        tree(1, 26, 4796, page=0, name="tree-4796"),
        # eight running requests of different lengths with wide trees, over pages
        tree(8, 64, 8191, page=64, name="tree-batch"),
        # two long documents
        tree(2, 13, 100003, page=64, name="tree-long"),
        # one user, a chain of five drafts, the 32003-word vocabulary
        verify(1, 6, 32003, branch=1, name="verify-chain"),
        # eight requests, trees of 32 nodes, the 128256-word vocabulary
        verify(8, 32, 128256, branch=3, name="verify-tree"),
        # the accepted nodes of one request become its last cache rows, in all layers
        compact(1, 26, 4796, layers=32, width=1024, page=0, name="compact-one"),
        # ... of sixteen requests over pages
        compact(16, 64, 1021, layers=32, width=1024, page=64, name="compact-batch"),
        # a request is forked or moved: forty pages of 64 rows, keys and values of 32 layers
        {"kind": "pages", "pools": 64, "pages": 256, "copied": 40, "page": 64, "width": 1024, "name": "pages-40"},
        # a short answer distilled from a teacher's eight best, bf16 logits of an odd vocabulary
        distill(48, 32003, 8, bf16=True, hard=0.0, tau=1.0, share=1.0, name="distill-short"),
        # a batch of instructions, of which the answers count, with the labels' share and a temperature
        distill(2048, 32000, 64, bf16=False, hard=0.3, tau=2.0, share=0.6, name="distill-sft"),
        # a full sequence of 4096 rows over the largest vocabulary
        distill(4096, 128256, 64, bf16=False, hard=0.0, tau=1.0, share=1.0, name="distill-4096"),
    ]


def tree(batch, nodes, length, page, heads=32, kv_heads=8, dim=128, name=None):
    return named({"kind": "tree", "batch": batch, "nodes": nodes, "length": length, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim}, name)


def verify(batch, nodes, vocab, branch, drawn=True, name=None):
    return named({"kind": "verify", "batch": batch, "nodes": nodes, "vocab": vocab, "branch": branch, "drawn": drawn}, name)


def compact(batch, nodes, length, layers, width, page, name=None):
    return named({"kind": "compact", "batch": batch, "nodes": nodes, "length": length, "layers": layers, "width": width, "page": page}, name)


def distill(rows, vocab, top, bf16, hard, tau, share, name=None):
    return named({"kind": "distill", "rows": rows, "vocab": vocab, "top": top, "bf16": bf16, "hard": hard, "tau": tau, "share": share}, name)


def named(case, name):
    return dict(case, name=name) if name else case


def spread(rng, lo, hi):
    """a whole number of [lo, hi], even over its logarithm"""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "verify", "compact", "pages", "distill", "distill"])
    if kind == "tree":
        batch, nodes = spread(rng, 1, 16), spread(rng, 1, 128)
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (16, 16, 128), (8, 1, 128), (16, 4, 96), (12, 4, 64)])
        most = min(120000, 2000000000 // (batch * nodes * heads * dim), 200000 // batch)
        return tree(batch, nodes, spread(rng, 1, max(2, most)), rng.choice([0, 0, 16, 48, 64, 128]), heads, kv_heads, dim)
    if kind == "verify":
        return verify(spread(rng, 1, 8), spread(rng, 1, 32), rng.choice([32000, 32003, 128256, spread(rng, 100, 128256)]), rng.choice([1, 2, 4]), rng.random() < 0.7)
    if kind == "compact":
        return compact(spread(rng, 1, 16), spread(rng, 2, 64), spread(rng, 1, 2000), rng.choice([4, 16, 32]), rng.choice([128, 512, 1000, 1024]), rng.choice([0, 16, 64]))
    if kind == "pages":
        pages = spread(rng, 8, 256)
        return {"kind": kind, "pools": rng.choice([8, 24, 64]), "pages": pages, "copied": spread(rng, 1, max(1, min(40, pages // 2))), "page": rng.choice([16, 64]),
                "width": rng.choice([256, 1000, 1024])}
    rows, vocab = spread(rng, 1, 4096), rng.choice([32000, 32003, 128256, spread(rng, 100, 128256)])
    return distill(rows, vocab, spread(rng, 1, 128), rng.random() < 0.4, rng.choice([0.0, 0.0, 0.25, 0.5]), rng.choice([1.0, 1.0, 2.0, 0.7]), rng.choice([1.0, 0.5]))


# ------------------------------------------------------------------------------------------------------------------------ inputs
def of_case(case):
    """numbers that only the case fixes: lengths, trees and pages, from a generator of their own (`work` needs them too)"""
    return np.random.default_rng([case["batch"], case["nodes"], case.get("length", 0), case.get("vocab", 0)])


def lengths_of(case):
    """cached rows of each sequence: the first as long as the case says, the others down to a quarter of it"""
    r = of_case(case)
    return [case["length"]] + [max(1, int(case["length"] * r.uniform(0.25, 1.0))) for _ in range(case["batch"] - 1)]


def sizes_of(case):
    """nodes of each sequence's tree: the first is full, others may be smaller"""
    r = of_case(case)
    return [case["nodes"]] + [int(r.integers((case["nodes"] + 1) // 2, case["nodes"] + 1)) for _ in range(case["batch"] - 1)]


def parents_of(case, r):
    """[batch, nodes]: node 0 is the last token that is certain, children come after their parents and siblings side by side"""
    n, branch = case["nodes"], case.get("branch", 3)
    out = np.full((case["batch"], n), -1, np.int64)
    for b in range(case["batch"]):
        out[b, 1:] = np.sort([max(0, (i - 1) // branch - int(r.integers(0, 2)) * (branch > 1)) for i in range(1, n)])
    return out


def words_of(parents):
    """[batch, nodes, words] int64: bit j of row i says that node i sees node j (itself and its ancestors)"""
    batch, n = parents.shape
    sees = np.zeros((batch, n, -(-n // 64) * 64), bool)
    for b in range(batch):
        for i in range(n):
            if parents[b, i] >= 0:
                sees[b, i] = sees[b, parents[b, i]]
            sees[b, i, i] = True
    return np.packbits(sees, axis=-1, bitorder="little").view("<i8").reshape(batch, n, -1)


def tables_of(lengths, extra, page, r):
    """a page table [batch, most pages] of pages in random order, and the pages of the pool"""
    need = [-(-(n + extra) // page) for n in lengths]
    order = r.permutation(sum(need) + 3)
    table = np.full((len(lengths), max(need)), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    st = {"case": case}
    if case["kind"] == "tree":
        B, T, H, G, D = case["batch"], case["nodes"], case["heads"], case["kv_heads"], case["dim"]
        lengths = lengths_of(case)
        st["q"] = rnd(B, T, H, D).mul_(1.5).to(BF16)
        if case["page"]:
            table, pages = tables_of(lengths, T, case["page"], r)
            st["table"], shape = dev(table, torch.int32), (pages, case["page"], G, D)
        else:
            st["table"], shape = None, (B, -(-(max(lengths) + T) // 2048) * 2048, G, D)
        st["k"], st["v"] = (torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=g) for _ in range(2))
        st["lengths"], st["nodes"] = dev(lengths, torch.int32), dev(sizes_of(case), torch.int32)
        st["mask"] = dev(words_of(parents_of(case, r)))
        st["out"] = rnd(B, T, H, D).mul_(1e-3).to(BF16)         # rows behind a small tree stay as they were
    elif case["kind"] == "verify":
        B, T, V = case["batch"], case["nodes"], case["vocab"]
        parents = parents_of(case, r)
        z = rnd(B, T, V).mul_(3)
        d = z + rnd(B, T, V).mul_(0.7)
        st["target"], st["draft"] = torch.softmax(z, -1), torch.softmax(d, -1) if case["drawn"] else None
        of = dev(np.maximum(parents, 0))[:, :, None].expand(B, T, V)
        noise = torch.empty(B, T, V, device="cuda").exponential_(generator=g).log_().neg_()
        st["tokens"] = (d.gather(1, of) + noise).argmax(-1)    # a node's token is drawn from its parent's distribution
        st["parents"], st["nodes"] = dev(parents, torch.int32), dev(sizes_of(case), torch.int32)
        st["uniform"] = torch.rand(B, T, generator=g, device="cuda")
    elif case["kind"] == "compact":
        B, T, W, n = case["batch"], case["nodes"], case["width"], 2 * case["layers"]
        lengths = lengths_of(case)
        if case["page"]:
            table, pages = tables_of(lengths, T, case["page"], r)
            st["table"], shape = dev(table, torch.int32), (n, pages, case["page"], W)
        else:
            st["table"], shape = None, (n, B, -(-(max(lengths) + T) // 512) * 512, W)
        st["kv"] = torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=g)
        # the accepted path of a tree numbered level by level: every node past the first level lies behind the rows that it moves to
        count = r.integers(2, max(3, min(9, T // 2 + 1)), B)
        path = np.full((B, T), -1, np.int64)
        for b in range(B):
            path[b, 0] = 0
            c = min(int(count[b]), T // 2 + 1)
            path[b, 1:c] = np.sort(r.choice(np.arange(c, T), c - 1, replace=False)) if T - c >= c - 1 else np.arange(1, c)
            count[b] = c
        st["path"], st["count"], st["lengths"] = dev(path, torch.int32), dev(count, torch.int32), dev(lengths, torch.int32)
    elif case["kind"] == "pages":
        st["kv"] = torch.empty((case["pools"], case["pages"], case["page"], case["width"]), dtype=BF16, device="cuda").normal_(generator=g)
        order = r.permutation(case["pages"])
        st["src"], st["dst"] = dev(order[:case["copied"]], torch.int32), dev(order[-case["copied"]:], torch.int32)
    else:
        R, V, K = case["rows"], case["vocab"], min(case["top"], case["vocab"])
        padded = -(-V // 8) * 8
        z = rnd(R, padded).mul_(2.5)
        st["logits"] = z.to(BF16) if case["bf16"] else z
        # the teacher's best lie high in the student's logits too; a few entries at a row's end are missing
        places = torch.stack([torch.randperm(V, generator=g, device="cuda")[:K] for _ in range(min(R, 64))])
        ids = (places[torch.arange(R, device="cuda") % places.shape[0]] + torch.arange(R, device="cuda")[:, None] * 131) % V
        t = torch.sort(rnd(R, K).mul_(2), -1, descending=True).values
        some = torch.randint(max(1, K // 2), K + 1, (R, 1), generator=g, device="cuda")
        st["ids"], st["teacher"] = torch.where(torch.arange(K, device="cuda")[None] < some, ids, -1), t
        st["logits"].scatter_add_(1, ids, t.to(st["logits"].dtype))
        on = dev(np.arange(R) < math.ceil(R * case["share"]))[torch.randperm(R, generator=g, device="cuda")]
        st["weight"] = on.float() / on.sum()
        st["target"] = torch.randint(0, V, (R,), generator=g, device="cuda") if case["hard"] else None
    return st


# ------------------------------------------------------------------------------------------------------------------------ one pass
def run(st):
    return {"tree": run_tree, "verify": run_verify, "compact": run_compact, "pages": run_pages, "distill": run_distill}[st["case"]["kind"]](st)


def run_tree(st):
    if own:
        from leopard_b200 import ops
        return ops.tree_attention(st["q"], st["k"], st["v"], st["lengths"], st["mask"], nodes=st["nodes"], page_table=st["table"], out=st["out"])
    q, lengths, out = st["q"], st["lengths"].long(), st["out"]
    B, T, H, D = q.shape
    G = st["k"].shape[2]
    most = st["case"]["length"] + T
    at = torch.arange(most, device="cuda")
    if st["table"] is None:
        k, v = st["k"][:, :most], st["v"][:, :most]
    else:
        size = st["case"]["page"]
        page = st["table"].long()[:, at // size].clamp(min=0)
        k, v = st["k"][page, at % size], st["v"][page, at % size]
    node = at[None] - lengths[:, None]                          # [B, most]: the node that a row holds, negative in the past
    word = st["mask"][torch.arange(B, device="cuda")[:, None], :, (node.clamp(0, T - 1) // 64)].transpose(1, 2)
    sees = (node < 0)[:, None] | ((node >= 0) & (node < st["nodes"][:, None]))[:, None] & ((word >> (node.clamp(0, T - 1) % 64)[:, None]) & 1).bool()
    s = torch.einsum("btghd,bkgd->bghtk", q.float().view(B, T, G, H // G, D), k.float()) * D ** -0.5
    s = s.masked_fill_(~sees[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1)
    o = torch.einsum("bghtk,bkgd->bghtd", p, v.float()) / torch.where(total > 0, total, 1.0)[..., None]
    there = torch.arange(T, device="cuda")[None] < st["nodes"][:, None]
    return out.copy_(torch.where(there[:, :, None, None], o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(BF16), out))


def run_verify(st):
    if own:
        from leopard_b200 import ops
        return ops.verify_draft(st["target"], st["tokens"], st["parents"], st["uniform"], draft=st["draft"], nodes=st["nodes"])
    target, draft, tokens, parents, u = st["target"], st["draft"], st["tokens"], st["parents"], st["uniform"].double()
    B, T, V = target.shape
    rows = torch.arange(B, device="cuda")
    cur, p = torch.zeros(B, dtype=torch.long, device="cuda"), target[:, 0].double()
    accepted = [torch.ones(B, dtype=torch.bool, device="cuda")]
    for c in range(1, T):                                       # children come after their parents: one sweep over the nodes is the walk
        child = (parents[:, c] == cur) & (c < st["nodes"])
        x = tokens[:, c:c + 1]
        q = draft[rows, cur].double() if draft is not None else torch.zeros_like(p).scatter_(1, x, 1.0)
        yes = child & (u[:, c] * q.gather(1, x)[:, 0] < p.gather(1, x)[:, 0])
        rest = (p - q).clamp_(min=0)
        total = rest.sum(-1, keepdim=True)
        p = torch.where((child & ~yes)[:, None] & (total > 0), rest / total, p)
        p = torch.where(yes[:, None], target[:, c].double(), p)
        cur = torch.where(yes, c, cur)
        accepted.append(yes)
    on = torch.stack(accepted, 1)
    place = torch.where(on, on.cumsum(1) - 1, T)
    path = torch.full((B, T + 1), -1, device="cuda").scatter_(1, place, torch.arange(T, device="cuda").expand(B, T))
    path[:, T] = -1
    below = p.cumsum(-1)
    token = (below > u[:, :1] * below[:, -1:]).int().argmax(-1)
    return path[:, :T].int(), on.sum(1).int(), token


def run_compact(st):
    if own:
        from leopard_b200 import ops
        return ops.cache_compact(st["kv"], st["lengths"], st["path"], st["count"], page_table=st["table"])
    kv, path = st["kv"], st["path"].long()
    B, T = path.shape
    size = st["case"]["page"] or kv.shape[2]
    j = torch.arange(T, device="cuda")[None].expand(B, T)
    on = j < st["count"][:, None]
    src, dst = (st["lengths"].long()[:, None] + torch.where(on, w, 0) for w in (path, j))
    # entries behind the count move each sequence's first row to itself
    table = st["table"].long() if st["table"] is not None else torch.arange(B, device="cuda")[:, None]
    src, dst = (table.gather(1, x // size) * size + x % size for x in (src, dst))
    flat = kv.view(kv.shape[0], -1, kv.shape[-1])
    flat[:, dst.reshape(-1)] = flat[:, src.reshape(-1)]
    return kv


def run_pages(st):
    if own:
        from leopard_b200 import ops
        return ops.cache_copy_pages(st["kv"], st["src"], st["dst"])
    st["kv"][:, st["dst"].long()] = st["kv"][:, st["src"].long()]
    return st["kv"]


def run_distill(st):
    case, V = st["case"], st["case"]["vocab"]
    hard, tau = case["hard"], case["tau"]
    if own:
        from leopard_b200 import ops
        return ops.distill_fwd_bwd(st["logits"], st["ids"], st["teacher"], st["weight"], V, temperature=tau, target=st["target"], hard=hard)
    on = st["weight"] != 0
    z = st["logits"][:, :V].float()
    there = st["ids"] >= 0
    ids = st["ids"].clamp(min=0)
    lt = torch.log_softmax((st["teacher"].float() / tau).masked_fill(~there, float("-inf")), -1)
    t = lt.exp()
    lp = torch.log_softmax(z / tau, -1)
    loss = (1 - hard) * tau * tau * torch.where(there, t * (lt - lp.gather(1, ids)), 0.0).sum(-1)
    d = lp.exp_().scatter_add_(1, ids, -t).mul_((1 - hard) * tau)
    if hard:
        lh = torch.log_softmax(z, -1)
        loss = loss - hard * lh.gather(1, st["target"][:, None])[:, 0]
        d += hard * lh.exp_().scatter_add_(1, st["target"][:, None], torch.full_like(loss, -1.0)[:, None])
    out = torch.zeros(st["logits"].shape, dtype=BF16, device="cuda")
    out[:, :V] = d * st["weight"][:, None]
    return torch.where(on, loss, 0.0), out


# ------------------------------------------------------------------------------------------------------------------------ what is needed
def work(case):
    if case["kind"] == "tree":
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        rows = sum(n + t for n, t in zip(lengths_of(case), sizes_of(case)))
        q = sum(sizes_of(case)) * H * D
        return {"bytes": 4 * rows * G * D + 4 * q, "flops": sum(4 * t * H * D * (n + t // 2) for n, t in zip(lengths_of(case), sizes_of(case)))}
    if case["kind"] == "verify":                                # the last row of each sequence, and a word of the others
        passes = 2 if case["drawn"] else 1
        return {"bytes": case["batch"] * (4 * passes * case["vocab"] + case["nodes"] * (4 * passes + 20)), "flops": 3 * case["batch"] * case["vocab"]}
    if case["kind"] == "compact":
        moved = case["batch"] * max(1, min(5, case["nodes"] // 2))
        return {"bytes": moved * 2 * case["layers"] * case["width"] * 2 * 2, "flops": 0}
    if case["kind"] == "pages":
        return {"bytes": 2 * case["copied"] * case["pools"] * case["page"] * case["width"] * 2, "flops": 0}
    R, V = case["rows"], case["vocab"]
    on = math.ceil(R * case["share"])
    return {"bytes": on * V * (2 if case["bf16"] else 4) + R * V * 2 + 12 * on * case["top"], "flops": 6 * on * V}


# ------------------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "tree":
        out = st["out"].double()
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        for b, (n, t) in enumerate(zip(lengths_of(case), sizes_of(case))):
            if st["table"] is None:
                k, v = st["k"][b, :n + t], st["v"][b, :n + t]
            else:
                pages = st["table"][b, :-(-(n + t) // case["page"])].long()
                k, v = (x[pages].reshape(-1, G, D)[:n + t] for x in (st["k"], st["v"]))
            bits = np.unpackbits(st["mask"][b].cpu().numpy().view(np.uint8), axis=-1, bitorder="little")[:t, :t]
            hidden = torch.zeros(t, n + t, device="cuda", dtype=F64)
            hidden[:, n:] = dev(np.where(bits, 0.0, -np.inf))
            for h in range(H):
                kh, vh = k[:, h // (H // G)].double(), v[:, h // (H // G)].double()
                w = torch.softmax(st["q"][b, :t, h].double() @ kh.T / math.sqrt(D) + hidden, -1)
                out[b, :t, h] = w @ vh
        return out
    if kind == "verify":
        host = {k: None if st[k] is None else st[k].cpu().numpy() for k in ("target", "draft", "tokens", "parents", "nodes", "uniform")}
        B, T = host["tokens"].shape
        paths, counts, nexts = np.full((B, T), -1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.int64)
        for b in range(B):
            cur, walk, p = 0, [0], host["target"][b, 0].astype(np.float64)
            while cur is not None:
                found = None
                for c in (c for c in range(cur + 1, int(host["nodes"][b])) if host["parents"][b, c] == cur):
                    x = host["tokens"][b, c]
                    q = host["draft"][b, cur].astype(np.float64) if host["draft"] is not None else np.eye(1, p.size, x)[0]
                    if np.float64(host["uniform"][b, c]) * q[x] < p[x]:
                        found = c
                        break
                    left = np.maximum(p - q, 0)
                    p = left / left.sum() if left.sum() > 0 else p
                if found is not None:
                    walk.append(found)
                    p = host["target"][b, found].astype(np.float64)
                cur = found
            paths[b, :len(walk)], counts[b] = walk, len(walk)
            c = np.cumsum(p)
            nexts[b] = int(np.searchsorted(c, np.float64(host["uniform"][b, 0]) * c[-1], side="right"))
        return paths, counts, nexts
    if kind == "compact":
        kv, size = st["kv"].clone(), case["page"] or st["kv"].shape[2]
        where = lambda b, i: (b if st["table"] is None else int(st["table"][b, i // size]), i % size)  # noqa: E731
        for b, n in enumerate(lengths_of(case)):
            for j in range(int(st["count"][b])):
                (sp, sr), (dp, dr) = where(b, n + int(st["path"][b, j])), where(b, n + j)
                kv[:, dp, dr] = st["kv"][:, sp, sr]
        return kv
    if kind == "pages":
        kv = st["kv"].clone()
        for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
            kv[:, d] = st["kv"][:, s]
        return kv
    V, hard, tau = case["vocab"], case["hard"], case["tau"]
    loss, grad = [], []
    for a in range(0, case["rows"], 256):
        z, ids, w = st["logits"][a:a + 256, :V].double(), st["ids"][a:a + 256], st["weight"][a:a + 256].double()
        there = ids >= 0
        e = torch.where(there, torch.exp(st["teacher"][a:a + 256].double() / tau), 0.0)
        t = e / e.sum(-1, keepdim=True)
        lse = torch.logsumexp(z / tau, -1, keepdim=True)
        at = z.gather(1, ids.clamp(min=0)) / tau - lse
        soft = torch.where(there, t * (torch.log(t) - at), 0.0).sum(-1) * tau * tau
        d = torch.exp(z / tau - lse)
        d.scatter_add_(1, ids.clamp(min=0), torch.where(there, -t, 0.0))
        one, d = (1 - hard) * soft, d * (1 - hard) * tau
        if hard:
            y, lz = st["target"][a:a + 256, None], torch.logsumexp(z, -1, keepdim=True)
            one = one + hard * (lz - z.gather(1, y))[:, 0]
            g = torch.exp(z - lz)
            g.scatter_add_(1, y, -torch.ones_like(lz))
            d = d + hard * g
        loss.append(torch.where(w != 0, one, 0.0))
        grad.append(torch.nn.functional.pad(d * w[:, None], (0, st["logits"].shape[1] - V)))
    return torch.cat(loss), torch.cat(grad)
