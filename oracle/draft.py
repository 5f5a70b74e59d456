"""Drafting in 64 bits, from the definitions: attention of a tree of nodes over a cache, verification of drafted tokens, cache rows, distillation.
Test infrastructure; torch on any device, loops where they say it most plainly."""
import torch

F64 = torch.float64


def tree_sees(parents):
    """[B, T] parents -> bool [B, T, T]: node i sees itself and its ancestors; a parent that does not lie before its child ends the walk."""
    B, T = parents.shape
    sees = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            at = i
            while at >= 0:
                sees[b, i, at] = True
                up = int(parents[b, at])
                at = up if up < at else -1
    return sees


def tree_words(sees):
    """bool [B, T, T] -> int64 [B, T, ceil(T / 64)]"""
    B, T, _ = sees.shape
    words = -(-T // 64)
    out = torch.zeros(B, T, words, dtype=torch.int64)
    for j in range(T):
        bit = 1 << (j % 64)
        out[:, :, j // 64] |= sees[:, :, j].long() * (bit - (1 << 64) if bit >= 1 << 63 else bit)
    return out


def tree_attention(q, k, v, lengths, sees, nodes=None, page_table=None, scale=None):
    """-> (out, weight): out [B, T, H, D] in 64 bits, weight its sum with |v| in the place of v (what roundings of the weights are relative to)"""
    B, T, H, D = q.shape
    P, S, G, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    out, weight = torch.zeros(B, T, H, D, dtype=F64, device=q.device), torch.zeros(B, T, H, D, dtype=F64, device=q.device)
    for b in range(B):
        n = T if nodes is None else max(0, min(T, int(nodes[b])))
        past = max(0, int(lengths[b]))
        cap = S * (1 if page_table is None else page_table.shape[1])
        keys = [i for i in range(min(past + n, cap))]
        place = [(b if page_table is None else int(page_table[b, i // S]), i % S) for i in keys]
        there = [i for i, (p, _) in zip(keys, place) if 0 <= p < P]
        if not there:
            continue
        pages = torch.tensor([place[i][0] for i in there], device=q.device)
        rows = torch.tensor([place[i][1] for i in there], device=q.device)
        kb, vb = k[pages, rows].double(), v[pages, rows].double()               # [keys, G, D]
        at = torch.tensor(there, device=q.device)
        see = torch.ones(n, len(there), dtype=torch.bool, device=q.device)
        tail = at >= past
        see[:, tail] = sees[b, :n].to(q.device)[:, at[tail] - past]
        for h in range(H):
            s = scale * (q[b, :n, h].double() @ kb[:, h // (H // G)].T)
            s = torch.where(see, s, -torch.inf)
            top = s.amax(-1, keepdim=True)
            w = torch.where(see, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
            total = w.sum(-1, keepdim=True)
            w = torch.where(total == 0, 0.0, w / total)
            vh = vb[:, h // (H // G)]
            seen = torch.where(see[:, :, None], w[:, :, None] * vh[None], 0.0)   # what a row does not see has no part in it
            out[b, :n, h], weight[b, :n, h] = seen.sum(1), seen.abs().sum(1)
    return out, weight


def verify_draft(target, tokens, parents, uniform, draft=None, nodes=None):
    """the walk of one sequence after the other, as the definition has it"""
    B, T, V = target.shape
    target, uniform = target.double().cpu().clamp(min=0).nan_to_num(0.0), uniform.double().cpu()
    draft = None if draft is None else draft.double().cpu().clamp(min=0).nan_to_num(0.0)
    paths, counts, tokens_out = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32), torch.full((B,), -1, dtype=torch.int64)
    for b in range(B):
        n = T if nodes is None else min(T, int(nodes[b]))
        if n <= 0:
            continue
        cur, walk, p = 0, [0], target[b, 0].clone()
        while True:
            found = -1
            for c in range(cur + 1, n):
                if int(parents[b, c]) != cur:
                    continue
                x = int(tokens[b, c])
                if not 0 <= x < V:
                    continue
                qx = 1.0 if draft is None else float(draft[b, cur, x])
                if float(uniform[b, c]) * qx < float(p[x]):
                    found = c
                    break
                left = p.clone()
                if draft is None:
                    left[x] = max(0.0, float(left[x]) - 1.0)
                else:
                    left = (left - draft[b, cur]).clamp(min=0)
                if float(left.sum()) > 0:
                    p = left / left.sum()
            if found < 0:
                break
            walk.append(found)
            cur, p = found, target[b, found].clone()
        paths[b, :len(walk)], counts[b] = torch.tensor(walk, dtype=torch.int32), len(walk)
        below = p.cumsum(0)
        hit = torch.nonzero(below > float(uniform[b, 0]) * float(below[-1]))
        tokens_out[b] = int(hit[0]) if hit.numel() else -1
    return paths, counts, tokens_out


def cache_compact(pool, lengths, path, count, page_table=None):
    """pool [pages, page_size, width] -> the pool with the accepted rows in their places"""
    P, S, _ = pool.shape
    out = pool.clone()

    def place(b, i):
        if i < 0 or int(lengths[b]) < 0:
            return None
        at = int(lengths[b]) + i
        if at // S >= (1 if page_table is None else page_table.shape[1]):
            return None
        page = b if page_table is None else int(page_table[b, at // S])
        return (page, at % S) if 0 <= page < P else None
    for b in range(path.shape[0]):
        for j in range(min(int(count[b]), path.shape[1])):
            s, d = place(b, int(path[b, j])), place(b, j)
            if s is not None and d is not None:
                out[d] = pool[s]
    return out


def distill(logits, ids, teacher, weight, vocab, temperature=1.0, target=None, hard=0.0):
    """-> (loss, dlogits) in 64 bits"""
    z = logits[:, :vocab].double()
    R = z.shape[0]
    loss, grad = torch.zeros(R, dtype=F64, device=z.device), torch.zeros(logits.shape, dtype=F64, device=z.device)
    for r in range(R):
        w = float(weight[r])
        if w == 0:
            continue
        there = [k for k in range(ids.shape[1]) if 0 <= int(ids[r, k]) < vocab and float(teacher[r, k]) != -float("inf")]
        if there and hard < 1:
            at = ids[r, there].long()
            lt = torch.log_softmax(teacher[r, there].double() / temperature, -1)
            lp = torch.log_softmax(z[r] / temperature, -1)
            loss[r] += (1 - hard) * temperature ** 2 * (lt.exp() * (lt - lp[at])).sum()
            g = lp.exp()
            g.index_put_((at,), -lt.exp(), accumulate=True)
            grad[r, :vocab] += w * (1 - hard) * temperature * g
        if hard and target is not None and 0 <= int(target[r]) < vocab:
            lp = torch.log_softmax(z[r], -1)
            loss[r] -= hard * lp[int(target[r])]
            g = lp.exp()
            g[int(target[r])] -= 1
            grad[r, :vocab] += w * hard * g
    return loss, grad
