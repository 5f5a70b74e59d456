"""Serving many continuations of one prompt in 64 bits, from the definitions: step tables, rotary positions and cache rows, attention over a shared prefix, token draws.
Test infrastructure; torch on any device, loops where they say it most plainly."""
import math

import torch

F64 = torch.float64


def step_tables(lengths, new, page_table, free, used, page_size, rows):
    """-> (row_seq, row_pos, slots, row0, page_table, used) as lists; the arguments stay as they are"""
    table, used = [list(map(int, r)) for r in page_table], int(used[0])
    used = min(max(used, 0), len(free))
    seq, pos, slots, row0 = [], [], [], [0]
    for b, (n, t) in enumerate(zip(lengths.tolist(), new.tolist())):
        n, t = max(n, 0), max(t, 0)
        for page in range(n // page_size, -(-(n + t) // page_size) if t else 0):
            if page < len(table[b]) and table[b][page] < 0 and used < len(free):
                table[b][page] = int(free[used])
                used += 1
        for i in range(n, n + t):
            page = table[b][i // page_size] if i // page_size < len(table[b]) else -1
            seq.append(b)
            pos.append(i)
            slots.append(page * page_size + i % page_size if page >= 0 else -1)
        row0.append(row0[-1] + t)
    pad = [-1] * max(0, rows - len(seq))
    return (seq + pad)[:rows], (pos + pad)[:rows], (slots + pad)[:rows], row0, table, used


def rotary(x, positions, inv_freq, layout="half", scale=1.0, inverse=False):
    """-> (y, size): y in 64 bits, size = scale (|x_i| + |x_i'|) of each value's pair, what roundings are relative to"""
    n = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()[None]
    c, s = (torch.cos(angle) * scale)[:, None], (torch.sin(angle) * scale * (-1 if inverse else 1))[:, None]
    x = x.double()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if layout == "interleaved" else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = abs(scale) * (a.abs() + b.abs())
    return y, size


def append(pool, x, slots):
    """rows of x at their slots of pool [pages, page_size, heads, D], in place"""
    size = pool.shape[1]
    for r, slot in enumerate(slots.tolist()):
        if 0 <= slot < pool.shape[0] * size:
            pool[slot // size, slot % size] = x[r]
    return pool


def prefix_attention(q, k, v, lengths, prefix, new=None, page_table=None, prefix_k=None, prefix_v=None, scale=None):
    """-> (out, weight): out [B, T, H, D] in 64 bits, weight its sum with |v| in the place of v (what roundings of the weights are relative to)"""
    B, T, H, D = q.shape
    P, S, G, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    out, weight = torch.zeros(B, T, H, D, dtype=F64, device=q.device), torch.zeros(B, T, H, D, dtype=F64, device=q.device)

    def rows(b, first, last):
        """rows [first, last) of request b's pages that are there, and which"""
        at = [(i, int(page_table[b, i // S]) if page_table is not None else b, i % S if page_table is not None else i) for i in range(first, last)]
        at = [x for x in at if 0 <= x[1] < P]
        i, page, row = (torch.tensor([x[n] for x in at], dtype=torch.long, device=q.device) for n in range(3))
        return i, k[page, row].double(), v[page, row].double()
    room = S if page_table is None else S * page_table.shape[1]
    for b in range(B):
        n = T if new is None else max(0, min(T, int(new[b])))
        past = max(0, int(lengths[b]) - prefix)
        if page_table is not None:
            i0, k0, v0 = rows(0, 0, min(prefix, room))
            i1, k1, v1 = rows(b, prefix, min(prefix + past + n, room))
            i1 = i1 - prefix
        else:
            i0, k0, v0 = (torch.arange(prefix, device=q.device), prefix_k.double(), prefix_v.double()) if prefix else (torch.arange(0, device=q.device), k[b, :0].double(), v[b, :0].double())
            i1, k1, v1 = rows(b, 0, min(past + n, room))
        see = torch.cat([torch.ones(n, len(i0), dtype=torch.bool, device=q.device), i1[None] <= past + torch.arange(n, device=q.device)[:, None]], 1)
        kb, vb = torch.cat([k0, k1]), torch.cat([v0, v1])
        if not kb.shape[0]:
            continue
        for h in range(H):
            s = scale * (q[b, :n, h].double() @ kb[:, h // (H // G)].T)
            s = torch.where(see, s, -torch.inf)
            top = s.amax(-1, keepdim=True)
            w = torch.where(see, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
            total = w.sum(-1, keepdim=True)
            w = torch.where(total == 0, 0.0, w / total)
            seen = torch.where(see[:, :, None], w[:, :, None] * vb[None, :, h // (H // G)], 0.0)      # what a row does not see has no part in it
            out[b, :n, h], weight[b, :n, h] = seen.sum(1), seen.abs().sum(1)
    return out, weight


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """-> list of tokens"""
    out = []
    of = lambda x, i: float(torch.as_tensor(x, dtype=torch.float32).flatten()[i if torch.is_tensor(x) else 0])  # noqa: E731
    for i, row in enumerate(logits.double().cpu()):
        t, k, p, least = of(temperature, i), int(top_k[i]) if torch.is_tensor(top_k) else top_k, of(top_p, i), of(min_p, i)
        z = [(-math.inf if math.isnan(x) else x) for x in row.tolist()]
        top = max(z)
        if top == -math.inf:
            out.append(-1)
            continue
        if not t > 0:
            out.append(z.index(top))
            continue
        words = sorted((v for v in range(len(z)) if z[v] > -math.inf and (top < math.inf or z[v] == top)), key=lambda v: (-z[v], v))
        weight = {v: 1.0 if z[v] == top else math.exp((z[v] - top) / t) for v in words}
        if k > 0:
            words = words[:k]
        if p < 1:
            mass, all_of, kept = 0.0, math.fsum(weight[v] for v in words), []
            for v in words:
                if kept and not mass < p * all_of:
                    break
                kept.append(v)
                mass += weight[v]
            words = kept
        words = sorted(v for v in words if weight[v] >= min(max(least, 0.0), 1.0))
        limit, mass = float(uniform[i]) * math.fsum(weight[v] for v in words), 0.0
        for v in words:
            mass += weight[v]
            if mass > limit:
                break
        out.append(v)
    return out
