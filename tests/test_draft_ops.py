"""Drafting: trees of drafted tokens attended over a cache, verification, accepted rows and pages, distillation — each against its definition in 64 bits
(oracle/draft.py), at the sizes, masks and layouts where it can go wrong; refusals without a GPU."""
import ctypes as C
import math

import pytest
import torch

from leopard_b200 import _lib, ops
from oracle import draft as O

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def random_parents(B, T, seed, chain=False):
    g = gen(seed, "cpu")
    p = torch.full((B, T), -1, dtype=torch.int32)
    for i in range(1, T):
        p[:, i] = i - 1 if chain else (torch.rand(B, generator=g) * i).int().clamp(max=i - 1)
    return p


# ------------------------------------------------------------------------------------------------------------ refusals (no GPU)
def test_struct_layout_and_limits_match_the_header(tmp_path):
    import re
    import subprocess
    from pathlib import Path
    inc = Path(__file__).resolve().parents[1] / "include"
    lines = ['printf("%zu\\n", sizeof(lp_tree_attn_desc));'] + [f'printf("%zu\\n", offsetof(lp_tree_attn_desc, {n}));' for n, _ in _lib.TreeAttnDesc._fields_]
    src = tmp_path / "a.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "leopard_b200.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-I", str(inc), str(src), "-o", str(tmp_path / "a")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(_lib.TreeAttnDesc)] + [getattr(_lib.TreeAttnDesc, n).offset for n, _ in _lib.TreeAttnDesc._fields_]
    assert int(re.search(r"#define LP_TREE_MAX_NODES (\d+)", (inc / "leopard_b200.h").read_text())[1]) == _lib.TREE_MAX_NODES


def tree_desc(**kw):
    """a descriptor whose numbers are in order (its addresses are not touched before the checks are through)"""
    base = dict(q=1 << 20, q_batch=4096, q_node=1024, q_head=128, k=1 << 20, k_page=65536, k_row=256, k_head=128, v=1 << 20, v_page=65536, v_row=256, v_head=128,
                out=1 << 20, o_batch=4096, o_node=1024, o_head=128, page_table=1 << 20, ld_table=4, max_pages=4, n_pages=9, page_size=64, lengths=1 << 20,
                nodes=None, mask=1 << 20, mask_batch=4, mask_node=1, B=2, T=4, H=8, KVH=2, D=128, scale=0.1)
    return _lib.TreeAttnDesc(**{**base, **kw})


@pytest.mark.parametrize("change, word", [
    (dict(B=0), "B=0"), (dict(B=5000), "B=5000"), (dict(T=0), "T=0"), (dict(T=257), "T=257"), (dict(H=9), "9 query heads over 2"), (dict(KVH=0), "over 0"),
    (dict(D=72), "heads of 72"), (dict(page_size=0), "of 0 rows"), (dict(n_pages=0), "0 pages"), (dict(max_pages=0), "0 a sequence"),
    (dict(max_pages=1 << 20, page_size=1 << 12), "too many"), (dict(q=None), "null"), (dict(lengths=None), "null"), (dict(mask=None), "null"),
    (dict(ld_table=3), "ld_table 3"), (dict(page_table=None), "4 pages"), (dict(page_table=None, max_pages=1, n_pages=1), "1 pages there"),
    (dict(k_row=252), "multiples of 8"), (dict(q=(1 << 20) + 2), "16-byte aligned"),
])
def test_tree_attention_refusals(native_lib, change, word):
    d = tree_desc(**change)
    rc = native_lib.lp_tree_attention(C.byref(d), C.c_void_p(1 << 20), 1 << 40, None)
    assert rc == -1 and word in native_lib.lp_last_error().decode()


def test_tree_attention_refuses_a_small_workspace(native_lib):
    d = tree_desc()
    need = native_lib.lp_tree_attention_workspace_bytes(C.byref(d))
    assert need > 0
    assert native_lib.lp_tree_attention(C.byref(d), C.c_void_p(1 << 20), need - 1, None) == -1
    assert b"workspace too small" in native_lib.lp_last_error()
    assert native_lib.lp_tree_attention(C.byref(d), None, need, None) == -1


def test_other_refusals_are_status_codes(native_lib):
    p = C.c_void_p(1 << 20)
    L = native_lib
    assert L.lp_tree_mask(p, 3, 1, 4, p, None, None) == -1
    assert L.lp_tree_mask(p, 300, 1, 257, p, None, None) == -1
    assert L.lp_verify_draft(None, 0, 0, None, 0, 0, p, p, p, None, 1, 1, 5, p, p, p, None) == -1
    assert L.lp_verify_draft(p, 0, 0, None, 0, 0, p, p, p, None, 1, 1025, 5, p, p, p, None) == -1
    assert L.lp_verify_draft(p, 0, 0, None, 0, 0, p, p, p, None, 1, 4, 0, p, p, p, None) == -1
    one = (C.c_void_p * 1)(1 << 20)
    assert L.lp_cache_compact(one, 0, 1, 4096, 64, 64, 8, 64, None, 0, 2, p, p, 4, p, 1, 4, None) == -1            # no table, two pages a sequence
    assert L.lp_cache_compact(one, 0, 1, 4096, 64, 64, 8, 64, None, 0, 1, p, p, 4, p, 9, 4, None) == -1            # nine sequences, eight pages
    assert L.lp_cache_compact(one, 0, 1, 4096, 32, 64, 8, 64, p, 2, 2, p, p, 4, p, 1, 4, None) == -1               # rows overlap
    assert L.lp_cache_copy_pages(one, 0, 1, 64, 4096, 8, p, p, 1, None) == -1                                      # pages overlap
    assert L.lp_cache_copy_pages(one, 0, 0, 4096, 4096, 8, p, p, 1, None) == -1
    assert L.lp_cache_copy_pages(one, 0, 1, 4096, 4096, 8, p, p, 0, None) == 0                                     # nothing to do
    args = dict(K=4, temp=1.0, hard=0.0, target=None, V=10, Vp=10, ldd=10)

    def distill(**kw):
        a = {**args, **kw}
        return L.lp_distill_fwd_bwd(p, 1, 16, p, 1, 2000, p, 1, 2000, a["K"], p, a["target"], a["temp"], a["hard"], p, p, a["ldd"], 2, a["V"], a["Vp"], None)
    assert [distill(**kw) for kw in (dict(K=0), dict(K=1025), dict(temp=0.0), dict(temp=-1.0), dict(temp=float("nan")), dict(hard=0.5), dict(hard=1.5, target=p),
                                     dict(Vp=9, ldd=10), dict(V=11), dict(ldd=8))] == [-1] * 10


def test_wrappers_refuse_what_is_not_on_a_gpu():
    z = torch.zeros
    with pytest.raises(TypeError, match="parents"):
        ops.tree_mask(z(1, 4, dtype=torch.int32))
    with pytest.raises(TypeError, match="q must"):
        ops.tree_attention(z(1, 4, 8, 128, dtype=BF16), z(1, 64, 2, 128, dtype=BF16), z(1, 64, 2, 128, dtype=BF16), z(1, dtype=torch.int32), z(1, 4, 1, dtype=torch.int64))
    with pytest.raises(TypeError, match="target"):
        ops.verify_draft(z(1, 4, 10), z(1, 4, dtype=torch.int64), z(1, 4, dtype=torch.int32), z(1, 4))
    with pytest.raises(TypeError, match="pools"):
        ops.cache_compact(z(2, 3, 4, 8), z(1, dtype=torch.int32), z(1, 4, dtype=torch.int32), z(1, dtype=torch.int32))
    with pytest.raises(TypeError, match="logits"):
        ops.distill_fwd_bwd(z(2, 10), z(2, 3, dtype=torch.int64), z(2, 3), z(2), 10)


# ------------------------------------------------------------------------------------------------------------ trees
@gpu
@pytest.mark.parametrize("B, T, chain", [(1, 1, False), (3, 26, False), (2, 64, True), (2, 65, False), (1, 256, True), (5, 130, False)])
def test_tree_mask(B, T, chain):
    p = random_parents(B, T, B * 1000 + T, chain)
    mask, depth = ops.tree_mask(p.cuda())
    sees = O.tree_sees(p)
    assert torch.equal(mask.cpu(), O.tree_words(sees)) and torch.equal(depth.cpu(), (sees.sum(-1) - 1).int())


@gpu
def test_tree_mask_ends_walks_that_do_not_go_back():
    p = torch.tensor([[-1, 0, 2, 5, 3, -7]], dtype=torch.int32)
    mask, depth = ops.tree_mask(p.cuda())
    assert torch.equal(mask.cpu(), O.tree_words(O.tree_sees(p))) and depth.tolist() == [[0, 1, 0, 0, 1, 0]]


def attention_case(B, T, H, G, D, lengths, nodes=None, page=0, seed=0, chain=False, spare=2):
    g = gen(seed)
    c = {"q": (torch.randn(B, T, H, D, generator=g, device="cuda") * 1.5).to(BF16)}
    if page:
        need = [-(-(n + T) // page) for n in lengths]
        order = torch.randperm(sum(need) + spare, generator=gen(seed, "cpu")).int()
        table = torch.full((B, max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        c["page_table"], shape = table.cuda(), (sum(need) + spare, page, G, D)
    else:
        c["page_table"], shape = None, (B, max(lengths) + T + 5, G, D)
    c["k"], c["v"] = (torch.randn(shape, generator=g, device="cuda").to(BF16) for _ in range(2))
    c["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    c["nodes"] = None if nodes is None else torch.tensor(nodes, dtype=torch.int32, device="cuda")
    c["sees"] = O.tree_sees(random_parents(B, T, seed + 1, chain))
    return c


def attend(c, **kw):
    a = {k: c[k] for k in ("q", "k", "v", "lengths", "nodes", "page_table")}
    return ops.tree_attention(mask=O.tree_words(c["sees"]).cuda(), **{**a, **kw})


def close(got, c, scale=None, rows=None):
    """Roundings to bf16 (half a step is 2^-8 of the value): each weight before the second product, relative to the weights' sum of |v|, and the output.  Scores: a sum of D
    products in fp32 whose additions may be cut off (2^-23 of the sum of magnitudes each): delta, and weights move by 2 delta.  Weights and sums of fp32: under 2^-12."""
    want, weight = O.tree_attention(c["q"], c["k"], c["v"], c["lengths"], c["sees"], c["nodes"], c["page_table"], scale)
    D = c["q"].shape[-1]
    s = D ** -0.5 if scale is None else abs(scale)
    delta = s * c["q"].float().abs().sum(-1, keepdim=True).double() * float(c["k"][c["k"].isfinite()].float().abs().max()) * 2.0 ** -23
    tol = 2.0 ** -8 * (want.abs() + weight) + (2 * delta + 2.0 ** -12) * weight + 1e-30
    n = c["q"].shape[1]
    for b in range(want.shape[0]):
        t = n if c["nodes"] is None else int(c["nodes"][b])
        x, y = got[b, :t].double(), want[b, :t]
        same = (x == y) | (x.isnan() & y.isnan())
        bad = ~(same | ((x - y).abs() <= tol[b, :t]))
        assert not bad.any(), (b, torch.nonzero(bad)[:4].tolist(), float((x - y)[bad].abs().max()))


SHAPES = [
    # B, T, H, G, D, lengths, nodes, page
    (1, 1, 32, 8, 128, [0], None, 0), (1, 1, 32, 8, 128, [1], None, 0), (1, 1, 4, 4, 128, [700], None, 0), (1, 1, 32, 8, 128, [4796], None, 0),
    (1, 26, 32, 8, 128, [63], None, 0), (1, 26, 32, 8, 128, [64], None, 64), (2, 5, 8, 2, 64, [129, 38], None, 16), (3, 7, 12, 4, 96, [300, 0, 65], [7, 3, 0], 48),
    (4, 64, 32, 8, 128, [1021, 5, 511, 64], [64, 64, 1, 33], 64), (2, 70, 8, 1, 128, [130, 257], [70, 66], 64), (1, 256, 8, 2, 128, [333], None, 128),
    (2, 128, 4, 4, 64, [1000, 1], None, 0), (1, 3, 24, 8, 128, [2049], None, 1), (1, 13, 32, 8, 128, [20011], None, 64), (2, 9, 6, 2, 96, [31, 32], None, 5),
    (1, 100, 16, 1, 128, [77], None, 64), (33, 2, 8, 2, 64, list(range(33)), None, 16), (1, 2, 32, 1, 64, [64], None, 0),
]


@gpu
@pytest.mark.parametrize("B, T, H, G, D, lengths, nodes, page", SHAPES)
def test_tree_attention(B, T, H, G, D, lengths, nodes, page):
    c = attention_case(B, T, H, G, D, lengths, nodes, page, seed=T * 7 + D)
    out = torch.full((B, T, H, D), 7.0, dtype=BF16, device="cuda")
    got = attend(c, out=out)
    close(got, c)
    if nodes:
        for b, n in enumerate(nodes):                     # rows that a sequence does not have stay
            assert bool((got[b, n:] == 7.0).all())
    assert torch.equal(attend(c, out=torch.full_like(out, 7.0)), got)


@gpu
@pytest.mark.parametrize("scale", [0.02, -0.07, 0.0])
def test_tree_attention_takes_any_scale(scale):
    c = attention_case(2, 9, 8, 2, 128, [200, 31], page=64, seed=5)
    close(attend(c, scale=scale), c, scale)


@gpu
def test_tree_attention_of_views():
    """heads as columns of a wider projection, keys and values as halves of one pool's rows"""
    c = attention_case(2, 11, 8, 2, 128, [150, 77], page=32, seed=6)
    qkv = torch.randn(2 * 11, 12 * 128 + 8, device="cuda", generator=gen(1)).to(BF16)
    q = qkv[:, :1024].view(2, 11, 8, 128)
    q.copy_(c["q"])
    pool = torch.randn(c["k"].shape[0], 32, 4, 128, device="cuda", generator=gen(2)).to(BF16)
    pool[:, :, :2], pool[:, :, 2:] = c["k"], c["v"]
    out = torch.zeros(11, 2, 8 * 128 + 16, dtype=BF16, device="cuda")
    got = attend(c, q=q, k=pool[:, :, :2], v=pool[:, :, 2:], out=out[:, :, 8:1032].unflatten(2, (8, 128)).transpose(0, 1))
    close(got, c)
    assert torch.equal(got, attend(c)) and bool((out[:, :, :8] == 0).all()) and bool((out[:, :, 1032:] == 0).all())


@gpu
@pytest.mark.parametrize("T, H, G", [(9, 8, 2), (40, 32, 8), (70, 8, 2)])
def test_rows_that_see_nothing_are_zeros_and_see_no_nan(T, H, G):
    c = attention_case(2, T, H, G, 128, [0, 0], page=64, seed=8)
    c["sees"][0, 3] = False                               # sees nothing at all
    c["sees"][1, :, :] = False
    got = attend(c)
    close(got, c)
    assert bool((got[0, 3] == 0).all()) and bool((got[1] == 0).all())
    # stale rows of the pool behind the nodes, and pages that nobody holds
    c = attention_case(2, T, H, G, 128, [100, 3], [T - 1, 2], page=64, seed=9)
    clean = attend(c)
    held = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for b, n in enumerate([100 + T - 1, 5]):
        for i in range(n):
            held[int(c["page_table"][b, i // 64]), i % 64] = True
    for t in (c["k"], c["v"]):
        t[~held.cuda()] = float("nan")
    again = attend(c)
    for b, n in enumerate([T - 1, 2]):
        assert torch.equal(again[b, :n], clean[b, :n])


@gpu
@pytest.mark.parametrize("past", [0, 50, 64, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("T", [9, 66])
def test_values_of_a_node_reach_the_rows_that_see_it_alone(past, bad, T):
    c = attention_case(1, T, 8, 2, 128, [past], page=16, seed=10)
    clean = attend(c).clone()
    node = 4
    at = past + node
    c["v"][int(c["page_table"][0, at // 16]), at % 16, 1, 5] = bad
    got = attend(c)
    sees = c["sees"][0, :, node]
    assert bool(sees.any()) and not bool(sees.all())
    for i in range(T):
        for h in range(8):
            hit = got[0, i, h, 5]
            if sees[i] and h >= 4:
                assert bool(hit.isnan()) if math.isnan(bad) else float(hit) == bad
                other = torch.arange(128, device="cuda") != 5
                assert torch.equal(got[0, i, h][other], clean[0, i, h][other])
            else:
                assert torch.equal(got[0, i, h], clean[0, i, h])
    # a key that is not finite: its own rows' affair too
    c["v"][int(c["page_table"][0, at // 16]), at % 16, 1, 5] = 0
    c["k"][int(c["page_table"][0, at // 16]), at % 16, 0, 3] = float("nan")
    got = attend(c)
    for i in range(T):
        assert bool(got[0, i, :4].isnan().all()) == bool(sees[i])


@gpu
def test_pages_that_are_not_there_are_not_seen():
    c = attention_case(2, 6, 8, 2, 64, [300, 200], page=32, seed=11)
    c["page_table"][0, 2] = -1
    c["page_table"][0, 5] = c["k"].shape[0]
    c["page_table"][1, 0] = -9
    close(attend(c), c)
    c["lengths"][1] = 32 * c["page_table"].shape[1] + 5    # longer than its table: what is there is seen, the nodes are not
    close(attend(c), c)
    c["lengths"][0] = -4                                   # as none
    close(attend(c), c)
    c["page_table"][:] = -1
    assert bool((attend(c) == 0).all())


@gpu
def test_one_page_of_many_sequences():
    """a shared prefix: the same pages stand in several tables, and twice in one"""
    c = attention_case(3, 4, 8, 2, 128, [128, 128, 128], page=64, seed=12)
    c["page_table"][1, :2] = c["page_table"][0, :2]
    c["page_table"][2, 1] = c["page_table"][2, 0]
    close(attend(c), c)


@gpu
@pytest.mark.parametrize("B, T, H, G, D", [(2048, 1, 2, 1, 64), (1024, 20, 4, 2, 64), (1025, 33, 1, 1, 96)])
def test_the_largest_batches(B, T, H, G, D):
    c = attention_case(B, T, H, G, D, [(i * 37) % 90 for i in range(B)], page=16, seed=B)
    close(attend(c), c)


@gpu
def test_offsets_beyond_32_bits():
    """a pool of 4.5 GB: its last pages lie past 2^32 bytes and 2^31 elements"""
    pages = 70000
    k = torch.zeros(pages, 64, 4, 128, dtype=BF16, device="cuda")
    c = attention_case(1, 5, 8, 4, 128, [130], page=64, seed=13)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    for i in range(3):
        k[int(table[0, i])] = c["k"][int(c["page_table"][0, i])]
    v = torch.zeros_like(k)
    for i in range(3):
        v[int(table[0, i])] = c["v"][int(c["page_table"][0, i])]
    assert torch.equal(attend(c, k=k, v=v, page_table=table), attend(c))


@gpu
def test_tree_attention_wrapper_refusals():
    c = attention_case(2, 4, 8, 2, 128, [20, 30], page=16, seed=14)
    for change, err in ((dict(q=c["q"].float()), TypeError), (dict(k=c["k"][..., :64]), ValueError), (dict(lengths=c["lengths"].long()), TypeError),
                        (dict(lengths=c["lengths"][:1]), ValueError), (dict(page_table=c["page_table"][:1]), ValueError), (dict(nodes=c["lengths"][:1]), ValueError),
                        (dict(out=c["q"]), ValueError), (dict(q=c["q"].transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
                        (dict(q=torch.zeros(2, 4, 9, 128, dtype=BF16, device="cuda")), _lib.NativeError), (dict(out=c["q"][:1]), ValueError)):
        with pytest.raises(err):
            attend(c, **change)
    with pytest.raises(ValueError):
        ops.tree_attention(c["q"], c["k"], c["v"], c["lengths"], torch.zeros(2, 4, 2, dtype=torch.int64, device="cuda"), page_table=c["page_table"])
    with pytest.raises(ValueError):                        # more sequences than caches of their own
        ops.tree_attention(c["q"], c["k"][:1], c["v"][:1], c["lengths"], O.tree_words(c["sees"]).cuda())
    assert ops.tree_attention(c["q"][:0], c["k"], c["v"], c["lengths"][:0], O.tree_words(c["sees"]).cuda()[:0], page_table=c["page_table"][:0]).shape == (0, 4, 8, 128)


# ------------------------------------------------------------------------------------------------------------ verification
def verify_case(B, T, V, seed, drawn=True, spread=0.7, chain=False):
    g = gen(seed)
    parents = random_parents(B, T, seed, chain)
    z = torch.randn(B, T, V, generator=g, device="cuda") * 3
    d = z + torch.randn(B, T, V, generator=g, device="cuda") * spread
    of = parents.clamp(min=0).long().cuda()[:, :, None].expand(B, T, V)
    noise = torch.empty(B, T, V, device="cuda").exponential_(generator=g).log_().neg_()
    return dict(target=torch.softmax(z, -1), tokens=(d.gather(1, of) + noise).argmax(-1), parents=parents.cuda(), uniform=torch.rand(B, T, generator=g, device="cuda"),
                draft=torch.softmax(d, -1) if drawn else None)


def same(got, want):
    for x, y in zip(got, want):
        assert torch.equal(x.cpu(), y), (x.cpu(), y)


@gpu
@pytest.mark.parametrize("B, T, V", [(1, 1, 1), (1, 1, 32003), (2, 2, 5), (5, 6, 33), (3, 17, 1000), (2, 32, 32000), (40, 4, 100), (1, 64, 128256), (2, 200, 77), (2, 12, 131072), (2, 12, 131073), (3, 9, 4097),
                                     (1, 5, 400007)])
@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("chain", [True, False])
def test_verify_draft(B, T, V, drawn, chain):
    for seed in range(3):
        c = verify_case(B, T, V, seed * 100 + T, drawn, 0.7 if seed else 3.0, chain)
        nodes = None if seed == 0 else torch.randint(0, T + 1, (B,), generator=gen(seed, "cpu"), dtype=torch.int32)
        same(ops.verify_draft(**c, nodes=None if nodes is None else nodes.cuda()), O.verify_draft(**c, nodes=nodes))


@gpu
def test_verify_draft_at_the_borders():
    V = 40
    t = torch.zeros(1, 4, V, device="cuda")
    t[0, 0, 3], t[0, 0, 9] = 0.25, 0.75
    t[0, 1, 5] = t[0, 2, 6] = t[0, 3, 7] = 1.0
    parents = torch.tensor([[-1, 0, 0, 0]], dtype=torch.int32, device="cuda")

    def go(tokens, uniform, draft=None, target=t, parents=parents):
        c = dict(target=target, tokens=torch.tensor([tokens], device="cuda"), parents=parents, uniform=torch.tensor([uniform], device="cuda"), draft=draft)
        got = ops.verify_draft(**c)
        same(got, O.verify_draft(**c))
        return [x.tolist()[0] for x in got]
    # u equal to p is not below it; the first token whose running sum is above u, the border itself goes to the next
    assert go([0, 3, 9, 9], [0.0, 0.25, 0.999, 0.5]) == [[0, 2, -1, -1], 2, 6]
    assert go([0, 8, 8, 8], [0.25, 0.0, 0.0, 0.0]) == [[0, -1, -1, -1], 1, 9]
    assert go([0, 8, 8, 8], [0.2499999, 0.0, 0.0, 0.0]) == [[0, -1, -1, -1], 1, 3]
    # the same token twice: refused once, it is gone
    assert go([0, 3, 3, 3], [0.1, 0.9, 0.0, 0.0]) == [[0, -1, -1, -1], 1, 9]
    # all the mass refused: P stays
    assert go([0, 3, 9, 3], [0.1, 0.5, 0.999, 0.3]) == [[0, 2, -1, -1], 2, 6]
    one = torch.zeros(1, 4, V, device="cuda")
    one[:, :, 11] = 1.0
    assert go([0, 11, 2, 3], [0.4, 1.0, 0.0, 0.0], target=one) == [[0, -1, -1, -1], 1, 11]
    # tokens that are none, parents that never come, an empty distribution, negative and NaN probabilities
    assert go([0, -1, V, 1 << 40], [0.5, 0.0, 0.0, 0.0]) == [[0, -1, -1, -1], 1, 9]
    assert go([0, 9, 9, 9], [0.5, 0.0, 0.0, 0.0], parents=torch.tensor([[-1, 1, 3, 77]], dtype=torch.int32, device="cuda")) == [[0, -1, -1, -1], 1, 9]
    assert go([0, 9, 9, 9], [0.5, 0.0, 0.0, 0.0], target=torch.zeros_like(t)) == [[0, -1, -1, -1], 1, -1]
    odd = t.clone()
    odd[0, 0, 20], odd[0, 0, 1] = -3.0, float("nan")
    assert go([0, 20, 1, 9], [0.9, 0.0, 0.0, 0.7], target=odd) == [[0, 3, -1, -1], 2, 7]
    # equal distributions accept whatever u says
    assert go([0, 9, 9, 9], [0.9, 0.99999994, 0.0, 0.0], draft=t.clone()) == [[0, 1, -1, -1], 2, 5]


@gpu
def test_verify_draft_keeps_the_targets_distribution():
    """the next token after one drafted one is distributed as the target says: frequencies over 40,000 sequences, five standard deviations"""
    B, V = 40000, 7
    g = gen(3)
    p, q = torch.softmax(torch.randn(V, generator=g, device="cuda"), -1), torch.softmax(torch.randn(V, generator=g, device="cuda"), -1)
    tokens = torch.stack([torch.zeros(B, dtype=torch.int64, device="cuda"), torch.multinomial(q, B, True, generator=g), torch.multinomial(q, B, True, generator=g)], 1)
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32, device="cuda").repeat(B, 1)
    path, count, nxt = ops.verify_draft(p.expand(B, 3, V).contiguous(), tokens, parents, torch.rand(B, 3, generator=g, device="cuda"), draft=q.expand(B, 3, V))
    first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
    freq = torch.bincount(first, minlength=V).double() / B
    assert bool(((freq - p.double()).abs() < 5 * (p.double() * (1 - p.double()) / B).sqrt()).all())


@gpu
def test_verify_draft_of_views_and_refusals():
    c = verify_case(3, 5, 50, 4)
    wide = torch.full((3, 7, 64), -1.0, device="cuda")
    wide[:, 1:6, 3:53] = c["target"]
    same(ops.verify_draft(**{**c, "target": wide[:, 1:6, 3:53]}), O.verify_draft(**c))
    for change, err in ((dict(target=c["target"].double()), TypeError), (dict(tokens=c["tokens"].int()), TypeError), (dict(uniform=c["uniform"][:, :4]), ValueError),
                        (dict(draft=c["draft"][:, :4]), ValueError), (dict(parents=c["parents"].t().contiguous().t()), ValueError),
                        (dict(target=c["target"].transpose(1, 2).contiguous().transpose(1, 2)), ValueError), (dict(nodes=torch.zeros(2, dtype=torch.int32, device="cuda")), ValueError)):
        with pytest.raises(err):
            ops.verify_draft(**{**c, **change})


# ------------------------------------------------------------------------------------------------------------ cache rows and pages
def compact_case(B, T, page, width, dtype, n, seed, lengths):
    g = gen(seed, "cpu")
    need = [-(-(x + T) // page) for x in lengths] if page else None
    shape = (n, sum(need) + 2, page, width) if page else (n, B, max(lengths) + T, width)
    pools = torch.randint(0, 250, shape, generator=g).to(dtype).cuda()
    table = None
    if page:
        order = torch.randperm(sum(need) + 2, generator=g).int()
        table, at = torch.full((B, max(need)), -1, dtype=torch.int32), 0
        for b, k in enumerate(need):
            table[b, :k] = order[at:at + k]
            at += k
        table = table.cuda()
    path, count = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        c = int(torch.randint(0, T + 1, (1,), generator=g))
        count[b] = c
        path[b, :c] = torch.randperm(T, generator=g)[:c].sort().values
    return pools, torch.tensor(lengths, dtype=torch.int32).cuda(), path.cuda(), count.cuda(), table


@gpu
@pytest.mark.parametrize("B, T, page, width, dtype, n, lengths", [
    (1, 5, 0, 128, BF16, 4, [7]), (3, 26, 16, 1024, BF16, 2, [40, 0, 15]), (2, 64, 48, 33, BF16, 3, [1, 100]), (2, 256, 64, 8, torch.float32, 2, [0, 63]),
    (4, 9, 1, 7, torch.uint8, 5, [0, 1, 2, 3]), (1, 3, 4, 6, BF16, 300, [5]), (2, 17, 0, 1000, torch.float32, 2, [3, 9]),
])
def test_cache_compact(B, T, page, width, dtype, n, lengths):
    for seed in range(3):
        pools, *rest = compact_case(B, T, page, width, dtype, n, seed, lengths)
        want = torch.stack([O.cache_compact(p, *rest) for p in pools])
        as_list = [p.clone() for p in pools]
        assert ops.cache_compact(pools, *rest) is pools and torch.equal(pools, want)
        ops.cache_compact(as_list, *rest)
        assert torch.equal(torch.stack(as_list), want)


@gpu
def test_cache_compact_leaves_what_is_not_there():
    pools, lengths, path, count, table = compact_case(2, 6, 4, 16, BF16, 2, 0, [5, 9])
    path[0], count[0] = torch.tensor([0, 2, 3, 5, 77, -3], dtype=torch.int32), 6
    path[1], count[1] = torch.tensor([1, 2, 3, 4, 5, -1], dtype=torch.int32), 99      # more than there are: T of them
    table[1, 3] = -1
    table[0, 2] = 1 << 30
    want = torch.stack([O.cache_compact(p, lengths, path, torch.tensor([4, 5]), table) for p in pools])
    ops.cache_compact(pools, lengths, path, count, table)
    assert torch.equal(pools, want)
    lengths[0], lengths[1] = -1, 2 ** 31 - 1
    ops.cache_compact(pools, lengths, path, count, table)
    assert torch.equal(pools, want)


@gpu
def test_cache_compact_of_the_decoders_cache():
    kv = torch.randn(3, 2, 40, 64, device="cuda", generator=gen(1)).to(BF16)
    lengths, path, count = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([20], [[0, 3, 4, 9, -1]], [4]))
    want = kv.clone()
    want[:, :, 20:24] = kv[:, :, [20, 23, 24, 29]]
    ops.cache_compact(kv.flatten(0, 1).unsqueeze(1), lengths, path, count)
    assert torch.equal(kv, want)


@gpu
@pytest.mark.parametrize("n, pages, page, width, dtype, copied", [(1, 2, 1, 1, torch.uint8, 1), (64, 40, 64, 1024, BF16, 13), (3, 9, 16, 33, BF16, 4), (300, 6, 4, 8, torch.float32, 3),
                                                                 (2, 8, 5, 7, torch.float32, 4)])
def test_cache_copy_pages(n, pages, page, width, dtype, copied):
    g = gen(copied, "cpu")
    pools = torch.randint(0, 250, (n, pages, page, width), generator=g).to(dtype).cuda()
    order = torch.randperm(pages, generator=g).int().cuda()
    src, dst = order[:copied].contiguous(), order[pages - copied:].contiguous()
    want = pools.clone()
    want[:, dst.long()] = pools[:, src.long()]
    as_list = [p.clone() for p in pools]
    assert ops.cache_copy_pages(pools, src, dst) is pools and torch.equal(pools, want)
    ops.cache_copy_pages(as_list, src, dst)
    assert torch.equal(torch.stack(as_list), want)


@gpu
def test_cache_copy_pages_of_one_to_many_and_of_none():
    pools = torch.randn(2, 8, 4, 16, device="cuda", generator=gen(2))
    want = pools.clone()
    want[:, [3, 5]] = pools[:, [1]]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.cache_copy_pages(pools, i32(1, 1, -1, 8, 2, 6, 1 << 30), i32(3, 5, 0, 4, -2, 9, 7))
    assert torch.equal(pools, want)
    assert ops.cache_copy_pages(pools, i32(), i32()) is pools
    with pytest.raises(ValueError):
        ops.cache_copy_pages(pools, i32(1), i32(1, 2))
    with pytest.raises(ValueError):
        ops.cache_copy_pages(pools.transpose(1, 2), i32(1), i32(2))
    with pytest.raises(ValueError):
        ops.cache_copy_pages([pools[0], pools[1, :, :2]], i32(1), i32(2))


# ------------------------------------------------------------------------------------------------------------ distillation
def distill_case(R, V, K, seed, dtype=torch.float32, pad=0, share=0.7, labels=True):
    g = gen(seed)
    logits = (torch.randn(R, V + pad, generator=g, device="cuda") * 2.5).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g, device="cuda")[:K] for _ in range(R)])
    weight = torch.rand(R, generator=g, device="cuda") * (torch.rand(R, generator=g, device="cuda") < share)
    return dict(logits=logits, ids=ids, teacher=torch.randn(R, K, generator=g, device="cuda") * 2, weight=weight,
                target=torch.randint(0, V, (R,), generator=g, device="cuda") if labels else None)


def distill_close(c, V, got=None, **kw):
    loss, d = ops.distill_fwd_bwd(vocab=V, **c, **kw) if got is None else got
    wl, wd = O.distill(vocab=V, **c, **kw)
    tau, hard = kw.get("temperature", 1.0), kw.get("hard", 0.0)
    # sums of V exponentials in fp32, dealt to 128 threads or more, and their tree (2^-24 an addition); an exponential of x is off by |x| 2^-23 of itself and 2^-21
    # (x within 64: what is smaller has no part in fp32 sums); a term of the loss is a difference of logits, each rounded once.
    z = c["logits"][:, :V].float()
    z = z[z.isfinite()]
    big = float(z.abs().max()) if z.numel() else 1.0
    sums = (V / 128 + 16) * 2.0 ** -24 + 64 * 2.0 ** -23 / min(tau, 1.0) + 2.0 ** -21
    some = (2 * sums + 2.0 ** -22 * (2 * big / min(tau, 1.0) + 20)) * ((1 - hard) * tau * tau + hard)
    ok = (loss.double() - wl).abs() <= some + wl.abs() * 2.0 ** -22
    assert bool((ok | (loss == wl) | (loss.isnan() & wl.isnan())).all()), float((loss.double() - wl).abs().max())
    # gradient: rounded to bf16 once; p and t are off by `sums` of themselves (t over K of them), and neither is above 1
    w = c["weight"].double()[:, None]
    p = torch.softmax(c["logits"][:, :V].double() / tau, -1) * (1 - hard) * tau + torch.softmax(c["logits"][:, :V].double(), -1) * hard
    p = torch.nn.functional.pad(p, (0, wd.shape[1] - V)).nan_to_num(1.0)
    tol = 2.0 ** -8 * wd.abs() + w * 3 * sums * (p + (wd.abs() / w.clamp(min=1e-30))) + 2.0 ** -133
    x = d.double()
    assert bool((((x - wd).abs() <= tol) | (x == wd) | (x.isnan() & wd.isnan())).all()), float(((x - wd).abs() - tol).max())
    return loss, d


@gpu
@pytest.mark.parametrize("R, V, K, dtype, pad", [(1, 1, 1, torch.float32, 1), (3, 10, 10, torch.float32, 0), (5, 1000, 8, BF16, 0), (7, 32003, 33, torch.float32, 5),
                                                 (4, 32003, 64, BF16, 5), (2, 128256, 128, torch.float32, 0), (3, 4099, 1024, torch.float32, 3), (130, 257, 5, BF16, 1),
                                                 (2, 300001, 16, torch.float32, 1), (2, 500003, 7, BF16, 0)])
@pytest.mark.parametrize("temperature, hard", [(1.0, 0.0), (2.0, 0.3), (0.5, 1.0), (1.0, 0.5)])
def test_distill(R, V, K, dtype, pad, temperature, hard):
    c = distill_case(R, V, K, R + V, dtype, pad)
    first = distill_close(c, V, temperature=temperature, hard=hard)
    assert all(torch.equal(x, y) for x, y in zip(first, ops.distill_fwd_bwd(vocab=V, **c, temperature=temperature, hard=hard)))
    assert bool((first[1][:, V:] == 0).all())
    off = c["weight"] == 0
    assert bool((first[0][off] == 0).all()) and bool((first[1][off] == 0).all())


@gpu
@pytest.mark.parametrize("R, V, share", [(1300000, 10, 0.9), (1300000, 10, 0.1), (70000, 600, 0.5)])
def test_distill_of_many_rows(R, V, share):
    """more rows than a cluster's list holds, most with a weight and most without: the same few rows over and over"""
    c = distill_case(50, V, 3, R, share=2.0, labels=False)
    c["weight"] = torch.ones(50, device="cuda")
    loss, d = distill_close(c, V)
    at = torch.arange(R, device="cuda") % 50
    on = torch.rand(R, generator=gen(R), device="cuda") < share
    got = ops.distill_fwd_bwd(vocab=V, **{**{k: v[at] if v is not None else None for k, v in c.items()}, "weight": on.float()})
    assert torch.equal(got[0], torch.where(on, loss[at], 0.0))
    assert torch.equal(got[1], torch.where(on[:, None], d[at], 0.0))


@gpu
@pytest.mark.parametrize("V, K", [(50, 6), (40000, 40)])
def test_distill_of_missing_and_repeated_entries(V, K):
    c = distill_case(8, V, K, V, share=2.0)
    c["ids"][0, 2:] = -1                       # a short list
    c["ids"][1, :] = V                         # none
    c["ids"][2, 1] = c["ids"][2, 0]            # the same token twice, three times
    c["ids"][2, 4] = c["ids"][2, 0]
    c["ids"][3, 0] = c["target"][3]            # the label among them
    c["ids"][4, 1:3] = c["target"][4]
    c["teacher"][5, :3] = -float("inf")        # no mass
    c["teacher"][6, :] = -float("inf")
    c["target"][5], c["target"][7] = -100, V   # no label
    for kw in (dict(), dict(hard=0.4, temperature=1.5), dict(hard=1.0)):
        distill_close(c, V, **kw)
    c["ids"] = c["ids"].int()
    c["teacher"] = c["teacher"].to(BF16)
    distill_close(c, V, hard=0.4)
    c["target"] = None
    distill_close(c, V)


@gpu
def test_distill_of_logits_that_are_not_finite():
    V, K = 3001, 5
    c = distill_case(6, V, K, 1, share=2.0, pad=3, labels=False)
    c["logits"][:, V:] = float("nan")          # padding is not read
    c["logits"][0, 100:200] = -float("inf")    # tokens that are ruled out
    c["ids"][0] = torch.arange(5, device="cuda")
    c["logits"][2] *= 1e4
    c["logits"][4, 17] = float("nan")
    c["weight"][5], c["logits"][5] = 0.0, float("nan")
    loss, d = distill_close({k: v[:4] if v is not None else None for k, v in c.items()}, V)
    assert bool((d[0, 100:200] == 0).all())
    loss, d = ops.distill_fwd_bwd(vocab=V, **c)
    assert bool(loss[4].isnan()) and float(loss[5]) == 0 and bool((d[5] == 0).all()) and bool((d[:, V:] == 0).all())
    c["ids"][1, 0] = 150
    c["logits"][1, 150] = -float("inf")        # the teacher wants what the student rules out
    assert float(ops.distill_fwd_bwd(vocab=V, **c)[0][1]) == float("inf")


@gpu
@pytest.mark.parametrize("V, dtype, kw", [(40000, torch.float32, dict()), (40000, BF16, dict(hard=0.4, temperature=1.5)), (3001, torch.float32, dict(hard=1.0)),
                                          (140000, BF16, dict(hard=0.3, temperature=0.5)), (128256, torch.float32, dict(temperature=0.01))])
def test_distill_of_tokens_masked_by_large_values(V, dtype, kw):
    """Whole stretches at a mask's value, down to the type's lowest: as if they were -inf.  A row that is all mask is a row of equal logits."""
    c = distill_case(4, V, 6, V, dtype, share=2.0)
    c["ids"] %= 100
    c["target"] %= 100
    kept = torch.arange(V, device="cuda") < 2000
    want = ops.distill_fwd_bwd(vocab=V, **{**c, "logits": c["logits"].masked_fill(~kept, -float("inf"))}, **kw)
    assert bool(want[0].isfinite().all() and want[1].isfinite().all())
    for mask in (-1e6, -1e10, -1e30, torch.finfo(dtype).min):
        got = ops.distill_fwd_bwd(vocab=V, **{**c, "logits": c["logits"].masked_fill(~kept, mask)}, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), mask
        d = ops.distill_fwd_bwd(vocab=V, **{**c, "logits": torch.full_like(c["logits"], mask)}, **kw)
        equal = ops.distill_fwd_bwd(vocab=V, **{**c, "logits": torch.zeros_like(c["logits"])}, **kw)
        # equal logits z have equal exponents s, which need not be 0: z / tau ln^-1 2 is rounded once, |s| <= 2^-25 of it and <= 64.  2^s cancels out of p but for the roundings
        # of a sum and a quotient, so a gradient is the same before its rounding to bf16 within 2^-20: one step after it.  The loss has -s ln 2 + log(V 2^s): a rounding each of
        # 2^-23 (64 + log V), and 2^s is off by 2^-21.
        assert bool(((d[0] - equal[0]).abs() <= 2.0 ** -15 + 2.0 ** -22 * equal[0].abs()).all()), mask
        assert bool(((d[1].double() - equal[1].double()).abs() <= 2.0 ** -7 * equal[1].double().abs()).all()), mask


@gpu
@pytest.mark.parametrize("temperature, hard", [(1.0, 0.0), (1.7, 0.35)])
def test_distill_gradient_against_differences(temperature, hard):
    """central differences of the 64-bit loss over whole directions (the loss is smooth: their error is of the step's square)"""
    c = distill_case(3, 60, 7, 9, share=2.0)
    kw = dict(vocab=60, temperature=temperature, hard=hard)
    _, d = ops.distill_fwd_bwd(**c, **kw)
    for seed in range(4):
        way = torch.randn(3, 60, generator=gen(seed), device="cuda", dtype=torch.float64)
        step = 1e-4
        at = [(O.distill(**{**c, "logits": c["logits"].double() + s * step * way}, **kw)[0] * c["weight"].double()).sum() for s in (1, -1)]
        want = (at[0] - at[1]) / (2 * step)
        slack = float((d.double() * way).abs().sum()) * 2.0 ** -8 + 1e-6 + 60 * 3 * 2.0 ** -16 * float(way.abs().max())
        assert abs(float((d.double() * way).sum()) - float(want)) <= slack


@gpu
def test_distill_of_views_and_refusals():
    c = distill_case(6, 90, 4, 2)
    want = ops.distill_fwd_bwd(vocab=90, **c, hard=0.2)
    wide = torch.randn(6, 131, device="cuda")
    wide[:, 3:93] = c["logits"]
    ids = torch.zeros(6, 9, dtype=torch.int64, device="cuda")
    ids[:, 2:6] = c["ids"]
    got = ops.distill_fwd_bwd(vocab=90, **{**c, "logits": wide[:, 3:93], "ids": ids[:, 2:6]}, hard=0.2)
    distill_close(c, 90, got=got, hard=0.2)
    assert torch.allclose(got[0], want[0], rtol=1e-6, atol=1e-6)
    for change, err in ((dict(logits=c["logits"].double()), TypeError), (dict(ids=c["ids"].float()), TypeError), (dict(weight=c["weight"][:5]), ValueError),
                        (dict(teacher=c["teacher"][:, :3]), ValueError), (dict(vocab=91), ValueError), (dict(vocab=0), ValueError), (dict(target=c["target"].int()), TypeError),
                        (dict(target=None, hard=0.5), _lib.NativeError), (dict(temperature=0.0), _lib.NativeError), (dict(logits=c["logits"].t().contiguous().t()), ValueError)):
        with pytest.raises(err):
            ops.distill_fwd_bwd(**{**dict(vocab=90), **c, **change})
    empty = ops.distill_fwd_bwd(vocab=90, **{k: v[:0] for k, v in c.items()})
    assert empty[0].shape == (0,) and empty[1].shape == (0, 90)


@gpu
def test_rows_that_share_their_memory():
    """strides of zero are followed where the call takes a stride, and refused where a row's length is the least distance"""
    c = attention_case(3, 5, 4, 2, 64, [40, 7, 22], page=16, seed=30)
    same = dict(q=c["q"][:1].expand(3, -1, -1, -1), lengths=c["lengths"])
    got = ops.tree_attention(same["q"], c["k"], c["v"], c["lengths"], O.tree_words(c["sees"])[:1].expand(3, -1, -1).cuda(), None, c["page_table"])
    close(got, {**c, "q": same["q"], "sees": c["sees"][:1].expand(3, -1, -1)})
    with pytest.raises(ValueError, match="page_table"):
        attend(c, page_table=c["page_table"][:1].expand(3, -1))
    with pytest.raises(ValueError, match="parents"):
        ops.tree_mask(random_parents(1, 5, 1).cuda().expand(3, -1))
    pools, lengths, path, count, table = compact_case(3, 5, 16, 8, BF16, 2, 3, [40, 7, 22])
    for change in (dict(path=path[:1].expand(3, -1)), dict(page_table=table[:1].expand(3, -1))):
        with pytest.raises(ValueError, match="share"):
            ops.cache_compact(pools, **{**dict(lengths=lengths, path=path, count=count, page_table=table), **change})
    d = distill_case(3, 40, 4, 1)
    for name in ("logits", "ids", "teacher"):
        with pytest.raises(ValueError, match=name):
            ops.distill_fwd_bwd(vocab=40, **{**d, name: d[name][:1].expand(3, -1)})


# ------------------------------------------------------------------------------------------------------------ streams, graphs
@gpu
def test_calls_on_other_streams_and_in_graphs():
    """each operator on a side stream, and captured and replayed with new inputs; two graphs that run one after the other share nothing"""
    a = attention_case(2, 20, 8, 2, 128, [500, 40], page=64, seed=20)
    v = verify_case(2, 8, 3000, 5)
    d = distill_case(4, 3000, 9, 6)
    pools, *rest = compact_case(2, 20, 64, 64, BF16, 4, 7, [500, 40])
    want = attend(a), ops.verify_draft(**v), ops.distill_fwd_bwd(vocab=3000, **d)
    words = O.tree_words(a["sees"]).cuda()
    call = lambda: (ops.tree_attention(a["q"], a["k"], a["v"], a["lengths"], words, a["nodes"], a["page_table"]), ops.verify_draft(**v),  # noqa: E731
                    ops.distill_fwd_bwd(vocab=3000, **d))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call()
    s.synchronize()
    flat = lambda r: [r[0], *r[1], *r[2]]  # noqa: E731
    assert all(torch.equal(x, y) for x, y in zip(flat(got), flat(want)))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call())
    a["q"].mul_(-0.5)
    a["lengths"].copy_(torch.tensor([77, 130], dtype=torch.int32))
    v["uniform"].copy_(1 - v["uniform"] * 0.999 - 0.0005)
    d["logits"].mul_(0.5)
    for g in graphs:
        g.replay()
    want = call()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(flat(o), flat(want)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.cache_compact(pools, *rest)
    before = pools.clone()
    g.replay()
    assert torch.equal(pools, torch.stack([O.cache_compact(p, *rest) for p in before]))


@gpu
def test_calls_at_once_on_streams_and_from_threads():
    """the same operators on two streams, launched by two threads, side by side: what each gives alone"""
    import threading
    work = []
    for i in range(2):
        a = attention_case(3, 40 if i else 5, 8, 2, 128, [900, 40, 2000], page=64, seed=40 + i)
        v = verify_case(4, 9, 40000, 41 + i)
        d = distill_case(60, 40000, 20, 42 + i)
        words = O.tree_words(a["sees"]).cuda()
        work.append(lambda a=a, v=v, d=d, words=words: [ops.tree_attention(a["q"], a["k"], a["v"], a["lengths"], words, a["nodes"], a["page_table"]), *ops.verify_draft(**v),
                                                        *ops.distill_fwd_bwd(vocab=40000, **d)])
    want = [w() for w in work]
    torch.cuda.synchronize()
    got, streams = [[], []], [torch.cuda.Stream() for _ in range(2)]

    def run(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i].append(work[i]())
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert len(g) == 20 and all(torch.equal(x, y) for one in g for x, y in zip(one, w))
