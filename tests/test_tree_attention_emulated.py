"""The tcgen05 kernel of the tree attention on the CPU (tests/emu): the protocol of its warps over several pieces, its tile and page indexing, masks, and the joining of an item's pieces, against
the definition in 64 bits."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from leopard_b200 import _lib
from oracle import draft as O

ROOT = Path(__file__).resolve().parents[1]
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def emu(tmp_path_factory):
    out = tmp_path_factory.mktemp("emu_tree")
    common = (ROOT / "leopard_b200/csrc/lp_common.cuh").read_text()
    a = common.rindex("// ----", 0, common.index("// UMMA descriptors"))
    (out / "emu_helpers.inc").write_text("namespace lp {\n" + common[a:common.rindex("}  // namespace lp")] + "\n}\n")
    shared = (ROOT / "leopard_b200/csrc/lp_treeattn.cuh").read_text()
    (out / "tree_shared.inc").write_text(shared[shared.index("struct TreeArgs {"):shared.index("// the tcgen05 kernel (")]
                                         + shared[shared.index("// a sequence's part of the line"):shared.index("#endif\n\n}  // namespace lp")])
    src = (ROOT / "leopard_b200/csrc/lp_treeattn_tc.cu").read_text()
    body = src[src.index("struct TreeTc {"):src.index("// rows of a TMA box: a cache of one page")].replace("  extern __shared__ uint8_t smem_raw[];\n", "")
    assert "asm" not in body
    (out / "tree_tc_kernel.inc").write_text(body)
    lib = out / "libtree.so"
    r = subprocess.run(["g++", "-std=c++20", "-O2", "-pthread", "-shared", "-fPIC", "-I", str(out), "-I", str(ROOT / "tests/emu"), "-I", str(ROOT / "include"),
                        str(ROOT / "tests/emu/treeattn_tc_emu.cpp"), "-o", str(lib)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return C.CDLL(str(lib))


def cut(total, cta, ctas):
    return total // ctas * cta + min(cta, total % ctas)


def joined(c, out, part, ml, ctas, rows, want):
    """what the join kernel does, from the lengths: the pieces of each item that no CTA has whole"""
    B, T, H, D = c["q"].shape
    G, group = c["k"].shape[2], c["q"].shape[2] // c["k"].shape[2]
    cap = c["k"].shape[1] * (1 if c["page_table"] is None else c["page_table"].shape[1])
    items, first = [], 0
    for b in range(B):
        n = T if c["nodes"] is None else int(c["nodes"][b])
        tiles = -(-min(int(c["lengths"][b]) + n, cap) // 128) if n else 0
        for g in range(G):
            for blk in range(-(-n * group // rows)):
                items.append((b, g, blk, n, first, tiles))
                first += tiles
    cuts = [cut(first, i, ctas) for i in range(ctas + 1)]
    real = [it for it in items if it[5]]
    most = 0                                                     # few items have CTAs of their own: of this many tiles, if that is little above an equal share
    if real and len(real) <= ctas and first > (4 if B == 1 else 1) * ctas:
        if B == 1:
            most = -(-real[0][5] // (ctas // len(real)))
            most = 0 if most > first // ctas + 6 else most
        else:
            most = next((m for m in range(first // ctas + 1, first // ctas + 7, 2) if sum(-(-it[5] // m) for it in real) <= ctas), 0)
    next_cta = 0
    for b, g, blk, n, at, tiles in real:
        mine = [i for i in range(ctas) if cuts[i] < at + tiles and cuts[i + 1] > at]
        starts = [cuts[i] <= at for i in mine]
        if most:
            own = -(-tiles // most)
            mine, starts = list(range(next_cta, next_cta + own)), [i == 0 for i in range(own)]
            next_cta += own
        if len(mine) < 2:
            continue
        for r in range(min(rows, n * group - blk * rows)):
            slots = [2 * i + int(x) for i, x in zip(mine, starts)]
            m, l = ml[slots, r, 0].double(), ml[slots, r, 1].double()
            f = torch.where(m == -torch.inf, 1.0, torch.exp2(m - m.max()))
            s = (l * f).sum()
            row = blk * rows + r
            out[b, row // group, g * group + row % group] = ((part[slots, :, r].reshape(len(slots), D).double() * f[:, None]).sum(0) / s if s != 0 else torch.zeros(D, dtype=torch.float64)).to(BF16)
    return out


def case(B, T, H, G, D, lengths, nodes, page, seed, shared_tree=False):
    g = torch.Generator().manual_seed(seed)
    c = {"q": (torch.randn(B, T, H, D, generator=g) * 1.5).to(BF16)}
    if page:
        need = [-(-(n + T) // page) for n in lengths]
        order = torch.randperm(sum(need) + 2, generator=g).int()
        table, at = torch.full((B, max(need)), -1, dtype=torch.int32), 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        c["page_table"], shape = table, (sum(need) + 2, page, G, D)
    else:
        c["page_table"], shape = None, (B, max(lengths) + T + 3, G, D)
    c["k"], c["v"] = (torch.randn(shape, generator=g).to(BF16) for _ in range(2))
    c["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    c["nodes"] = None if nodes is None else torch.tensor(nodes, dtype=torch.int32)
    parents = torch.full((B, T), -1, dtype=torch.int32)
    for i in range(1, T):
        parents[:, i] = (torch.rand(B, generator=g) * i).int().clamp(max=i - 1)
    c["sees"] = O.tree_sees(parents)
    return c


def run(emu, c, ctas, split):
    B, T, H, D = c["q"].shape
    P, S, G, _ = c["k"].shape
    rows = 128 if T * (H // G) <= 128 else 256
    box = 128 if c["page_table"] is None else next(x for x in (128, 64, 32, 16, 8) if S % x == 0)
    words = O.tree_words(c["sees"])
    out = torch.full((B, T, H, D), 7.0).to(BF16)
    part, ml = torch.full((2 * ctas, D // 4, rows, 4), float("nan")), torch.full((2 * ctas, rows, 2), float("nan"))
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    d = _lib.TreeAttnDesc(ptr(c["q"]), *c["q"].stride()[:3], ptr(c["k"]), *c["k"].stride()[:3], ptr(c["v"]), *c["v"].stride()[:3], ptr(out), *out.stride()[:3],
                          ptr(c["page_table"]), 0 if c["page_table"] is None else c["page_table"].shape[1], 1 if c["page_table"] is None else c["page_table"].shape[1], P, S,
                          ptr(c["lengths"]), ptr(c["nodes"]), ptr(words), words.stride(0), words.stride(1), B, T, H, G, D, D ** -0.5)
    emu.emu_tree_tc(C.byref(d), ctas, rows, box, int(split and rows <= 128), C.c_void_p(part.data_ptr()), C.c_void_p(ml.data_ptr()))
    want, weight = O.tree_attention(c["q"], c["k"], c["v"], c["lengths"], c["sees"], c["nodes"], c["page_table"])
    return joined(c, out, part, ml, ctas, rows, want), want, weight


def check(got, c, want, weight):
    """tolerances: roundings of the weights and of the output to bf16 (2^-8 of each), sums in fp32 (2^-12 is ample)"""
    for b in range(want.shape[0]):
        t = want.shape[1] if c["nodes"] is None else int(c["nodes"][b])
        x, y = got[b, :t].double(), want[b, :t]
        ok = ((x - y).abs() <= 2.0 ** -8 * (y.abs() + weight[b, :t]) + 2.0 ** -12 * weight[b, :t]) | (x == y) | (x.isnan() & y.isnan())
        assert bool(ok.all()), (b, float((x - y).abs().max()))
        assert bool((got[b, t:] == 7.0).all())


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("B, T, H, G, D, lengths, nodes, page, ctas", [
    (1, 40, 4, 4, 128, [100], None, 0, 1),                      # one stream, several items a CTA
    (1, 40, 4, 4, 128, [600], None, 64, 3),                     # items cut between CTAs
    (2, 20, 8, 1, 128, [300, 40], [20, 3], 16, 2),              # both streams in the first sequence, one in the second
    (2, 65, 2, 1, 64, [130, 128], [65, 64], 128, 3),            # two mask words
    (1, 36, 4, 1, 96, [0], None, 32, 1),                        # nodes only, columns beyond a head
    (1, 150, 4, 2, 64, [127], None, 8, 4),                      # two blocks of rows, pages of eight
    (3, 34, 1, 1, 128, [1, 0, 255], [1, 0, 34], 0, 2),          # a sequence without nodes
    (2, 33, 2, 2, 64, [1100, 90], None, 64, 2),                 # many tiles a piece, rings that wrap
    (1, 33, 2, 1, 64, [700], None, 64, 9),                      # few tiles a CTA
    (1, 33, 1, 1, 64, [1400], None, 64, 2),                     # an item with CTAs of its own
    (2, 40, 1, 1, 64, [500, 20], [40, 0], 0, 20),               # ... beside a sequence without nodes
    (3, 40, 1, 1, 64, [0, 260, 20], [0, 40, 33], 0, 17),
])
def test_the_kernel_is_green_under_the_emulator(emu, B, T, H, G, D, lengths, nodes, page, ctas, split):
    c = case(B, T, H, G, D, lengths, nodes, page, T + D)
    got, want, weight = run(emu, c, ctas, split)
    check(got, c, want, weight)


@pytest.mark.parametrize("H, G, split", [(4, 4, True), (4, 4, False), (4, 1, False)])
def test_masks_pages_and_values_that_are_not_finite(emu, H, G, split):
    c = case(1, 40, H, G, 64, [200], None, 32, 5)
    c["sees"][0, 7] = False
    c["page_table"][0, 1] = -1
    c["page_table"][0, 4] = c["k"].shape[0]
    held = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for i in range(240):
        p = int(c["page_table"][0, i // 32])
        if 0 <= p < c["k"].shape[0]:
            held[p, i % 32] = True
    for t in (c["k"], c["v"]):
        t[~held] = float("nan")                                 # rows that nobody holds
    at = 200 + 3
    c["v"][int(c["page_table"][0, at // 32]), at % 32, 0, 5] = float("inf")
    c["v"][int(c["page_table"][0, at // 32]), at % 32, 0, 40] = float("nan")
    got, want, weight = run(emu, c, 2, split)
    check(got, c, want, weight.nan_to_num(0, 0))


@pytest.mark.parametrize("split", [True, False])
def test_a_row_that_sees_nothing_is_zeros(emu, split):
    c = case(1, 40, 4, 4, 64, [0], None, 0, 6)
    c["sees"][0, 5] = False
    got, want, weight = run(emu, c, 1, split)
    check(got, c, want, weight)
    assert bool((got[0, 5] == 0).all())
