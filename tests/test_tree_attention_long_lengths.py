"""Lengths beyond what a cache or a page table holds: what is there is seen, rows past it are not, nor the nodes that would stand there (tree attention; the tcgen05 kernel on the
CPU, both kernels on a GPU)."""
import ctypes as C

import pytest

import test_draft_ops as D
from test_tree_attention_emulated import case, check, emu, run  # noqa: F401 (emu: a fixture)


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("beyond", [-30, 0, 5, 64, 200, 2 ** 31 - 400])
@pytest.mark.parametrize("rows, page", [(150, 0), (64, 32), (200, 0), (300, 8)])
def test_the_tcgen05_kernel_under_the_emulator(emu, rows, page, beyond, split):  # noqa: F811
    T = 20
    c = case(2, T, 4, 1, 64, [rows - T, 20], [T, 7], page, 3)
    if not page:
        c["k"], c["v"] = c["k"][:, :rows].contiguous(), c["v"][:, :rows].contiguous()
    capacity = c["k"].shape[1] * (1 if c["page_table"] is None else c["page_table"].shape[1])
    c["lengths"][0] = capacity + beyond
    got, want, weight = run(emu, c, 2, split)
    check(got, c, want, weight)


@D.gpu
@pytest.mark.parametrize("beyond", [-30, 0, 5, 64, 200, 2 ** 31 - 10000])
@pytest.mark.parametrize("B, T, H, G, rows, page", [
    (1, 1, 32, 8, 150, 0), (2, 9, 8, 2, 200, 8),        # mma.sync
    (2, 20, 8, 2, 150, 0), (3, 40, 4, 2, 700, 8),       # tcgen05, both streams
    (2, 70, 8, 2, 300, 0), (2, 150, 4, 2, 1000, 8),     # tcgen05, more than 128 rows
    (30, 20, 8, 2, 150, 0),                             # ... and many sequences
])
def test_both_kernels(B, T, H, G, rows, page, beyond):
    c = D.attention_case(B, T, H, G, 128, [max(rows - T, 0)] + [17 + 3 * b for b in range(B - 1)], None, page, seed=rows + T)
    if not page:
        c["k"], c["v"] = c["k"][:, :rows].contiguous(), c["v"][:, :rows].contiguous()
    c["lengths"][0] = c["k"].shape[1] * (1 if c["page_table"] is None else c["page_table"].shape[1]) + beyond
    D.close(D.attend(c), c)
    c["lengths"][:] = c["lengths"][0].item()
    D.close(D.attend(c), c)


def test_tables_end_where_a_tile_does_in_32_bits(native_lib):
    most = (2 ** 31 - 128) // 64
    for pages, word in ((most, b"workspace too small"), (most + 1, b"too many")):
        d = D.tree_desc(max_pages=pages, ld_table=pages)
        assert native_lib.lp_tree_attention(C.byref(d), C.c_void_p(1 << 20), 0, None) == -1 and word in native_lib.lp_last_error()
