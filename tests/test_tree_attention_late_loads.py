"""The tcgen05 kernel of the tree attention when one of its loads lands late, or one of its warps comes late: the same outputs, and no wait that never ends.  Runs the kernel's source on the
CPU (tests/emu/treeattn_tc_emu.cpp), each case in a process of its own, since a wait that never ends ends the process."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest

import test_tree_attention_emulated as T

ROOT = Path(__file__).resolve().parents[1]
# loads that belong to the which-th announcement of bytes (a tile's K, its V, the next tile's K ...) land `ms` later than the others; a warp starts `ms` later
LATE = r"""
inline int g_begun = 0, g_late_load = -1, g_late_warp = -1, g_late_ms = 0;
inline std::vector<std::thread> g_landing;
inline void late_begin(uint64_t* bar, uint32_t bytes) { mbar_arrive_expect_tx(bar, bytes); ++g_begun; }
inline void late_load_4d(void* dst, const Map4* m, uint64_t* bar, int c0, int c1, int c2, int c3) {
  if (g_begun - 1 != g_late_load) return tma_load_4d(dst, m, bar, c0, c1, c2, c3);
  g_landing.emplace_back([=] {
    std::this_thread::sleep_for(std::chrono::milliseconds(g_late_ms));
    tma_load_4d(dst, m, bar, c0, c1, c2, c3);
  });
}
inline void late_warp(int warp) { if (warp == g_late_warp) std::this_thread::sleep_for(std::chrono::milliseconds(g_late_ms)); }
extern "C" void emu_tree_late(int load, int warp, int ms) {
  for (auto& t : g_landing) t.join();
  g_landing.clear();
  g_begun = 0, g_late_load = load, g_late_warp = warp, g_late_ms = ms;
}
"""


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    out = tmp_path_factory.mktemp("emu_tree_late")
    common = (ROOT / "leopard_b200/csrc/lp_common.cuh").read_text()
    a = common.rindex("// ----", 0, common.index("// UMMA descriptors"))
    (out / "emu_helpers.inc").write_text("namespace lp {\n" + common[a:common.rindex("}  // namespace lp")] + "\n}\n")
    shared = (ROOT / "leopard_b200/csrc/lp_treeattn.cuh").read_text()
    (out / "tree_shared.inc").write_text(shared[shared.index("struct TreeArgs {"):shared.index("// the tcgen05 kernel (")]
                                         + shared[shared.index("// a sequence's part of the line"):shared.index("#endif\n\n}  // namespace lp")])
    src = (ROOT / "leopard_b200/csrc/lp_treeattn_tc.cu").read_text()
    body = src[src.index("struct TreeTc {"):src.index("// rows of a TMA box: a cache of one page")].replace("  extern __shared__ uint8_t smem_raw[];\n", "")
    for old, new in (("tma_load_4d(", "late_load_4d("), ("mbar_arrive_expect_tx(full, HEAD_BYTES)", "late_begin(full, HEAD_BYTES)"),
                     ("  if (warp == 0) {\n", "  late_warp(warp);\n  if (warp == 0) {\n")):
        assert body.count(old) == 1, old
        body = body.replace(old, new)
    (out / "tree_tc_kernel.inc").write_text(LATE + body)
    lib = out / "libtree.so"
    r = subprocess.run(["g++", "-std=c++20", "-O2", "-pthread", "-shared", "-fPIC", "-DEMU_DEADLOCK_MS=5000", "-I", str(out), "-I", str(ROOT / "tests/emu"), "-I", str(ROOT / "include"),
                        str(ROOT / "tests/emu/treeattn_tc_emu.cpp"), "-o", str(lib)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return lib


def child(lib, load, warp, split, lengths, nodes):
    """one run, in a process of its own"""
    emu = C.CDLL(lib)
    B, most = len(lengths), max(nodes)
    c = T.case(B, most, 1, 1, 64, lengths, nodes, 0, 3)
    emu.emu_tree_late(load, warp, 400)
    got, want, weight = T.run(emu, c, 1, split)
    emu.emu_tree_late(-1, -1, 0)
    T.check(got, c, want, weight)


def apart(lib, *args):
    code = f"import sys; sys.path[:0] = [{str(ROOT)!r}, {str(ROOT / 'tests')!r}]\nimport test_tree_attention_late_loads as L\nL.child({str(lib)!r}, *{args!r})"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-1500:])


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("load", [0, 1, 2, 3, 4, 5, 8, 9])       # K, V of the first tiles and of one further on
def test_a_load_that_lands_late(library, load, split):
    apart(library, load, -1, split, [1100], [33])


@pytest.mark.parametrize("warp", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("split", [True, False])
def test_a_warp_that_comes_late(library, warp, split):
    """... to pieces of one tile, which the first stream does alone, and to two that both have"""
    apart(library, -1, warp, split, [60, 20, 90, 300, 10, 150], [33, 20, 33, 33, 5, 33])


def test_a_warp_that_comes_late_to_pieces_that_are_not_its_own(library):
    apart(library, -1, 2, True, [60, 20], [33, 20])
