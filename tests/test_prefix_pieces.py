"""How the attention over a shared prefix is cut into pieces: the plan of a call and the line of the prefix's tiles (lp_prefixattn.cu, lp_prefixattn.cuh), compiled for the host.  For whatever number of rows
the requests turn out to bring, every tile of every item is in one CTA's range, every CTA that the join reads of an item has a part of it, and no two pieces have the same place in the workspace."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

from leopard_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]
DRIVER = r"""
#include <algorithm>
#include <cstdio>
#include <vector>
#include "leopard_b200.h"
#define __device__
#define __forceinline__ inline
using std::max; using std::min;
struct float2 { float x, y; };
static int sm_count() { return 148; }
namespace lp {
#include "pieces.inc"
static int wrong(const char* what, long long a, long long b) { std::printf("%s: %lld %lld\n", what, a, b); return 1; }
// facts: whether the tcgen05 kernel takes it, items, CTAs of an item (0: one line for all), cost of the last blocks' tiles, CTAs
extern "C" int check_pieces(const lp_prefix_attn_desc* d, int rows, long long* facts) {
  PrefixArgs a;
  prefix_plan(d, a);
  facts[0] = facts[1] = facts[2] = facts[3] = facts[4] = 0;
  if (!a.pre_ctas || !rows) return 0;
  const bool tc = a.pre_rows > 16;
  const PrefixLine l = pa_line(a, rows);
  facts[0] = tc, facts[1] = l.items, facts[2] = l.own, facts[3] = tc ? l.last_cost : 0, facts[4] = a.pre_ctas;
  const long long tiles = a.pre_tiles;
  std::vector<char> seen((size_t)l.items * tiles, 0), place((size_t)a.pre_slots, 0);
  std::vector<int> parts(l.items, 0), low(l.items, 1 << 30), high(l.items, -1);
  auto piece = [&](int cta, int item, long long t0, long long n) {
    if (n <= 0 || item < 0 || item >= l.items || t0 < 0 || t0 + n > tiles) return wrong("piece", cta, item);
    for (long long t = t0; t < t0 + n; ++t)
      if (seen[item * tiles + t]++) return wrong("tile twice", item, t);
    const long long slot = (long long)item + cta;
    if (slot < 0 || slot >= a.pre_slots || place[slot]++) return wrong("place", item, cta);
    ++parts[item];
    low[item] = std::min(low[item], cta), high[item] = std::max(high[item], cta);
    return 0;
  };
  for (int cta = 0; cta < a.pre_ctas; ++cta) {
    if (tc) {
      long long from, to;
      pa_range(a, l, cta, from, to);
      for (long long u = from; u < to;) {
        const PrefixPiece p = pa_piece(a, u, to);
        if (p.kvh != p.item % a.d.KVH || p.r0 != p.item / a.d.KVH * a.pre_rows || p.r0 >= rows) return wrong("item", p.item, p.r0);
        if (piece(cta, p.item, p.t0, p.n)) return 1;
        u += p.n;
      }
    } else if (l.own && cta < l.items * l.own) {
      const int item = cta / l.own, k = cta - item * l.own;
      if (piece(cta, item, pa_cut(a.pre_tiles, k, l.own), pa_cut(a.pre_tiles, k + 1, l.own) - pa_cut(a.pre_tiles, k, l.own))) return 1;
    }
  }
  for (size_t i = 0; i < seen.size(); ++i)
    if (!seen[i]) return wrong("no CTA has tile", (long long)i / tiles, (long long)i % tiles);
  for (int r = 0; r < rows; r += tc ? 1 : 5)
    for (int kvh = 0; kvh < a.d.KVH; ++kvh) {
      int n, in;
      long long slot;
      pa_pieces_of(a, rows, kvh, r, n, slot, in);
      const int item = r / a.pre_rows * a.d.KVH + kvh;
      if (n != parts[item] || slot != (long long)item + low[item] || high[item] - low[item] + 1 != n || in != r % a.pre_rows) return wrong("pieces of row", r, kvh);
    }
  return 0;
}
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    out = tmp_path_factory.mktemp("pieces")
    shared, host, tc = ((ROOT / "leopard_b200/csrc" / n).read_text() for n in ("lp_prefixattn.cuh", "lp_prefixattn.cu", "lp_prefixattn_tc.cu"))

    def part(text, first, last):
        a = text.index(first)
        return text[a:text.index(last, a)]
    (out / "pieces.inc").write_text(
        part(shared, "constexpr int PA_MAX_BATCH", "// the tcgen05 kernel for many rows") + part(shared, "constexpr int PA_SLACK", "#endif")
        + part(tc, "static int prefix_box", "template <int DH>\nstatic int launch_tc") + part(host, "constexpr long long PA_TC_WORK", "}  // namespace lp"))
    (out / "pieces.cpp").write_text(DRIVER)
    lib = out / "libpieces.so"
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", str(out), "-I", str(ROOT / "include"), str(out / "pieces.cpp"), "-o", str(lib)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    emu = C.CDLL(str(lib))

    def run(B, T, H, G, D, prefix, own, page, rows):
        width = -(-(prefix + own + T) // page) if page else 1
        d = _lib.PrefixAttnDesc(k_page=1 << 20, k_row=G * D, k_head=D, v_page=1 << 20, v_row=G * D, v_head=D, prefix_k=None if page else 16, prefix_v=None if page else 16, pk_row=G * D, pk_head=D, pv_row=G * D,
                                pv_head=D, page_table=16 if page else None, ld_table=width, max_pages=width, n_pages=width * B, page_size=page or own + T, prefix=prefix, B=B, T=T, H=H, KVH=G, D=D, scale=0.1)
        facts = (C.c_longlong * 5)()
        assert emu.check_pieces(C.byref(d), rows, facts) == 0, (B, T, H, G, D, prefix, own, page, rows)
        return tuple(facts)
    return run


def test_every_tile_has_its_cta_and_every_piece_its_place(check):
    r = random.Random(5)
    kinds = set()
    for _ in range(4000):
        G = r.choice([1, 2, 4, 8, 16])
        H, D = G * r.choice([1, 2, 3, 4, 8]), r.choice([64, 96, 128])
        T = r.choice([1, 1, 2, 7, 24, 100])
        B = min(round(2 ** r.uniform(0, 10)), max(1, 6000 // (T * H // G)))
        prefix = round(2 ** r.uniform(0, 15))
        tokens = r.choice([B * T, B * T, r.randint(0, B * T), 1])
        tc, items, own, last, ctas = check(B, T, H, G, D, prefix, r.choice([1, 40, 600]), r.choice([0, 8, 16, 24, 48, 64, 1000, 5]), tokens * (H // G))
        if items:
            kinds.add((tc, own > 0, last, items > ctas))
    # the tcgen05 kernel with CTAs of an item's own and in one line, with last blocks of either cost, with more items than CTAs and fewer; the other one
    assert {(0, True, 0, False), (1, True, 10, False), (1, True, 7, False), (1, False, 10, False), (1, False, 7, False), (1, False, 10, True), (1, False, 7, True)} <= kinds, kinds


@pytest.mark.parametrize("B, T, prefix", [(16, 24, 100003), (64, 1, 32771), (96, 32, 1000), (1000, 1, 500), (4, 1, 4796)])
def test_however_few_rows_the_requests_bring(check, B, T, prefix):
    for tokens in sorted({1, 2, 31, 32, 33, 63, 64, 65, B * T // 3, B * T // 2 + 1, B * T - 1, B * T}):
        if 0 < tokens <= B * T:
            check(B, T, 32, 8, 128, prefix, 24, 64, tokens * 4)
