"""Serving many continuations of one prompt: step tables, rotary positions and cache rows, attention over a shared prefix, token draws — each against its definition in 64 bits
(oracle/serve.py), at the sizes, masks and layouts where it can go wrong; refusals without a GPU."""
import ctypes as C
import math

import pytest
import torch

from leopard_b200 import _lib, ops
from leopard_b200.sampling import Sampler, SamplingParams
from oracle import serve as O

gpu = pytest.mark.gpu
BF16, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=I32, device="cuda")


# ------------------------------------------------------------------------------------------------------------ refusals (no GPU)
@pytest.mark.parametrize("struct, name", [(_lib.RotaryAppendDesc, "lp_rotary_append_desc"), (_lib.PrefixAttnDesc, "lp_prefix_attn_desc")])
def test_struct_layouts_match_the_header(tmp_path, struct, name):
    import re
    import subprocess
    from pathlib import Path
    inc = Path(__file__).resolve().parents[1] / "include"
    lines = [f'printf("%zu\\n", sizeof({name}));'] + [f'printf("%zu\\n", offsetof({name}, {n}));' for n, _ in struct._fields_]
    src = tmp_path / "a.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "leopard_b200.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-I", str(inc), str(src), "-o", str(tmp_path / "a")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(struct)] + [getattr(struct, n).offset for n, _ in struct._fields_]
    assert int(re.search(r"#define LP_PREFIX_MAX_NEW (\d+)", (inc / "leopard_b200.h").read_text())[1]) == _lib.PREFIX_MAX_NEW


def prefix_desc(**kw):
    """a descriptor whose numbers are in order (its addresses are not touched before the checks are through)"""
    base = dict(q=1 << 20, q_batch=4096, q_token=1024, q_head=128, k=1 << 20, k_page=65536, k_row=256, k_head=128, v=1 << 20, v_page=65536, v_row=256, v_head=128, prefix_k=None, pk_row=0,
                pk_head=0, prefix_v=None, pv_row=0, pv_head=0, out=1 << 36, o_batch=4096, o_token=1024, o_head=128, page_table=1 << 20, ld_table=4, max_pages=4, n_pages=9, page_size=64,
                lengths=1 << 20, fresh=None, prefix=100, B=2, T=4, H=8, KVH=2, D=128, scale=0.1)
    return _lib.PrefixAttnDesc(**{**base, **kw})


@pytest.mark.parametrize("change, word", [
    (dict(B=0), "B=0"), (dict(B=2049), "B=2049"), (dict(T=0), "T=0"), (dict(T=257), "T=257"), (dict(H=9), "9 query heads over 2"), (dict(KVH=0), "over 0"), (dict(H=2048, KVH=2048), "1024 at most"),
    (dict(D=72), "heads of 72"), (dict(page_size=0), "of 0 rows"), (dict(n_pages=0), "0 pages"), (dict(max_pages=0), "0 a request"), (dict(max_pages=1 << 20, page_size=1 << 12), "too many"),
    (dict(B=2048, T=256, H=64, KVH=2), "too many"), (dict(prefix=-1), "prefix -1"), (dict(prefix=257), "prefix of 257 rows in 4 pages"), (dict(prefix_k=1 << 20, prefix_v=1 << 20), "of its own"),
    (dict(page_table=None, max_pages=1), "nowhere"), (dict(page_table=None, max_pages=1, prefix_k=1 << 20), "of its own"), (dict(q=None), "null"), (dict(lengths=None), "null"),
    (dict(ld_table=3), "ld_table 3"), (dict(page_table=None, prefix=0), "4 pages"), (dict(page_table=None, prefix=0, max_pages=1, n_pages=1), "1 pages there"),
    (dict(k_row=252), "multiples of 8"), (dict(q=(1 << 20) + 2), "16-byte aligned"), (dict(o_token=120), "share their memory"),
])
def test_prefix_attention_refusals(native_lib, change, word):
    d = prefix_desc(**change)
    rc = native_lib.lp_prefix_attention(C.byref(d), C.c_void_p(1 << 20), 1 << 40, None)
    assert rc == -1 and word in native_lib.lp_last_error().decode(), native_lib.lp_last_error()


def test_prefix_attention_refuses_a_small_workspace(native_lib):
    d = prefix_desc()
    need = native_lib.lp_prefix_attention_workspace_bytes(C.byref(d))
    assert need > 0
    assert native_lib.lp_prefix_attention(C.byref(d), C.c_void_p(1 << 20), need - 1, None) == -1
    assert b"workspace too small" in native_lib.lp_last_error()
    assert native_lib.lp_prefix_attention(C.byref(d), None, need, None) == -1
    assert native_lib.lp_prefix_attention_workspace_bytes(C.byref(prefix_desc(D=80))) == 0


def test_other_refusals_are_status_codes(native_lib):
    p, L = C.c_void_p(1 << 20), native_lib

    def tables(**kw):
        a = {**dict(B=3, W=4, ld=4, size=16, free=p, n=5, used=C.c_void_p(1 << 31), rows=8), **kw}
        return L.lp_step_tables(p, p, C.c_void_p(1 << 34), a["ld"], a["W"], a["size"], a["free"], a["n"], a["used"], a["B"], a["rows"], p, p, p, p, None)
    assert [tables(**kw) for kw in (dict(B=0), dict(B=8193), dict(W=0), dict(size=0), dict(ld=3), dict(rows=-1), dict(n=-1), dict(free=None), dict(used=None), dict(W=1 << 20, ld=1 << 20, size=1 << 12),
                                    dict(rows=(1 << 30) + 1))] == [-1] * 11

    def rotary(**kw):
        a = {**dict(x=p, rows=5, heads=4, D=64, yr=256, yh=64, n=32, freq=p, pos=p), **kw}
        return L.lp_rotary(a["x"], 256, 64, C.c_void_p(1 << 34), a["yr"], a["yh"], 0, a["rows"], a["heads"], a["D"], a["pos"], 0, a["freq"], a["n"], 0, 1.0, 0, None)
    assert [rotary(**kw) for kw in (dict(x=None), dict(pos=None), dict(freq=None), dict(rows=-1), dict(heads=0), dict(D=0), dict(D=4097), dict(n=33), dict(n=-1), dict(yr=200), dict(yh=32))] == [-1] * 11
    assert rotary(rows=0) == 0
    base = dict(q=1 << 20, q_row=512, q_head=64, q_out=1 << 30, o_row=512, o_head=64, k=1 << 20, k_row=128, k_head=64, v=1 << 20, v_row=128, v_head=64, k_pool=1 << 32, kp_page=2048, kp_row=128,
                kp_head=64, v_pool=1 << 34, vp_page=2048, vp_row=128, vp_head=64, positions=1 << 20, inv_freq=1 << 20, slots=1 << 20, positions_64=0, n_freq=32, interleaved=0, fp32=0, rows=5, H=8,
                KVH=2, D=64, n_pages=3, page_size=16, scale=1.0)

    def append(**kw):
        return L.lp_rotary_append(C.byref(_lib.RotaryAppendDesc(**{**base, **kw})), None)
    assert [append(**kw) for kw in (dict(q=None), dict(slots=None), dict(k_pool=None), dict(rows=-1), dict(H=0), dict(KVH=0), dict(D=0), dict(n_freq=33), dict(n_pages=0), dict(page_size=0),
                                    dict(o_row=500), dict(kp_row=120), dict(vp_page=100))] == [-1] * 13
    assert append(rows=0) == 0 and L.lp_rotary_append(None, None) == -1

    def sample(**kw):
        a = {**dict(z=p, ld=100, t=1.0, k=0, pp=1.0, mp=0.0, rows=3, V=100), **kw}
        return L.lp_sample_tokens(a["z"], 1, a["ld"], p, None, a["t"], None, a["k"], None, a["pp"], None, a["mp"], a["rows"], a["V"], p, None)
    assert [sample(**kw) for kw in (dict(z=None), dict(V=0), dict(V=376833, ld=376833), dict(ld=99), dict(t=-0.5), dict(t=math.nan), dict(k=-1), dict(pp=0.0), dict(pp=1.5), dict(pp=math.nan),
                                    dict(mp=-0.1), dict(mp=1.1), dict(rows=-1))] == [-1] * 13
    assert sample(rows=0) == 0


def test_wrappers_refuse_what_is_not_on_a_gpu():
    z = torch.zeros
    with pytest.raises(TypeError, match="lengths"):
        ops.step_tables(z(2, dtype=I32), z(2, dtype=I32), z(2, 3, dtype=I32), z(4, dtype=I32), z(1, dtype=I32), 16, 8)
    with pytest.raises(TypeError, match="x must"):
        ops.rotary(z(2, 3, 8), z(2, dtype=I32), z(4))
    with pytest.raises(ValueError, match="layout"):
        ops.rotary(z(2, 3, 8), z(2, dtype=I32), z(4), layout="pairs")
    with pytest.raises(TypeError, match="q must"):
        ops.rotary_append(z(2, 3, 8), z(2, 1, 8), z(2, 1, 8), z(2, dtype=I32), z(4), z(2, 4, 1, 8), z(2, 4, 1, 8), z(2, dtype=I64))
    with pytest.raises(TypeError, match="q must"):
        ops.prefix_attention(z(1, 1, 8, 128, dtype=BF16), z(3, 64, 2, 128, dtype=BF16), z(3, 64, 2, 128, dtype=BF16), z(1, dtype=I32), 5)
    with pytest.raises(TypeError, match="logits"):
        ops.sample_tokens(z(2, 10), z(2))


def test_parts_of_one_product_are_told_apart(native_lib):
    """what may share memory and what may not, by the entry points' checks: all of these are refused or pass before anything runs (rows of heads of another strides are not known to be apart)"""
    base = dict(q=1 << 20, q_row=96, q_head=8, q_out=1 << 30, o_row=64, o_head=8, k=(1 << 20) + 8 * 8 * 4, k_row=96, k_head=8, v=(1 << 20) + 10 * 8 * 4, v_row=96, v_head=8, k_pool=1 << 32, kp_page=512, kp_row=16,
                kp_head=8, v_pool=(1 << 32) + 256 * 4, vp_page=512, vp_row=16, vp_head=8, positions=1 << 34, inv_freq=1 << 35, slots=1 << 36, positions_64=0, n_freq=4, interleaved=0, fp32=1, rows=5, H=8,
                KVH=2, D=8, n_pages=3, page_size=16, scale=1.0)

    def refused(**kw):
        rc = native_lib.lp_rotary_append(C.byref(_lib.RotaryAppendDesc(**{**base, **kw})), None)
        assert rc != 0      # (without a GPU what passes the checks does not launch)
        return rc == -1 and "share no memory" in native_lib.lp_last_error().decode()
    if torch.cuda.is_available():
        pytest.skip("addresses that nobody holds: for machines without a GPU")
    assert not refused() and not refused(q_out=1 << 20, o_row=96)                                    # apart; the queries in place, beside keys and values of the same rows
    assert refused(q_out=(1 << 20) + 32, o_row=96) and refused(q_out=(1 << 20) + 8 * 4, o_row=96, H=2)
    assert refused(q_out=(1 << 20) + 11 * 8 * 4, o_row=96, H=1) and not refused(q_out=(1 << 20) + 96 * 5 * 4, o_row=96)
    assert refused(v_pool=1 << 32) and refused(v_pool=(1 << 32) + 255 * 4) and refused(v_pool=(1 << 32) + 4 * 512 - 4) and not refused(v_pool=(1 << 32) + 4 * (2 * 512 + 256))
    assert refused(k_pool=1 << 20) and refused(slots=1 << 32) and refused(positions=(1 << 32) + 512 * 4 * 2) and refused(k_pool=(1 << 35) + 12)


# ------------------------------------------------------------------------------------------------------------ step tables
def tables_case(lengths, new, size, width=None, spare=3, seed=0, used=1):
    held = [-(-max(n, 0) // size) for n in lengths]
    need = max(-(-(max(n, 0) + max(t, 0)) // size) for n, t in zip(lengths, new))
    width = width or max(need, 1)
    order = torch.randperm(sum(held) + sum(-(-max(t, 0) // size) + 1 for t in new) + spare, generator=gen(seed, "cpu")).int()
    table, at = torch.full((len(lengths), width), -1, dtype=I32), 0
    for b, n in enumerate(held):
        table[b, :min(n, width)] = order[at:at + n][:width]
        at += n
    return torch.tensor(lengths, dtype=I32), torch.tensor(new, dtype=I32), table, order[at:], torch.tensor([used], dtype=I32)


def check_tables(case, size, rows):
    lengths, new, table, free, used = (x.cuda() for x in case)
    got = ops.step_tables(lengths, new, table, free, used, size, rows)
    want = O.step_tables(*case, size, rows)
    for name, g, w in zip(("row_seq", "row_pos", "slots", "row0", "page_table", "used"), (*got, table, used), (*want[:5], [want[5]])):
        assert g.tolist() == w, name
    assert [g.dtype for g in got] == [I32, I32, I64, I32]
    return table, used


@gpu
@pytest.mark.parametrize("lengths, new, size, rows", [
    ([0], [0], 16, 0), ([0], [1], 16, 1), ([15], [1], 16, 4), ([16], [1], 16, 3), ([7, 0, 64, 31], [1, 1, 0, 1], 16, 5), ([5, 0, 0, 90], [0, 0, 200, 3], 48, 256),
    ([1000] * 64, [1] * 64, 64, 64), ([3, -5, 40], [2, 4, -7], 8, 16), ([10, 20, 30], [50, 60, 70], 16, 100), ([0] * 300, [i % 3 for i in range(300)], 1, 301),
    ([i % 97 for i in range(1500)], [i % 5 for i in range(1500)], 16, 3001), ([12345], [20000], 16, 20000), ([7, 9], [9000, 9001], 64, 18002), ([i * 3 % 500 for i in range(8192)], [1] * 8192, 64, 8192),
    ([i % 40 for i in range(257)], [0] * 256 + [400], 4, 512),
])
def test_step_tables(lengths, new, size, rows):
    check_tables(tables_case(lengths, new, size, seed=len(lengths)), size, rows)


@gpu
def test_step_tables_when_pages_or_room_are_over():
    case = tables_case([5, 30, 0, 60], [40, 40, 100, 8], 16, seed=1)
    for n in (0, 1, 4, 7):                                # the list is over in the middle of a request
        check_tables((*case[:3], case[3][:n].contiguous(), case[4]), 16, 192)
    case = tables_case([5, 30], [40, 40], 16, width=3, seed=2)      # a table that is too narrow
    check_tables(case, 16, 80)
    for used in (-3, 10 ** 6):
        check_tables((*case[:4], torch.tensor([used], dtype=I32)), 16, 80)
    case[2][0, 1:] = torch.tensor([9, -7])                # pages that are there already, in the middle too
    check_tables(case, 16, 80)


@gpu
def test_step_tables_go_on_from_step_to_step():
    case = [x.cuda() for x in tables_case([10, 0, 33], [5, 20, 1], 8, width=12, spare=40, seed=3)]
    seen = set()
    for step in range(6):
        rows = int(case[1].sum())
        _, _, slots, _ = ops.step_tables(*case, 8, rows)
        assert int(slots.min()) >= 0 and not seen & set(slots.tolist())
        seen |= set(slots.tolist())
        case[0] += case[1]
        case[1].copy_(i32([step % 3, 7, 1]))


@gpu
def test_step_tables_wrapper_refusals():
    lengths, new, table, free, used = (x.cuda() for x in tables_case([5, 30], [4, 4], 16, seed=4))
    good = dict(lengths=lengths, new=new, page_table=table, free=free, used=used, page_size=16, rows=8)
    for change, err in ((dict(lengths=lengths.long()), TypeError), (dict(new=new[:1]), ValueError), (dict(page_table=table[:1]), ValueError), (dict(used=free[:2]), ValueError), (dict(free=table), ValueError),
                        (dict(rows=-1), ValueError), (dict(page_size=0), _lib.NativeError), (dict(page_table=table.t().contiguous().t()), ValueError), (dict(lengths=table[:, 0].contiguous().cpu()), TypeError),
                        (dict(free=table.view(-1)), _lib.NativeError), (dict(used=free[:1]), _lib.NativeError)):
        with pytest.raises(err):
            ops.step_tables(**{**good, **change})
    none = ops.step_tables(lengths[:0], new[:0], table[:0], free, used, 16, 3)
    assert none[0].tolist() == none[1].tolist() == none[2].tolist() == [-1] * 3 and none[3].tolist() == [0]


# ------------------------------------------------------------------------------------------------------------ rotary positions
def near(got, want, size):
    """cosine and sine: 2 steps of fp32 and the angle's own rounding to it, pi 2^-24; three more operations: under 2^-20 of |x| + |y|; the rounding to the result's type, half a step"""
    tol = 2.0 ** -20 * size + (2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24) * want.abs() + 1e-37
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (torch.nonzero(bad)[:4].tolist(), float((got.double() - want)[bad].abs().max()))


def freqs(n, base=10000.0):
    return (base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().cuda()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows, heads, D, n", [(1, 1, 2, 1), (1, 32, 128, 64), (7, 3, 96, 16), (64, 8, 64, 32), (2500, 2, 128, 32), (5, 4, 80, 20), (3, 2, 10, 3), (6, 2, 64, 0), (1300, 1, 48, 12), (9, 5, 512, 256)])
def test_rotary(rows, heads, D, n, layout, dtype):
    g = gen(rows + D)
    x = torch.randn(rows, heads, D, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 100000, (rows,), generator=g, device="cuda", dtype=I32)
    f = freqs(n)
    for inverse, scale in ((False, 1.0), (True, 1.37)):
        got = ops.rotary(x, pos, f, layout, scale, inverse)
        near(got, *O.rotary(x, pos, f, layout, scale, inverse))
        assert torch.equal(ops.rotary(x, pos.long(), f, layout, scale, inverse), got)
        into = x.clone()
        assert torch.equal(ops.rotary(into, pos, f, layout, scale, inverse, out=into), got) and torch.equal(into, got)


@gpu
def test_rotary_far_positions_and_scaled_frequencies():
    from leopard_b200.seqlm import RotaryConfig, YarnScaling, rotary_table
    f, scale = rotary_table(RotaryConfig(128, 500000.0, scaling=YarnScaling(16.0, 8192.0, 32.0, 1.0)))
    x = torch.randn(6, 4, 128, generator=gen(1), device="cuda")
    pos = torch.tensor([0, 1, -5, 10 ** 6, 2 ** 31 - 1, 10 ** 9], device="cuda")
    near(ops.rotary(x, pos, f.cuda(), scale=scale), *O.rotary(x, pos, f.cuda(), scale=scale))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotary_of_views(dtype):
    """heads as columns of a wider product, at places where no 16 bytes begin, heads apart, rows in another order; out too"""
    for off, heads, D, n in ((0, 4, 64, 32), (3, 4, 64, 32), (8, 3, 40, 12)):
        x = torch.randn(33, heads * D + 13, generator=gen(off), device="cuda").to(dtype)[:, off:off + heads * D].unflatten(1, (heads, D))
        out = torch.zeros(heads, 33, D + 5, dtype=dtype, device="cuda")
        pos = torch.arange(33, device="cuda", dtype=I32)
        got = ops.rotary(x, pos, freqs(n), out=out[:, :, 1:D + 1].transpose(0, 1))
        near(got, *O.rotary(x, pos, freqs(n)))
        assert not bool(out[:, :, 0].any()) and not bool(out[:, :, D + 1:].any())
        near(ops.rotary(x.flip(0).flip(0)[::2], pos[:17], freqs(n), "interleaved"), *O.rotary(x[::2], pos[:17], freqs(n), "interleaved"))


@gpu
def test_rotary_gradient_is_the_inverse():
    x = torch.randn(40, 6, 64, generator=gen(5), device="cuda")
    pos = torch.randint(0, 5000, (40,), generator=gen(6), device="cuda", dtype=I32)
    f, scale = freqs(24), 1.2
    w = torch.randn(40, 6, 64, generator=gen(7), device="cuda")
    for layout in ("half", "interleaved"):
        # by the formula: the gradient of sum(w y) is the turn back of w
        near(ops.rotary(w, pos, f, layout, scale, inverse=True), *O.rotary(w, pos, f, layout, scale, inverse=True))
        # by differences along a direction d: <w, y(x + d) - y(x - d)> / 2 = <grad, d>; y is linear, so any step does.  Each of 2 x 15,360 products is off by 2^-20 of its size at most.
        d = torch.randn(40, 6, 64, generator=gen(8), device="cuda")
        diff = ops.rotary(x + d, pos, f, layout, scale).double() - ops.rotary(x - d, pos, f, layout, scale).double()
        got = (ops.rotary(w, pos, f, layout, scale, inverse=True).double() * d.double()).sum()
        size = (w.double().abs() * (O.rotary(x + d, pos, f, layout, scale)[1] + O.rotary(x - d, pos, f, layout, scale)[1])).sum() + (d.double().abs() * O.rotary(w, pos, f, layout, scale)[1]).sum()
        # (x + d and x - d are rounded before: half a step each, turned)
        assert abs(float((w.double() * diff).sum() / 2 - got)) <= float(size) * (2.0 ** -20 + 2.0 ** -23)


@gpu
def test_rotary_wrapper_refusals():
    x, pos, f = torch.zeros(4, 2, 16, device="cuda"), torch.zeros(4, dtype=I32, device="cuda"), freqs(8)
    for args, kw, err in (((x.half(), pos, f), {}, TypeError), ((x, pos.float(), f), {}, TypeError), ((x, pos[:3], f), {}, ValueError), ((x, pos, f.double()), {}, TypeError), ((x, pos, freqs(9)), {}, ValueError),
                          ((x, pos, f), dict(out=x[:, :1]), ValueError), ((x, pos, f), dict(out=x.bfloat16()), TypeError), ((x[:, :, ::2], pos, freqs(4)), {}, ValueError),
                          ((x[:3], pos[:3], f), dict(out=x[1:]), _lib.NativeError), ((x, pos, f), dict(out=x[:1].expand(4, 2, 16).clone()[:1].expand(4, 2, 16)), _lib.NativeError)):
        with pytest.raises(err):
            ops.rotary(*args, **kw)
    assert ops.rotary(x[:0], pos[:0], f).shape == (0, 2, 16)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, H, G, D, n, size, layout", [(1, 32, 8, 128, 64, 64, "half"), (64, 8, 1, 128, 64, 16, "half"), (1300, 4, 2, 96, 24, 48, "interleaved"), (5, 3, 3, 20, 7, 3, "half"), (33, 12, 4, 64, 32, 1, "interleaved")])
def test_rotary_append(rows, H, G, D, n, size, layout, dtype):
    g = gen(rows * 3 + D)
    qkv = torch.randn(rows, H + 2 * G, D, generator=g, device="cuda").to(dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    pages = -(-rows // size) + 4
    pools = [torch.randn(pages, size, G, D, generator=g, device="cuda").to(dtype) for _ in range(2)]
    slots = torch.randperm(pages * size, generator=g, device="cuda")[:rows]
    for i, bad in ((0, -1), (rows // 2, pages * size), (rows - 1, -2 ** 40)):
        if rows > 4:
            slots[i] = bad
    pos = torch.randint(0, 30000, (rows,), generator=g, device="cuda", dtype=I32)
    f, scale = freqs(n), 0.8
    want = [p.double() for p in pools]
    turned, size_of = O.rotary(k, pos, f, layout, scale)
    O.append(want[0], turned, slots)
    O.append(want[1], v.double(), slots)
    sizes = O.append(want[0].abs(), size_of, slots)
    before, v_kept = qkv.clone(), v.clone()
    got = ops.rotary_append(q, k, v, pos, f, *pools, slots, layout, scale)
    near(got, *O.rotary(q, pos, f, layout, scale))
    near(pools[0], want[0], sizes)
    assert torch.equal(pools[1].double(), want[1]) and torch.equal(qkv, before)
    # the queries in place, beside keys and values of the same product; pools as halves of one
    both = torch.stack(pools, 1)
    again = ops.rotary_append(q, k, v, pos, f, both[:, 0], both[:, 1], slots, layout, scale, q_out=q)
    assert torch.equal(again, got) and torch.equal(both[:, 0], pools[0]) and torch.equal(both[:, 1], pools[1]) and torch.equal(v, v_kept)


@gpu
def test_rotary_append_wrapper_refusals():
    q, k = torch.zeros(4, 4, 16, device="cuda"), torch.zeros(4, 2, 16, device="cuda")
    pool, pos, slots, f = torch.zeros(3, 8, 2, 16, device="cuda"), torch.zeros(4, dtype=I32, device="cuda"), torch.arange(4, device="cuda"), freqs(8)
    good = dict(q=q, k=k, v=k.clone(), positions=pos, inv_freq=f, k_pool=pool, v_pool=pool.clone(), slots=slots)
    for change, err in ((dict(k=k.bfloat16()), TypeError), (dict(v=k[:, :1]), ValueError), (dict(slots=slots.int()), TypeError), (dict(slots=slots[:3]), ValueError), (dict(v_pool=pool), _lib.NativeError),
                        (dict(k_pool=pool[:, :, :1]), ValueError), (dict(q_out=q[:, :2]), ValueError), (dict(k=pool[0, :4]), _lib.NativeError), (dict(q_out=q[:1].expand(4, 4, 16)), _lib.NativeError),
                        (dict(layout="x"), ValueError), (dict(inv_freq=freqs(9)), ValueError)):
        with pytest.raises(err):
            ops.rotary_append(**{**good, **change})


# ------------------------------------------------------------------------------------------------------------ attention over a shared prefix
def prefix_case(B, T, H, G, D, prefix, own, new=None, page=0, seed=0, spare=2):
    g = gen(seed)
    c = {"q": (torch.randn(B, T, H, D, generator=g, device="cuda") * 1.5).to(BF16), "prefix": prefix, "prefix_k": None, "prefix_v": None, "page_table": None}
    if page:
        first = prefix // page
        need = [-(-(prefix + n + T) // page) - first for n in own]
        order = torch.randperm(first + sum(need) + spare, generator=gen(seed, "cpu")).int()
        table, at = torch.full((B, first + max(need)), -1, dtype=I32), first
        table[:, :first] = order[:first]
        for b, n in enumerate(need):
            table[b, first:first + n] = order[at:at + n]
            at += n
        c["page_table"], shape = table.cuda(), (len(order), page, G, D)
    else:
        shape = (B, max(own) + T + 5, G, D)
        c["prefix_k"], c["prefix_v"] = (torch.randn(prefix, G, D, generator=g, device="cuda").to(BF16) for _ in range(2))
    c["k"], c["v"] = (torch.randn(shape, generator=g, device="cuda").to(BF16) for _ in range(2))
    if page and prefix % page:
        for x in (c["k"], c["v"]):
            last = c["page_table"][:, first].long()
            x[last, :prefix % page] = x[last[:1], :prefix % page].clone()
    c["lengths"] = i32([prefix + n for n in own])
    c["new"] = None if new is None else i32(new)
    return c


def attend(c, **kw):
    return ops.prefix_attention(**{**{k: c[k] for k in ("q", "k", "v", "lengths", "prefix", "new", "page_table", "prefix_k", "prefix_v")}, **kw})


def close(got, c, scale=None):
    """Roundings to bf16 (half a step is 2^-8 of the value): each weight before the second product, relative to the weights' sum of |v|, and the output.  Scores: a sum of D products in fp32 whose additions may be
    cut off (2^-23 of the sum of magnitudes each): delta, and weights move by 2 delta.  Weights and sums of fp32: under 2^-12."""
    want, weight = O.prefix_attention(c["q"], c["k"], c["v"], c["lengths"], c["prefix"], c["new"], c["page_table"], c["prefix_k"], c["prefix_v"], scale)
    D = c["q"].shape[-1]
    s = D ** -0.5 if scale is None else abs(scale)
    top = max(float(x[x.isfinite()].float().abs().max()) for x in (c["k"], c["prefix_k"]) if x is not None and x.numel())
    delta = s * c["q"].float().abs().sum(-1, keepdim=True).double() * top * 2.0 ** -23
    tol = 2.0 ** -8 * (want.abs() + weight) + (2 * delta + 2.0 ** -12) * weight + 1e-30
    for b in range(want.shape[0]):
        t = c["q"].shape[1] if c["new"] is None else max(0, min(c["q"].shape[1], int(c["new"][b])))
        x, y = got[b, :t].double(), want[b, :t]
        same = (x == y) | (x.isnan() & y.isnan())
        bad = ~(same | ((x - y).abs() <= tol[b, :t]))
        assert not bad.any(), (b, torch.nonzero(bad)[:4].tolist(), float((x - y)[bad].abs().max()))


SHAPES = [
    # B, T, H, G, D, prefix, own, new, page
    (1, 1, 32, 8, 128, 0, [0], None, 0), (1, 1, 32, 8, 128, 1, [0], None, 0), (1, 1, 4, 4, 64, 0, [700], None, 16), (4, 1, 32, 8, 128, 4796, [40, 0, 17, 63], None, 64), (2, 1, 8, 8, 128, 130, [0, 5], None, 0),
    (3, 1, 32, 8, 96, 65, [64, 128, 1], [1, 0, 1], 48), (5, 1, 8, 1, 64, 200, [3, 2, 1, 0, 9], None, 16), (9, 1, 32, 8, 128, 1000, list(range(9)), None, 64), (64, 1, 32, 8, 128, 2051, [i * 7 for i in range(64)], None, 64),
    (40, 1, 32, 8, 128, 127, [i % 5 for i in range(40)], [i % 4 > 0 for i in range(40)], 16), (33, 1, 16, 4, 96, 129, [200] * 33, None, 0), (70, 1, 12, 4, 64, 513, list(range(70)), None, 128),
    (2, 24, 32, 8, 128, 300, [10, 0], [24, 5], 64), (3, 5, 8, 2, 64, 64, [0, 1, 70], None, 8), (2, 100, 16, 1, 128, 1030, [3, 0], [100, 99], 0), (6, 17, 8, 2, 96, 77, [0, 64, 63, 1, 5, 300], [17, 0, 3, 16, 1, 8], 48),
    (1, 256, 8, 2, 128, 333, [11], None, 64), (16, 24, 32, 8, 128, 1500, [i for i in range(16)], [(i * 5) % 25 for i in range(16)], 0), (2, 3, 24, 8, 128, 513, [9, 8], None, 1), (8, 1, 4, 2, 64, 40, [3] * 8, None, 5),
    (300, 1, 8, 2, 64, 260, [i % 30 for i in range(300)], None, 16), (12, 7, 32, 1, 64, 700, [i for i in range(12)], None, 64),
]


@gpu
@pytest.mark.parametrize("B, T, H, G, D, prefix, own, new, page", SHAPES)
def test_prefix_attention(B, T, H, G, D, prefix, own, new, page):
    c = prefix_case(B, T, H, G, D, prefix, own, new, page, seed=T * 7 + D + B)
    out = torch.full((B, T, H, D), 7.0, dtype=BF16, device="cuda")
    got = attend(c, out=out)
    close(got, c)
    for b, n in enumerate(new or []):                     # rows that a request does not have stay
        assert bool((got[b, int(n):] == 7.0).all())
    assert torch.equal(attend(c, out=torch.full_like(out, 7.0)), got)


# rows x key heads x keys enough for the tcgen05 kernel: up to 128 rows, a block of 256, a last one of up to 128, more items than CTAs; every head, pages that end inside a tile and whole tiles, few tiles
MANY = [
    (20, 1, 32, 8, 128, 4100, [i for i in range(20)], None, 64), (9, 1, 32, 8, 128, 7001, [3] * 9, [1, 1, 0, 1, 1, 1, 1, 1, 0], 16), (32, 1, 32, 8, 128, 2600, [0] * 32, None, 0),
    (40, 1, 32, 8, 128, 2051, [i % 70 for i in range(40)], [i % 4 > 0 for i in range(40)], 48), (70, 1, 32, 8, 128, 1153, [i for i in range(70)], None, 0), (8, 9, 32, 8, 128, 1280, [5 * i for i in range(8)], [i + 1 for i in range(8)], 128),
    (50, 1, 12, 4, 64, 4099, [i % 9 for i in range(50)], None, 8), (12, 5, 16, 4, 96, 3001, [64] * 12, [i % 6 for i in range(12)], 48), (13, 3, 8, 1, 128, 9000, [7] * 13, None, 64), (200, 2, 16, 16, 64, 640, [2] * 200, None, 16),
    (600, 1, 32, 8, 64, 257, [1] * 600, None, 64), (2, 100, 16, 1, 96, 5000, [3, 0], [100, 99], 0), (17, 1, 16, 16, 128, 10001, list(range(17)), None, 1000), (24, 16, 32, 8, 128, 2000, list(range(24)), [i % 17 for i in range(24)], 24),
]


@gpu
@pytest.mark.parametrize("B, T, H, G, D, prefix, own, new, page", MANY)
def test_prefix_attention_of_many_rows(B, T, H, G, D, prefix, own, new, page):
    test_prefix_attention(B, T, H, G, D, prefix, own, new, page)


@gpu
@pytest.mark.parametrize("B, prefix, page", [(20, 4100, 64), (40, 2051, 48), (70, 1153, 8)])
def test_many_rows_see_no_stale_rows_nor_pages_that_are_not_there(B, prefix, page):
    c = prefix_case(B, 1, 32, 8, 128, prefix, [b % 5 for b in range(B)], page=page, seed=19)
    clean = attend(c)
    held = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for b in range(B):
        for i in range(prefix + b % 5 + 1) if b == 0 else range(prefix // page * page, prefix + b % 5 + 1):
            held[int(c["page_table"][b, i // page]), i % page] = True
    for t in (c["k"], c["v"]):
        t[~held.cuda()] = float("nan")
    # (behind the prefix request 0's page holds its own rows: they are no other's)
    row = (int(c["page_table"][0, prefix // page]), prefix % page)
    c["k"][row], c["v"][row] = float("nan"), float("inf")
    again = attend(c)
    assert torch.equal(again[1:], clean[1:]) and bool(again[0].isnan().any())
    c["k"][row], c["v"][row] = 0.0, 0.0
    for i in (0, 3, prefix // page // 2):
        c["page_table"][:, i] = -1
    c["page_table"][0, 5] = c["k"].shape[0]
    c["page_table"][:, 7:9] = -2 ** 31
    close(attend(c), c)
    c["page_table"][:, :prefix // page] = -1               # nothing of the prefix's whole pages
    close(attend(c), c)
    c["page_table"][:] = -1
    assert bool((attend(c) == 0).all())


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("B, prefix", [(3, 300), (20, 4100), (70, 1153)])
def test_values_of_the_prefix_reach_all(B, prefix, bad):
    c = prefix_case(B, 1, 32, 8, 128, prefix, [b % 5 for b in range(B)], page=64, seed=20)
    clean = attend(c)
    c["v"][int(c["page_table"][0, 1]), 9, 3, 17] = bad
    got = attend(c)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:, :, 12:16, 17] = True                            # (weights that are 0 in fp32 make inf a NaN, as in the definition: 0 x inf)
    assert bool((~got[hit].isfinite()).all()) and torch.equal(got[~hit], clean[~hit])


@gpu
def test_weights_far_below_the_first_ones_do_not_count():
    """scores that grow by hundreds from tile to tile, and fall: maxima that are left behind, in both kernels"""
    for B, prefix in ((2, 700), (20, 4100), (70, 1153)):
        c = prefix_case(B, 1, 32, 8, 128, prefix, [40] * B, page=64, seed=21)
        ramp = torch.linspace(0.05, 6.0, c["k"].shape[0], device="cuda").to(BF16)[:, None, None, None]
        for k in (c["k"] * ramp, c["k"] * ramp.flip(0)):
            d = dict(c, k=k.contiguous())
            close(attend(d), d)


@gpu
@pytest.mark.parametrize("B, T", [(3, 1), (3, 20)])
def test_prefix_attention_is_attention_over_the_whole_sequence(B, T):
    """the same as tree attention of a chain over the same pages, but for roundings: requests that share their pages need no other call"""
    c = prefix_case(B, T, 32, 8, 128, 1000, [5, 64, 33], page=64, seed=3)
    chain = torch.arange(-1, T - 1, dtype=I32, device="cuda").expand(B, T).contiguous()
    tree = ops.tree_attention(c["q"], c["k"], c["v"], c["lengths"], ops.tree_mask(chain)[0], page_table=c["page_table"])
    assert float((attend(c).float() - tree.float()).abs().max()) <= 2 * 2.0 ** -8 * float(tree.float().abs().max() + c["v"].float().abs().max())
    close(tree, c)


@gpu
@pytest.mark.parametrize("scale", [0.02, -0.07, 0.0])
@pytest.mark.parametrize("B, prefix", [(2, 200), (40, 200), (40, 4200)])
def test_prefix_attention_takes_any_scale(B, prefix, scale):
    c = prefix_case(B, 2, 8, 2, 128, prefix, [31] * B, page=64, seed=5)
    close(attend(c, scale=scale), c, scale)


@gpu
@pytest.mark.parametrize("B, prefix", [(2, 150), (30, 150), (30, 4000)])
def test_prefix_attention_of_views(B, prefix):
    """heads as columns of a wider projection, keys and values as halves of one pool's rows, the prefix's too"""
    c = prefix_case(B, 3, 8, 2, 128, prefix, [7 + b for b in range(B)], page=32, seed=6)
    qkv = torch.randn(B * 3, 12 * 128 + 8, device="cuda", generator=gen(1)).to(BF16)
    q = qkv[:, :1024].view(B, 3, 8, 128)
    q.copy_(c["q"])
    pool = torch.randn(c["k"].shape[0], 32, 4, 128, device="cuda", generator=gen(2)).to(BF16)
    pool[:, :, :2], pool[:, :, 2:] = c["k"], c["v"]
    out = torch.zeros(3, B, 8 * 128 + 16, dtype=BF16, device="cuda")
    got = attend(c, q=q, k=pool[:, :, :2], v=pool[:, :, 2:], out=out[:, :, 8:1032].unflatten(2, (8, 128)).transpose(0, 1))
    close(got, c)
    assert torch.equal(got, attend(c)) and bool((out[:, :, :8] == 0).all()) and bool((out[:, :, 1032:] == 0).all())
    c = prefix_case(B, 3, 8, 2, 128, prefix, [7 + b for b in range(B)], seed=7)
    both = torch.stack([c["prefix_k"], c["prefix_v"]], 1)
    assert torch.equal(attend(c, prefix_k=both[:, 0], prefix_v=both[:, 1]), attend(c))
    heads_first = c["k"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(attend(c, k=heads_first), attend(c))


@gpu
@pytest.mark.parametrize("B, T", [(2, 9), (20, 3), (2, 1), (40, 1)])
def test_stale_rows_are_not_seen(B, T):
    """rows behind the requests' last ones, of pages that nobody holds, and behind the prefix in its last page: NaN there has no effect"""
    new = [(b * 3) % (T + 1) for b in range(B)]
    c = prefix_case(B, T, 8, 2, 128, 210, [b * 5 for b in range(B)], new, page=64, seed=9)
    clean = attend(c)
    held = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for b, n in enumerate(new):
        for i in range(210 + b * 5 + n):
            held[int(c["page_table"][b, i // 64]), i % 64] = True
    for t in (c["k"], c["v"]):
        t[~held.cuda()] = float("nan")
    again = attend(c)
    for b, n in enumerate(new):
        assert torch.equal(again[b, :n], clean[b, :n])


@gpu
@pytest.mark.parametrize("past", [0, 15, 16, 50, 64, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [96, 128])
def test_values_of_a_token_reach_the_rows_that_see_it_alone(past, bad, D):
    T, prefix = 9, 37
    c = prefix_case(2, T, 8, 2, D, prefix, [past, past], page=16, seed=10)
    clean = attend(c).clone()
    token = 4
    at = prefix + past + token
    where = (int(c["page_table"][0, at // 16]), at % 16)
    c["v"][(*where, 1, 5)] = bad
    got = attend(c)
    assert torch.equal(got[1], clean[1])
    other = torch.arange(D, device="cuda") != 5
    for i in range(T):
        for h in range(8):
            if i >= token and h >= 4:
                assert bool(got[0, i, h, 5].isnan()) if math.isnan(bad) else float(got[0, i, h, 5]) == bad
                assert torch.equal(got[0, i, h][other], clean[0, i, h][other])
            else:
                assert torch.equal(got[0, i, h], clean[0, i, h])
    # a key that is not finite: its own rows' affair too
    c["v"][(*where, 1, 5)] = 0
    c["k"][(*where, 0, 3)] = float("nan")
    got = attend(c)
    for i in range(T):
        assert bool(got[0, i, :4].isnan().all()) == (i >= token)


@gpu
@pytest.mark.parametrize("B", [2, 40])
def test_pages_that_are_not_there_are_not_seen(B):
    c = prefix_case(B, 2, 8, 2, 64, 200, [60] * B, page=32, seed=11)
    c["page_table"][0, 2] = -1
    c["page_table"][0, 5] = c["k"].shape[0]
    c["page_table"][1, 7] = -9
    close(attend(c), c)
    c["lengths"][1] = 32 * c["page_table"].shape[1] + 5    # longer than its table: what is there is seen
    c["lengths"][0] = 100                                  # shorter than the prefix: as long as it
    close(attend(c), c)
    c["lengths"][0] = -4
    close(attend(c), c)
    c["page_table"][:] = -1
    assert bool((attend(c) == 0).all())


@gpu
def test_new_tokens_out_of_range_count_as_none_or_all():
    c = prefix_case(3, 4, 8, 2, 64, 30, [5, 6, 7], [-3, 4, 9], seed=12)
    got = attend(c, out=torch.full((3, 4, 8, 64), 7.0, dtype=BF16, device="cuda"))
    close(got, c)
    assert bool((got[0] == 7).all())
    c["new"].zero_()
    assert bool((attend(c, out=torch.full((3, 4, 8, 64), 7.0, dtype=BF16, device="cuda")) == 7).all())


@gpu
@pytest.mark.parametrize("B, T, H, G, D", [(2048, 1, 2, 1, 64), (1024, 20, 4, 2, 64), (1025, 5, 1, 1, 96)])
def test_the_largest_batches(B, T, H, G, D):
    c = prefix_case(B, T, H, G, D, 300, [(i * 37) % 20 for i in range(B)], page=16, seed=B)
    close(attend(c), c)


@gpu
@pytest.mark.parametrize("B, prefix", [(2, 130), (40, 8100)])
def test_offsets_beyond_32_bits(B, prefix):
    """a pool of 4.5 GB: its last pages lie past 2^32 bytes and 2^31 elements"""
    pages = 70000
    c = prefix_case(B, 1, 8, 4, 128, prefix, [40] * B, page=64, seed=13)
    n = c["k"].shape[0]
    k, v = (torch.zeros(pages, 64, 4, 128, dtype=BF16, device="cuda") for _ in range(2))
    k[pages - n:], v[pages - n:] = c["k"], c["v"]
    assert torch.equal(attend(c, k=k, v=v, page_table=c["page_table"] + (pages - n)), attend(c))


@gpu
def test_prefix_attention_wrapper_refusals():
    c = prefix_case(2, 4, 8, 2, 128, 20, [3, 4], page=16, seed=14)
    for change, err in ((dict(q=c["q"].float()), TypeError), (dict(k=c["k"][..., :64]), ValueError), (dict(lengths=c["lengths"].long()), TypeError), (dict(lengths=c["lengths"][:1]), ValueError),
                        (dict(page_table=c["page_table"][:1]), ValueError), (dict(new=c["lengths"][:1]), ValueError), (dict(out=c["q"]), _lib.NativeError), (dict(prefix=10 ** 6), _lib.NativeError),
                        (dict(q=c["q"].transpose(2, 3).contiguous().transpose(2, 3)), ValueError), (dict(q=torch.zeros(2, 4, 9, 128, dtype=BF16, device="cuda")), _lib.NativeError),
                        (dict(out=c["q"][:1]), ValueError), (dict(prefix_k=c["k"][0], prefix_v=c["v"][0]), ValueError), (dict(page_table=None), ValueError), (dict(prefix=-1), _lib.NativeError)):
        with pytest.raises(err):
            attend(c, **change)
    d = prefix_case(2, 4, 8, 2, 128, 20, [3, 4], seed=15)
    for change, err in ((dict(prefix=21), ValueError), (dict(k=d["k"][:1], v=d["v"][:1]), ValueError), (dict(prefix_k=None), ValueError)):
        with pytest.raises(err):
            attend(d, **change)
    assert attend(d, prefix=0, prefix_k=None, prefix_v=None).shape == (2, 4, 8, 128)
    assert ops.prefix_attention(c["q"][:0], c["k"], c["v"], c["lengths"][:0], 20, page_table=c["page_table"][:0]).shape == (0, 4, 8, 128)


# ------------------------------------------------------------------------------------------------------------ token draws
def draws(z, u, **kw):
    got = ops.sample_tokens(z, u, **kw)
    assert got.dtype == I64 and got.tolist() == O.sample_tokens(z, u, **kw)
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_k=500, temperature=1.4), dict(top_p=0.9), dict(top_p=0.5, temperature=0.3), dict(top_p=1e-6),
            dict(min_p=0.1), dict(min_p=1.0), dict(top_k=30, top_p=0.8), dict(top_k=700, top_p=0.95, min_p=0.01), dict(top_p=0.999, min_p=0.3), dict(top_k=10 ** 6, top_p=0.9), dict(temperature=50.0, top_p=0.9)]


@gpu
@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sample_tokens(settings, dtype):
    for rows, V, spread in ((1, 1, 1.0), (3, 2, 1.0), (5, 7, 3.0), (4, 1000, 2.5), (6, 2048, 0.01), (3, 4097, 6.0), (2, 32003, 2.5), (40, 300, 1.0)):
        z = (torch.randn(rows, V, generator=gen(V + rows), device="cuda") * spread).to(dtype)
        draws(z, torch.rand(rows, generator=gen(V), device="cuda"), **settings)


@gpu
@pytest.mark.parametrize("settings", [dict(), dict(top_k=50), dict(top_p=0.9), dict(top_k=1000, top_p=0.99), dict(temperature=0.0), dict(min_p=0.02)])
@pytest.mark.parametrize("rows, V", [(1, 128256), (2, 100000), (2, 200000), (1, 376832)])
def test_sample_tokens_of_large_vocabularies(rows, V, settings):
    z = torch.randn(rows, V, generator=gen(V), device="cuda") * 2
    draws(z, torch.rand(rows, generator=gen(V + 1), device="cuda"), **settings)


@gpu
def test_each_row_has_its_settings():
    R = 48
    g = gen(3, "cpu")
    z = torch.randn(R, 5000, generator=gen(3), device="cuda") * 3
    pick = lambda values: torch.tensor(values)[torch.randint(0, len(values), (R,), generator=g)]  # noqa: E731
    kw = dict(temperature=pick([0.0, 0.5, 1.0, 2.0, -1.0, float("nan")]).float().cuda(), top_k=pick([0, 1, 5, 300, -4]).int().cuda(), top_p=pick([0.0, 0.3, 0.9, 1.0, 2.0]).float().cuda(),
              min_p=pick([0.0, 0.05, -1.0, 3.0]).float().cuda())
    draws(z, torch.rand(R, generator=gen(4), device="cuda"), **kw)


@gpu
@pytest.mark.parametrize("V", [600, 5000, 40000])
def test_equal_logits_go_by_their_index(V):
    """long runs of equal logits where the limit falls: words of the whole row, of one value, zeros of both signs"""
    u = torch.linspace(0, 0.999, 7, device="cuda")
    flat = torch.zeros(7, V, device="cuda")
    flat[:, 1::2] = -0.0
    steps = torch.randint(0, 4, (7, V), generator=gen(V), device="cuda").float()
    two = torch.where(torch.arange(V, device="cuda") % 3 == 0, 1.0, 1.0 + 2 ** -20).expand(7, V).contiguous()
    for z in (flat, steps, two):
        for kw in (dict(), dict(top_k=300), dict(top_k=V - 1), dict(top_p=0.5), dict(top_p=0.9999), dict(top_k=V // 2, top_p=0.7), dict(temperature=1e-30, top_p=0.5), dict(temperature=0.0)):
            draws(z, u, **kw)


@gpu
def test_masked_and_odd_logits():
    V = 9000
    z = torch.randn(12, V, generator=gen(1), device="cuda")
    z[0] = -math.inf                                       # nothing
    z[1] = math.nan
    z[2, :] = -math.inf
    z[2, 8999] = -3.0                                      # one word
    z[3, ::2] = torch.finfo(F32).min                       # masks of the type's lowest value
    z[4] = torch.finfo(F32).min
    z[5, [7, 100, 8000]] = math.inf                        # only these
    z[6, 5:] = math.nan
    z[7, 3] = torch.finfo(F32).max
    z[8] *= 1e30
    z[9] *= 1e-40
    z[10, 1:] = -math.inf
    z[11, :4000] = -1e10
    u = torch.rand(12, generator=gen(2), device="cuda")
    for kw in (dict(), dict(top_k=5), dict(top_k=4000), dict(top_p=0.9), dict(temperature=0.0), dict(min_p=0.5), dict(top_k=3000, top_p=0.5), dict(temperature=1e6)):
        draws(z, u, **kw)
    low = z[3:5].bfloat16().nan_to_num(neginf=torch.finfo(BF16).min)
    draws(low, u[:2], top_p=0.9)


@gpu
def test_uniform_at_its_ends():
    z = torch.randn(3, 3000, generator=gen(9), device="cuda")
    below_one = torch.tensor([1 - 2.0 ** -24] * 3, device="cuda")
    for kw in (dict(), dict(top_k=20), dict(top_p=0.7)):
        draws(z, torch.zeros(3, device="cuda"), **kw)
        draws(z, below_one, **kw)
        # what is no number of [0, 1) takes the first or the last kept word
        first, last = ops.sample_tokens(z, torch.zeros(3, device="cuda"), **kw), ops.sample_tokens(z, below_one, **kw)
        assert torch.equal(ops.sample_tokens(z, torch.tensor([-1.0, math.nan, 0.0], device="cuda"), **kw), first)
        assert bool((ops.sample_tokens(z, torch.full((3,), 2.0, device="cuda"), **kw) >= last).all())


@gpu
def test_draws_follow_the_distribution():
    """20,000 evenly spaced numbers: each word's share is its weight's, to within one draw at each of its ends"""
    z = torch.randn(1, 50, generator=gen(4), device="cuda")
    n = 20000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    for kw in (dict(temperature=0.8), dict(top_k=12), dict(top_p=0.8), dict(min_p=0.1)):
        got = torch.bincount(ops.sample_tokens(z.expand(n, 50).contiguous(), u.float(), **kw), minlength=50).double() / n
        w = torch.softmax(z[0].double() / kw.get("temperature", 1.0), -1).cpu()
        order = torch.argsort(w, descending=True)
        keep = torch.zeros(50, dtype=torch.bool)
        ws = w[order]
        keep[order] = (torch.arange(50) < kw.get("top_k", 50)) & (ws.cumsum(0) - ws < kw.get("top_p", 1.0)) & (ws >= kw.get("min_p", 0.0) * ws[0])
        w = torch.where(keep, w, 0.0)
        assert float((got.cpu() - w / w.sum()).abs().max()) <= 2.0 / n + 2.0 ** -22


@gpu
def test_sample_tokens_of_views():
    big = torch.randn(6, 5003, generator=gen(5), device="cuda")
    u = torch.rand(6, generator=gen(6), device="cuda")
    for z in (big[:, :5000], big[:, 3:4003], big[::2, :17], big.bfloat16()[:, 1:3000]):
        draws(z, u[:z.shape[0]], top_p=0.9)


@gpu
def test_sample_tokens_wrapper_refusals():
    z, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    for args, kw, err in (((z.half(), u), {}, TypeError), ((z, u[:2]), {}, ValueError), ((z, u.double()), {}, TypeError), ((z.t(), u), {}, ValueError), ((z, u), dict(top_k=-1), _lib.NativeError),
                          ((z, u), dict(top_p=0.0), _lib.NativeError), ((z, u), dict(top_p=u[:2]), ValueError), ((z, u), dict(top_k=u), TypeError), ((z, u), dict(temperature=-1.0), _lib.NativeError),
                          ((z[:1].expand(3, 10), u), {}, ValueError), ((torch.zeros(1, 400000, device="cuda"), u[:1]), {}, _lib.NativeError)):
        with pytest.raises(err):
            ops.sample_tokens(*args, **kw)
    assert ops.sample_tokens(z[:0], u[:0]).shape == (0,)


@gpu
def test_the_sampler_draws_by_it():
    z = torch.randn(5, 700, generator=gen(7), device="cuda")
    for kw in (dict(top_p=0.8), dict(min_p=0.1), dict(top_k=20, top_p=0.9)):
        p = SamplingParams(temperature=0.9, seed=11, **kw)
        want = ops.sample_tokens(z, torch.rand(5, generator=gen(11), device="cuda"), temperature=0.9, **kw)
        assert torch.equal(Sampler(p)(z), want)
    assert torch.equal(Sampler(SamplingParams(top_p=0.5))(z), z.argmax(-1))                      # greedy as before


# ------------------------------------------------------------------------------------------------------------ streams, graphs, devices
@gpu
def test_two_streams_and_a_captured_step():
    cs = [prefix_case(20, 1, 32, 8, 128, 4100, [30 + i for i in range(20)], page=64, seed=s) for s in (1, 2)]
    zs = [torch.randn(9, 40000, generator=gen(s), device="cuda") * 2 for s in (3, 4)]
    u = torch.rand(9, generator=gen(5), device="cuda")
    alone = [(attend(c), ops.sample_tokens(z, u, top_p=0.9)) for c, z in zip(cs, zs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        got = []
        for s, c, z in zip(streams, cs, zs):
            with torch.cuda.stream(s):
                got.append((attend(c), ops.sample_tokens(z, u, top_p=0.9)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, alone) for a, b in zip(x, y))
    graph = torch.cuda.CUDAGraph()
    c, z = cs[0], zs[0]
    with torch.cuda.graph(graph):
        out, tokens = attend(c), ops.sample_tokens(z, u, top_p=0.9)
    first = zs[0].clone()
    for other, oz, want in ((cs[1], zs[1], alone[1]), (prefix_case(20, 1, 32, 8, 128, 4100, [30 + i for i in range(20)], page=64, seed=1), first, alone[0])):
        for n in ("q", "k", "v", "page_table", "lengths"):
            c[n].copy_(other[n])
        z.copy_(oz)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(tokens, want[1])
