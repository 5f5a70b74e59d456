"""Outputs and pools whose places share their memory are refused by the drafting operators; those that lie between one another without sharing any are not."""
import ctypes as C

import pytest
import torch

import test_draft_ops as D
from leopard_b200 import _lib, ops
from oracle import draft as O

P = C.c_void_p(1 << 20)


# ------------------------------------------------------------------------------------------------------------ tree attention's output (no GPU)
@pytest.mark.parametrize("change", [dict(o_head=0), dict(o_node=0), dict(o_batch=0), dict(o_head=120), dict(o_node=512), dict(o_batch=3 * 1024 + 512),
                                    dict(o_node=128, o_head=128), dict(o_batch=-1024), dict(o_head=1 << 62, o_node=1 << 62)])
def test_tree_attention_refuses_rows_of_out_that_share_memory(native_lib, change):
    d = D.tree_desc(**change)
    assert native_lib.lp_tree_attention(C.byref(d), P, 1 << 40, None) == -1
    assert "share" in native_lib.lp_last_error().decode()


@pytest.mark.parametrize("change", [dict(o_node=128, o_head=512), dict(o_batch=128, o_node=256, o_head=1024), dict(o_batch=1 << 40), dict(o_batch=-4096), dict(B=1, o_batch=0),
                                    dict(T=1, o_node=0, o_batch=1024), dict(H=1, KVH=1, o_head=8)])
def test_tree_attention_takes_rows_of_out_in_any_order(native_lib, change):
    d = D.tree_desc(**change)
    assert native_lib.lp_tree_attention(C.byref(d), P, 0, None) == -1                      # (the next check)
    assert b"workspace too small" in native_lib.lp_last_error()


@D.gpu
def test_tree_attention_wrapper_refuses_such_outputs():
    c = D.attention_case(2, 4, 8, 2, 128, [20, 30], page=16, seed=14)
    one = torch.zeros(1, 1, 1, 128, dtype=D.BF16, device="cuda")
    for out in (one.expand(2, 4, 8, 128), torch.zeros(2, 4, 1, 128, dtype=D.BF16, device="cuda").expand(2, 4, 8, 128),
                torch.zeros(2 * 4 * 8 * 128, dtype=D.BF16, device="cuda").as_strided((2, 4, 8, 128), (512, 256, 128, 1))):
        with pytest.raises(_lib.NativeError, match="share"):
            D.attend(c, out=out)
    out = torch.zeros(8, 4, 2, 256, dtype=D.BF16, device="cuda").permute(2, 1, 0, 3)[..., :128]
    assert torch.equal(D.attend(c, out=out), D.attend(c))


# ------------------------------------------------------------------------------------------------------------ pools
def listed(*at):
    return (C.c_void_p * len(at))(*at)


M = 1 << 20


@pytest.mark.parametrize("pools, step, page, row", [
    (listed(M), 0, 0, 64), (listed(M), 0, 448, 64), (listed(M), 0, 96, 256), (listed(M), 0, -448, 64),         # pages within a pool
    (listed(M, M), 0, 512, 64), (listed(M, M + 64), 0, 512, 64), (listed(M, 2 * M, M + 4096 - 64), 0, 512, 64), (listed(M, M + 512 - 64), 0, 1024, 64),      # pools of a list
    (listed(M, M + 64, M + 112), 0, 2048, 256), (listed(M, M + 64), 0, 1856, 256), (listed(M, 2 * M, M + 64, M + 128 - 16), 0, 2048, 256),
    (listed(M), 64, 512, 64), (listed(M), 512, 512, 64), (listed(M), -64, 512, 64), (listed(M), 4096 - 64, 512, 64),      # pools that are a step apart
])
def test_cache_rows_refuse_pools_that_share_memory(native_lib, pools, step, page, row):
    n = len(pools) if not step else 3
    assert native_lib.lp_cache_compact(pools, step, n, page, row, 64, 8, 8, P, 4, 4, P, P, 4, P, 1, 4, None) == -1
    assert "share" in native_lib.lp_last_error().decode()


@pytest.mark.parametrize("pools, step, page", [(listed(M, M), 0, 512), (listed(M, M + 256), 0, 512), (listed(M, M + 4096 - 512 + 256), 0, 512), (listed(M), 512, 512), (listed(M), 256, 1024)])
def test_cache_pages_refuse_pools_that_share_memory(native_lib, pools, step, page):
    n = len(pools) if not step else 3
    assert native_lib.lp_cache_copy_pages(pools, step, n, page, 512, 8, P, P, 1, None) == -1
    assert "share" in native_lib.lp_last_error().decode()


@D.gpu
@pytest.mark.parametrize("order", [(0, 1, 2, 3), (1, 0, 2, 3), (1, 2, 0, 3), (2, 1, 0, 3)])
def test_pools_that_lie_between_one_another(order):
    """[pools, pages, page, width] held in any order of dimensions: one tensor, a list, and a list beside other pools"""
    for seed in range(2):
        pools, *rest = D.compact_case(3, 9, 4, 24, D.BF16, 6, seed, [40, 0, 15])
        want = torch.stack([O.cache_compact(p, *rest) for p in pools])
        there = pools.permute(order).contiguous().permute(torch.tensor(order).argsort().tolist())
        assert torch.equal(ops.cache_compact(there.clone(memory_format=torch.preserve_format), *rest), want)
        held, alone = there.clone(memory_format=torch.preserve_format), there[2].clone(memory_format=torch.preserve_format)
        assert held.stride() == there.stride()
        every = list(held)
        if alone.stride() == every[0].stride():
            every.insert(3, alone)
        ops.cache_compact(every, *rest)
        assert torch.equal(held, want) and (len(every) == 6 or torch.equal(alone, want[2]))
        src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 4], [2, 3]))
        if every[0].stride(1) == 24:                       # pages are contiguous
            again = want.clone()
            again[:, [2, 3]] = want[:, [0, 4]]
            ops.cache_copy_pages(list(held), src, dst)
            assert torch.equal(held, again)


@D.gpu
def test_wrappers_refuse_pools_that_share_memory():
    pools, *rest = D.compact_case(2, 5, 4, 16, D.BF16, 3, 0, [20, 7])
    src, dst = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, 1))
    for bad in ([pools[0], pools[1], pools[0]], [pools[0, :-1], pools[0, 1:]], pools[:, :1].expand(-1, pools.shape[1], -1, -1), pools.flatten().as_strided(pools.shape, (64, 64, 16, 1)),
                pools.flatten().as_strided(pools.shape, (pools.stride(0), 48, 16, 1))):
        with pytest.raises(_lib.NativeError, match="share"):
            ops.cache_compact(bad, *rest)
        with pytest.raises(_lib.NativeError, match="share|apart"):
            ops.cache_copy_pages(bad, src, dst)
