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
