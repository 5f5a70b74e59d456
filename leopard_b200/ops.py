"""Thin torch-tensor wrappers over the C ABI (one Python function per exported kernel entry point).

These add shape/dtype checks and output allocation only; no arithmetic happens in Python.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import ACT_NONE, ACT_GELU_TANH, ACT_GELU_ERF, ACT_SWIGLU, NORM_NONE, NORM_RMS, NORM_LAYER  # noqa: F401


def _chk_bf16(t, name):
    if t.dtype != torch.bfloat16 or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA bf16 tensor, got {t.dtype} on {t.device}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")


def gemm(a, w, bias=None, residual=None, act=ACT_NONE, out=None, out_fp32=False, res_row_mod=0, block_n=0):
    """out[M,N'] = act(a[M,K] @ w[N,K].T + bias) + residual   (see lp_gemm_bf16)."""
    _chk_bf16(a, "a")
    _chk_bf16(w, "w")
    M, K = a.shape
    N, K2 = w.shape
    if K != K2:
        raise ValueError(f"K mismatch {K} vs {K2}")
    n_out = N // 2 if act == ACT_SWIGLU else N
    if out is None:
        out = torch.empty((M, n_out), device=a.device, dtype=torch.float32 if out_fp32 else torch.bfloat16)
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != N):
        raise TypeError("bias must be fp32 [N]")
    if residual is not None:
        _chk_bf16(residual, "residual")
    rc = _lib.lib().lp_gemm_bf16(
        _lib.ptr(a), a.stride(0), _lib.ptr(w), w.stride(0), _lib.ptr(out), out.stride(0), M, N, K,
        _lib.ptr(bias), _lib.ptr(residual), residual.stride(0) if residual is not None else 0, res_row_mod,
        act, 1 if out.dtype == torch.float32 else 0, block_n, _lib.stream_ptr())
    _lib.check(rc, "lp_gemm_bf16")
    return out


def gemm_pick_block_n(M, N, act=ACT_NONE):
    return int(_lib.lib().lp_gemm_pick_block_n(M, N, act))


def row_stats(x, out=None):
    """(sum, sum of squares) per row of x bf16 [rows, width] -> fp32 [rows, 1, 2] (lp_row_stats): one partial per row."""
    _chk_bf16(x, "x")
    rows, width = x.shape
    if out is None:
        out = torch.empty((rows, 1, 2), device=x.device, dtype=torch.float32)
    rc = _lib.lib().lp_row_stats(_lib.ptr(x), x.stride(0), rows, width, _lib.ptr(out), _lib.stream_ptr())
    _lib.check(rc, "lp_row_stats")
    return out


def gemm_ex(a, w, bias=None, residual=None, act=ACT_NONE, out=None, out_fp32=False, res_row_mod=0, block_n=0, norm_mode=0,
            stats_in=None, colsum=None, eps=0.0, want_stats=False, rope=None, rope_heads=0, a_t=False, b_t=False):
    """lp_gemm_bf16_ex: lp_gemm_bf16 plus the epilogue fusions — `norm_mode` (NORM_RMS / NORM_LAYER) normalises the rows of
    `a` from `stats_in` fp32 [M, parts, 2] (w must be the gain-folded matrix; LAYER also needs `colsum` and the folded bias),
    `want_stats` returns (out, stats [M, parts, 2]) of the bf16 outputs, `rope` = (cos, sin) fp32 [M, 64] rotates the first
    `rope_heads` 128-column heads.  `a_t` / `b_t`: the operand is given transposed — a as At [K, M], w as Wt [K, N] — and is
    consumed as an MN-major tensor-core operand without a transposed copy (the SFT step's dgrad / wgrad)."""
    _chk_bf16(a, "a")
    _chk_bf16(w, "w")
    K, M = a.shape if a_t else a.shape[::-1]
    N = w.shape[1] if b_t else w.shape[0]
    if (w.shape[0] if b_t else w.shape[1]) != K:
        raise ValueError(f"K mismatch: a {tuple(a.shape)} (a_t={a_t}) vs w {tuple(w.shape)} (b_t={b_t})")
    n_out = N // 2 if act == ACT_SWIGLU else N
    if out is None:
        out = torch.empty((M, n_out), device=a.device, dtype=torch.float32 if out_fp32 else torch.bfloat16)
    d = _lib.GemmDesc()
    d.A, d.lda, d.W, d.ldw, d.C, d.ldc = _lib.ptr(a), a.stride(0), _lib.ptr(w), w.stride(0), _lib.ptr(out), out.stride(0)
    d.M, d.N, d.K = M, N, K
    d.bias = _lib.ptr(bias)
    d.residual, d.ldr, d.res_row_mod = _lib.ptr(residual), (residual.stride(0) if residual is not None else 0), res_row_mod
    d.act, d.out_fp32, d.block_n = act, 1 if out.dtype == torch.float32 else 0, block_n
    d.norm_mode = norm_mode
    if stats_in is not None:
        d.stats_in, d.stats_in_parts = _lib.ptr(stats_in), stats_in.shape[1]
    d.colsum, d.norm_eps = _lib.ptr(colsum), float(eps)
    stats = None
    if want_stats:
        bn = block_n or gemm_pick_block_n(M, N, act)
        d.block_n = bn
        parts = 2 * (-(-N // bn))
        stats = torch.empty((M, parts, 2), device=a.device, dtype=torch.float32)
        d.stats_out, d.stats_out_parts = _lib.ptr(stats), parts
    if rope is not None:
        d.rope_cos, d.rope_sin, d.rope_heads = _lib.ptr(rope[0]), _lib.ptr(rope[1]), rope_heads
    d.a_t, d.b_t = int(bool(a_t)), int(bool(b_t))
    rc = _lib.lib().lp_gemm_bf16_ex(C.byref(d), _lib.stream_ptr())
    _lib.check(rc, "lp_gemm_bf16_ex")
    return (out, stats) if want_stats else out


def attention(qkv, B, T, n_heads, n_kv_heads, head_dim, head_stride, q_off, k_off, v_off, causal, scale=None,
              out=None, variant=0):
    """out[B*T, n_heads*head_dim] = softmax(scale q k^T (+causal)) v on column slices of `qkv` (lp_attention_fwd)."""
    _chk_bf16(qkv, "qkv")
    if qkv.shape[0] != B * T:
        raise ValueError(f"qkv has {qkv.shape[0]} rows, expected B*T = {B * T}")
    if scale is None:
        scale = head_dim ** -0.5
    if out is None:
        out = torch.empty((B * T, n_heads * head_dim), device=qkv.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_attention_fwd(_lib.ptr(qkv), qkv.stride(0), B, T, n_heads, n_kv_heads, head_dim, head_stride,
                                     q_off, k_off, v_off, 1 if causal else 0, float(scale), _lib.ptr(out),
                                     out.stride(0), variant, _lib.stream_ptr())
    _lib.check(rc, "lp_attention_fwd")
    return out


def _chk_f32(t, name):
    if t is not None and (t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous()):
        raise TypeError(f"{name} must be a contiguous CUDA fp32 tensor")


def layernorm(x, gamma, beta, eps, shuffle_side=0, out=None):
    """LayerNorm over the last dim of x [M, D]; shuffle_side=26 stores the pixel-shuffled layout [M/4, 4D]."""
    _chk_bf16(x, "x")
    _chk_f32(gamma, "gamma")
    _chk_f32(beta, "beta")
    M, D = x.shape
    if out is None:
        shape = (M // 4, 4 * D) if shuffle_side else (M, D)
        out = torch.empty(shape, device=x.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_layernorm(_lib.ptr(x), x.stride(0), _lib.ptr(gamma), _lib.ptr(beta), _lib.ptr(out),
                                 out.stride(0), M, D, float(eps), shuffle_side, _lib.stream_ptr())
    _lib.check(rc, "lp_layernorm")
    return out


def rmsnorm(x, gamma, eps, out=None):
    _chk_bf16(x, "x")
    _chk_f32(gamma, "gamma")
    M, D = x.shape
    if out is None:
        out = torch.empty_like(x)
    rc = _lib.lib().lp_rmsnorm(_lib.ptr(x), x.stride(0), _lib.ptr(gamma), _lib.ptr(out), out.stride(0), M, D,
                               float(eps), _lib.stream_ptr())
    _lib.check(rc, "lp_rmsnorm")
    return out


def rope_table(pos, inv_freq):
    """pos int32 [S], inv_freq fp32 [half] -> (cos, sin) fp32 [S, half]."""
    S, half = pos.numel(), inv_freq.numel()
    cs = torch.empty((S, half), device=pos.device, dtype=torch.float32)
    sn = torch.empty_like(cs)
    rc = _lib.lib().lp_rope_table(_lib.ptr(pos), _lib.ptr(inv_freq), _lib.ptr(cs), _lib.ptr(sn), S, half,
                                  _lib.stream_ptr())
    _lib.check(rc, "lp_rope_table")
    return cs, sn


def rope_inplace(x, col0, n_heads, head_dim, cs, sn):
    _chk_bf16(x, "x")
    rc = _lib.lib().lp_rope_inplace(_lib.ptr(x), x.stride(0), x.shape[0], col0, n_heads, head_dim, _lib.ptr(cs),
                                    _lib.ptr(sn), _lib.stream_ptr())
    _lib.check(rc, "lp_rope_inplace")
    return x


def im2col_patch14(pixels, ldo=592):
    """pixels [N,C,H,W] fp32/bf16 -> bf16 [N*(H/14)*(W/14), ldo]."""
    N, Cc, H, W = pixels.shape
    pixels = pixels.contiguous()
    out = torch.empty((N * (H // 14) * (W // 14), ldo), device=pixels.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_im2col_patch14(_lib.ptr(pixels), 1 if pixels.dtype == torch.float32 else 0, _lib.ptr(out), ldo,
                                      N, Cc, H, W, _lib.stream_ptr())
    _lib.check(rc, "lp_im2col_patch14")
    return out


def embed_merge(ids, table, feats, image_id, rows_per_slot):
    """ids int64 [L]; table bf16 [V, D]; feats bf16 [rows, D] or None -> (out [S, D], n_slots, S) (lp_embed_merge)."""
    L = ids.numel()
    D = table.shape[1]
    n_feat = 0 if feats is None else feats.shape[0]
    cap = L + (n_feat // rows_per_slot) * (rows_per_slot - 1)
    out = torch.zeros((cap, D), device=table.device, dtype=torch.bfloat16)
    plan = torch.empty(2 * L + 2, device=table.device, dtype=torch.int32)
    rc = _lib.lib().lp_embed_merge(_lib.ptr(ids), L, image_id, rows_per_slot, _lib.ptr(table), table.stride(0),
                                   table.shape[0], _lib.ptr(feats), feats.stride(0) if feats is not None else 0,
                                   n_feat, _lib.ptr(out), out.stride(0), cap, D, _lib.ptr(plan), _lib.stream_ptr())
    _lib.check(rc, "lp_embed_merge")
    n_slots, S = plan[2 * L:].tolist()
    return out, n_slots, S


def pixel_shuffle(x2d, side):
    """x2d bf16 [B*side*side, D] -> [B*side*side/4, 4*D] (lp_pixel_shuffle)."""
    _chk_bf16(x2d, "x")
    M, D = x2d.shape
    out = torch.empty((M // 4, 4 * D), device=x2d.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_pixel_shuffle(_lib.ptr(x2d), x2d.stride(0), _lib.ptr(out), out.stride(0), M, D, side,
                                     _lib.stream_ptr())
    _lib.check(rc, "lp_pixel_shuffle")
    return out


def attention_cross(q, kv, B, Tq, Tk, n_heads, n_kv_heads, head_dim, k_off, v_off, scale=None, out=None):
    """Cross-attention: q [B*Tq, heads*head_dim], kv [B*Tk, ...] with K at k_off, V at v_off (lp_attention_cross)."""
    _chk_bf16(q, "q")
    _chk_bf16(kv, "kv")
    if scale is None:
        scale = head_dim ** -0.5
    if out is None:
        out = torch.empty((B * Tq, n_heads * head_dim), device=q.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_attention_cross(_lib.ptr(q), q.stride(0), _lib.ptr(kv), kv.stride(0), B, Tq, Tk, n_heads,
                                       n_kv_heads, head_dim, k_off, v_off, float(scale), _lib.ptr(out), out.stride(0),
                                       _lib.stream_ptr())
    _lib.check(rc, "lp_attention_cross")
    return out


def cross_entropy(logits, labels):
    """per-row CE in fp32: logits [R, V] (bf16 or fp32), labels int64 [R] (negative = ignored -> 0) (lp_cross_entropy)."""
    R, V = logits.shape
    out = torch.empty((R,), device=logits.device, dtype=torch.float32)
    labels = labels.to(logits.device, torch.long).contiguous()
    rc = _lib.lib().lp_cross_entropy(_lib.ptr(logits), 1 if logits.dtype == torch.float32 else 0, logits.stride(0),
                                     _lib.ptr(labels), _lib.ptr(out), R, V, _lib.stream_ptr())
    _lib.check(rc, "lp_cross_entropy")
    return out


# ------------------------------------------------------------------------------------------------------------------
# SFT step (lp_train.cu): backward of the glue ops, masked LM loss, optimizer.  Same rule: allocation and checks only.
# ------------------------------------------------------------------------------------------------------------------
def transpose(x, out=None):
    """out[c, r] = x[r, c] for a bf16 matrix view (last dim contiguous, even leading dimension) (lp_transpose_bf16)."""
    _chk_bf16(x, "x")
    rows, cols = x.shape
    if out is None:   # leading dimension padded to 8 elements (the GEMM's TMA maps need 16-byte row strides)
        out = torch.empty((cols, -(-rows // 8) * 8), device=x.device, dtype=torch.bfloat16)[:, :rows]
    rc = _lib.lib().lp_transpose_bf16(_lib.ptr(x), x.stride(0), rows, cols, _lib.ptr(out), out.stride(0), _lib.stream_ptr())
    _lib.check(rc, "lp_transpose_bf16")
    return out


_rms_bwd_ws = {}


def rmsnorm_bwd(x, gamma, dy, eps, dgamma, add=None, out=None):
    """dx = rmsnorm'(x; gamma) dy (+ add); dgamma (fp32 [D]) is overwritten (lp_rmsnorm_bwd)."""
    _chk_bf16(x, "x")
    _chk_bf16(dy, "dy")
    _chk_f32(gamma, "gamma")
    _chk_f32(dgamma, "dgamma")
    M, D = x.shape
    L = _lib.lib()
    ws = _rms_bwd_ws.get((x.device, D))
    if ws is None:
        ws = torch.empty(L.lp_rmsnorm_bwd_workspace_bytes(D), dtype=torch.uint8, device=x.device)
        _rms_bwd_ws[(x.device, D)] = ws
    if out is None:
        out = torch.empty((M, D), device=x.device, dtype=torch.bfloat16)
    rc = L.lp_rmsnorm_bwd(_lib.ptr(x), x.stride(0), _lib.ptr(gamma), _lib.ptr(dy), dy.stride(0), _lib.ptr(add),
                          add.stride(0) if add is not None else 0, _lib.ptr(out), out.stride(0), _lib.ptr(dgamma), M, D,
                          float(eps), _lib.ptr(ws), ws.numel(), _lib.stream_ptr())
    _lib.check(rc, "lp_rmsnorm_bwd")
    return out


_ln_bwd_ws = {}


def layernorm_bwd(x, gamma, dy, eps, dgamma, dbeta, add=None, out=None):
    """dx = layernorm'(x; gamma) dy (+ add); dgamma, dbeta (fp32 [D]) are overwritten (lp_layernorm_bwd)."""
    _chk_bf16(x, "x")
    _chk_bf16(dy, "dy")
    for t, n in ((gamma, "gamma"), (dgamma, "dgamma"), (dbeta, "dbeta")):
        _chk_f32(t, n)
    M, D = x.shape
    L = _lib.lib()
    ws = _ln_bwd_ws.get((x.device, D))
    if ws is None:
        ws = torch.empty(L.lp_layernorm_bwd_workspace_bytes(D), dtype=torch.uint8, device=x.device)
        _ln_bwd_ws[(x.device, D)] = ws
    if out is None:
        out = torch.empty((M, D), device=x.device, dtype=torch.bfloat16)
    rc = L.lp_layernorm_bwd(_lib.ptr(x), x.stride(0), _lib.ptr(gamma), _lib.ptr(dy), dy.stride(0), _lib.ptr(add),
                            add.stride(0) if add is not None else 0, _lib.ptr(out), out.stride(0), _lib.ptr(dgamma),
                            _lib.ptr(dbeta), M, D, float(eps), _lib.ptr(ws), ws.numel(), _lib.stream_ptr())
    _lib.check(rc, "lp_layernorm_bwd")
    return out


def pixel_unshuffle(d, side):
    """d bf16 [M/4, 4*D] (gradient of the shuffled layout) -> [M, D] (lp_pixel_unshuffle)."""
    _chk_bf16(d, "d")
    M4, D4 = d.shape
    out = torch.empty((M4 * 4, D4 // 4), device=d.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_pixel_unshuffle(_lib.ptr(d), d.stride(0), _lib.ptr(out), out.stride(0), M4 * 4, D4 // 4, side,
                                       _lib.stream_ptr())
    _lib.check(rc, "lp_pixel_unshuffle")
    return out


def rowmod_sum(d, T, out):
    """out[t] = sum_n d[n*T + t] (fp32 [T, D], overwritten) (lp_rowmod_sum)."""
    _chk_bf16(d, "d")
    _chk_f32(out, "out")
    rc = _lib.lib().lp_rowmod_sum(_lib.ptr(d), d.stride(0), d.shape[0] // T, T, d.shape[1], _lib.ptr(out), _lib.stream_ptr())
    _lib.check(rc, "lp_rowmod_sum")
    return out


def swiglu_fwd(gu, out=None):
    """gu bf16 [M, 2F] in the fused weight's interleaved column order -> silu(gate) * up [M, F] (lp_swiglu_fwd)."""
    _chk_bf16(gu, "gu")
    M, F2 = gu.shape
    if out is None:
        out = torch.empty((M, F2 // 2), device=gu.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_swiglu_fwd(_lib.ptr(gu), gu.stride(0), _lib.ptr(out), out.stride(0), M, F2 // 2, _lib.stream_ptr())
    _lib.check(rc, "lp_swiglu_fwd")
    return out


def swiglu_bwd(gu, dm, out=None):
    """gradient w.r.t. gu (same interleaved layout) given dm [M, F] (lp_swiglu_bwd)."""
    _chk_bf16(gu, "gu")
    _chk_bf16(dm, "dm")
    M, F2 = gu.shape
    if out is None:
        out = torch.empty((M, F2), device=gu.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_swiglu_bwd(_lib.ptr(gu), gu.stride(0), _lib.ptr(dm), dm.stride(0), _lib.ptr(out), out.stride(0), M,
                                  F2 // 2, _lib.stream_ptr())
    _lib.check(rc, "lp_swiglu_bwd")
    return out


def gelu_bwd(z, dy, act, out=None):
    _chk_bf16(z, "z")
    _chk_bf16(dy, "dy")
    M, N = z.shape
    if out is None:
        out = torch.empty((M, N), device=z.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_gelu_bwd(_lib.ptr(z), z.stride(0), _lib.ptr(dy), dy.stride(0), _lib.ptr(out), out.stride(0), M, N,
                                act, _lib.stream_ptr())
    _lib.check(rc, "lp_gelu_bwd")
    return out


def colsum(dy, out):
    """out[c] = sum_r dy[r, c] (fp32 [N], overwritten) (lp_colsum_bf16)."""
    _chk_bf16(dy, "dy")
    _chk_f32(out, "out")
    M, N = dy.shape
    rc = _lib.lib().lp_colsum_bf16(_lib.ptr(dy), dy.stride(0), M, N, _lib.ptr(out), _lib.stream_ptr())
    _lib.check(rc, "lp_colsum_bf16")
    return out


def ce_fwd_bwd(logits, target, weight, vocab):
    """logits [R, Vp] (fp32 or bf16; columns >= vocab are padding), target int64 [R], weight fp32 [R] ->
    (loss [R] fp32, dlogits bf16 [R, Vp]) (lp_ce_fwd_bwd)."""
    R, Vp = logits.shape
    loss = torch.empty((R,), device=logits.device, dtype=torch.float32)
    d = torch.empty((R, Vp), device=logits.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_ce_fwd_bwd(_lib.ptr(logits), 1 if logits.dtype == torch.float32 else 0, logits.stride(0),
                                  _lib.ptr(target), _lib.ptr(weight), _lib.ptr(loss), _lib.ptr(d), d.stride(0), R, vocab, Vp,
                                  _lib.stream_ptr())
    _lib.check(rc, "lp_ce_fwd_bwd")
    return loss, d


def embed_bwd(d, ids, image_id, dE):
    """dE[id] += d[r] for text rows (lp_embed_bwd); dE fp32 [V, D] must hold the running gradient (zeroed per step)."""
    _chk_bf16(d, "d")
    rc = _lib.lib().lp_embed_bwd(_lib.ptr(d), d.stride(0), _lib.ptr(ids), ids.numel(), image_id, _lib.ptr(dE), dE.stride(0),
                                 d.shape[1], dE.shape[0], _lib.stream_ptr())
    _lib.check(rc, "lp_embed_bwd")


def gather_rows(x, idx):
    """x bf16 [R, D], idx int32 [n] -> [n, D] (lp_gather_rows_bf16)."""
    _chk_bf16(x, "x")
    out = torch.empty((idx.numel(), x.shape[1]), device=x.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_gather_rows_bf16(_lib.ptr(x), x.stride(0), _lib.ptr(idx), idx.numel(), x.shape[1], _lib.ptr(out),
                                        out.stride(0), _lib.stream_ptr())
    _lib.check(rc, "lp_gather_rows_bf16")
    return out


def softmax_bwd(scores, dp, causal, scale, P=None, dS=None):
    """scores, dp fp32 [Sq, Sk] -> (P, dS) bf16 [Sq, Sk] (lp_softmax_bwd)."""
    Sq, Sk = scores.shape
    if P is None:
        P = torch.empty((Sq, Sk), device=scores.device, dtype=torch.bfloat16)
    if dS is None:
        dS = torch.empty((Sq, Sk), device=scores.device, dtype=torch.bfloat16)
    rc = _lib.lib().lp_softmax_bwd(_lib.ptr(scores), scores.stride(0), _lib.ptr(dp), dp.stride(0), _lib.ptr(P), P.stride(0),
                                   _lib.ptr(dS), dS.stride(0), Sq, Sk, 1 if causal else 0, float(scale), _lib.stream_ptr())
    _lib.check(rc, "lp_softmax_bwd")
    return P, dS


def accumulate(dst, src):
    """dst += src for contiguous fp32 tensors of equal size (lp_accumulate_f32)."""
    _chk_f32(dst, "dst")
    _chk_f32(src, "src")
    if dst.numel() != src.numel():
        raise ValueError("size mismatch")
    _lib.check(_lib.lib().lp_accumulate_f32(_lib.ptr(dst), _lib.ptr(src), dst.numel(), _lib.stream_ptr()),
               "lp_accumulate_f32")
    return dst


def grad_norm(flat_grads, max_norm, partial=None, out2=None):
    """Global L2 norm of the fp32 tensors in `flat_grads` -> device tensor [norm, clip coefficient]."""
    L = _lib.lib()
    dev = flat_grads[0].device
    if partial is None:
        partial = torch.empty(L.lp_grad_norm_workspace_bytes() // 4, dtype=torch.float32, device=dev)
    if out2 is None:
        out2 = torch.empty(2, dtype=torch.float32, device=dev)
    partial.zero_()
    for g in flat_grads:
        _chk_f32(g, "grad")
        _lib.check(L.lp_sumsq_accum(_lib.ptr(g), g.numel(), _lib.ptr(partial), _lib.stream_ptr()), "lp_sumsq_accum")
    _lib.check(L.lp_grad_norm_finish(_lib.ptr(partial), float(max_norm), _lib.ptr(out2), _lib.stream_ptr()),
               "lp_grad_norm_finish")
    return out2


def adamw_step(p, g, m, v, p16, step, lr, beta1, beta2, eps, weight_decay, norm_and_clip):
    """In-place FusedAdam (adam_w_mode) update of fp32 p / m / v from fp32 g; refreshes the bf16 copy p16 (or None)."""
    for t, n in ((p, "p"), (g, "g"), (m, "m"), (v, "v")):
        _chk_f32(t, n)
    rc = _lib.lib().lp_adamw_step(_lib.ptr(p), _lib.ptr(g), _lib.ptr(m), _lib.ptr(v), _lib.ptr(p16), p.numel(), float(lr),
                                  float(beta1), float(beta2), float(eps), float(weight_decay), int(step),
                                  _lib.ptr(norm_and_clip), _lib.stream_ptr())
    _lib.check(rc, "lp_adamw_step")


_attn_bwd_ws = {}


def attention_bwd(qkv, out, dout, B, T, n_heads, n_kv_heads, head_dim, q_off, k_off, v_off, causal, scale=None, dqkv=None,
                  head_stride=None):
    """Flash-style backward of `attention` (lp_attention_bwd): returns dqkv in the qkv column layout."""
    _chk_bf16(qkv, "qkv")
    _chk_bf16(out, "out")
    _chk_bf16(dout, "dout")
    if out.stride(0) != dout.stride(0):
        raise ValueError("out and dout must share their leading dimension")
    if scale is None:
        scale = head_dim ** -0.5
    if dqkv is None:
        dqkv = torch.zeros_like(qkv)
    L = _lib.lib()
    need = L.lp_attention_bwd_workspace_bytes(B, T, n_heads)
    ws = _attn_bwd_ws.get(qkv.device)
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, dtype=torch.uint8, device=qkv.device)
        _attn_bwd_ws[qkv.device] = ws
    rc = L.lp_attention_bwd(_lib.ptr(qkv), qkv.stride(0), _lib.ptr(out), _lib.ptr(dout), out.stride(0), B, T, n_heads,
                            n_kv_heads, head_dim, head_stride or head_dim, q_off, k_off, v_off, 1 if causal else 0,
                            float(scale), _lib.ptr(dqkv),
                            dqkv.stride(0), _lib.ptr(ws), ws.numel(), _lib.stream_ptr())
    _lib.check(rc, "lp_attention_bwd")
    return dqkv


# ---- parity mode (csrc/lp_parity.cu; sequencing in leopard_b200/parity.py) ---------------------------------------------------
def _chk_f32_rows(t, name):
    if t.dtype != torch.float32 or not t.is_cuda or t.dim() != 2 or t.stride(1) != 1:
        raise TypeError(f"{name} must be a CUDA fp32 matrix with contiguous rows")


def parity_split(x, out, layout):
    """x fp32 [M, K] (row stride arbitrary: column slices allowed) -> out bf16 [>= M, >= n K] three-term split along K
    (lp_parity_split; layouts in the header)."""
    _chk_f32_rows(x, "x")
    M, K = x.shape
    _lib.check(_lib.lib().lp_parity_split(_lib.ptr(x), x.stride(0), M, K, _lib.ptr(out), out.stride(0), layout, _lib.stream_ptr()),
               "lp_parity_split")
    return out


def parity_norm(x, gamma, beta, eps, rms):
    _chk_f32(x, "x")
    out = torch.empty_like(x)
    _lib.check(_lib.lib().lp_parity_norm(_lib.ptr(x), x.stride(0), _lib.ptr(gamma), _lib.ptr(beta), _lib.ptr(out), out.stride(0),
                                         x.shape[0], x.shape[1], float(eps), 1 if rms else 0, _lib.stream_ptr()), "lp_parity_norm")
    return out


def parity_act(x, kind):
    _chk_f32(x, "x")
    n_out = x.shape[1] // 2 if kind == ACT_SWIGLU else x.shape[1]
    out = torch.empty((x.shape[0], n_out), dtype=torch.float32, device=x.device)
    _lib.check(_lib.lib().lp_parity_act(_lib.ptr(x), x.stride(0), _lib.ptr(out), out.stride(0), x.shape[0], x.shape[1], kind,
                                        _lib.stream_ptr()), "lp_parity_act")
    return out


def parity_add_(y, x, row_mod=0):
    _chk_f32(y, "y")
    _chk_f32(x, "x")
    _lib.check(_lib.lib().lp_parity_add(_lib.ptr(y), y.stride(0), _lib.ptr(x), x.stride(0), y.shape[0], y.shape[1], row_mod,
                                        _lib.stream_ptr()), "lp_parity_add")
    return y


def parity_rope_(x, n_heads, head_dim, cs, sn):
    _chk_f32(x, "x")
    _lib.check(_lib.lib().lp_parity_rope(_lib.ptr(x), x.stride(0), x.shape[0], n_heads, head_dim, _lib.ptr(cs), _lib.ptr(sn),
                                         _lib.stream_ptr()), "lp_parity_rope")
    return x


def parity_softmax_(scores, Tk, scale, causal):
    _chk_f32(scores, "scores")
    _lib.check(_lib.lib().lp_parity_softmax(_lib.ptr(scores), scores.stride(0), scores.shape[0], Tk, float(scale),
                                            1 if causal else 0, _lib.stream_ptr()), "lp_parity_softmax")
    return scores


# ---- drafting (csrc/lp_treeattn.cu, lp_draft.cu, lp_distill.cu): trees of drafted tokens over a cache, their verification, the accepted rows, and the loss
# that trains a draft model.  Calls run on the current stream of the tensors' device.  A step makes these calls once a layer, so what is in order passes one
# condition; only what does not pass is looked at piece by piece, to say what is wrong. ---------------------------------------------------------------------
_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def _need(t, name, dtypes, dim=None, shape=None, device=None, contiguous=False, rows=False):
    """raises unless t is a CUDA tensor of one of these types, of this shape and device, contiguous (in its rows)"""
    kinds = "/".join(str(d).replace("torch.", "") for d in dtypes)
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in dtypes:
        raise TypeError(f"{name} must be a CUDA {kinds} tensor, got " + (f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__))
    if (dim is not None and t.dim() != dim) or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise ValueError(f"{name} must have {f'{dim} dimensions' if shape is None else f'the shape {tuple(shape)}'}, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call on {device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if rows and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    if rows and t.dim() == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: its rows must not share their memory")


def _overlaps(a, b):
    """whether two tensors' spans of memory meet"""
    if a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr():
        return False

    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((s - 1) * abs(st) for s, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _call(device, L, name, fn, *args):
    """fn(*args, stream) on the current stream of `device`"""
    i = device.index
    if torch._C._cuda_getDevice() == i:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        _lib.check_on(L, rc, name)


def tree_mask(parents):
    """parents int32 [B, T] (node 0 the last certain token, parents[b, 0] = -1, a parent lies before its children) -> (mask int64 [B, T, ceil(T / 64)], the
    bits of each node and its ancestors; depth int32 [B, T], its position behind the cached rows) (lp_tree_mask).  T <= 256."""
    _need(parents, "parents", (_I32,), 2, rows=True)
    B, T = parents.shape
    mask = torch.empty((B, T, -(-T // 64)), dtype=_I64, device=parents.device)
    depth = torch.empty((B, T), dtype=_I32, device=parents.device)
    if B and T:
        L = _lib.lib()
        _call(parents.device, L, "lp_tree_mask", L.lp_tree_mask, parents.data_ptr(), max(parents.stride(0), T), B, T, mask.data_ptr(), depth.data_ptr())
    return mask, depth


def _tree_refusals(q, k, v, lengths, mask, nodes, page_table, out):
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        if t is not None:
            _need(t, n, (_BF16,), 4, rows=True)
    B, T, _, D = q.shape
    dev = q.device
    if k.shape[3] != D or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    if out is not None and out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    for t, n in ((k, "k"), (v, "v")) + (((out, "out"),) if out is not None else ()):
        _need(t, n, (_BF16,), device=dev)
    _need(mask, "mask", (_I64,), 3, (B, T, -(-T // 64)), dev, rows=True)
    _need(lengths, "lengths", (_I32,), 1, (B,), dev, contiguous=True)
    if nodes is not None:
        _need(nodes, "nodes", (_I32,), 1, (B,), dev, contiguous=True)
    if page_table is not None:
        _need(page_table, "page_table", (_I32,), 2, (B, page_table.shape[-1]), dev, rows=True)
    elif k.shape[0] < B:
        raise ValueError(f"{B} sequences need a page table or a cache of their own each, k holds {k.shape[0]}")


def tree_attention(q, k, v, lengths, mask, nodes=None, page_table=None, scale=None, out=None):
    """Attention of the step's nodes over a cache that holds their keys and values behind the rows of the past (lp_tree_attention):
    q bf16 [B, T, H, D]; k, v bf16 [pages, page_size, KVH, D] (page_table int32 [B, max_pages]; -1: not there) or [B, rows, KVH, D]; lengths int32 [B], rows
    of the past, seen by every node; mask int64 [B, T, ceil(T / 64)] (tree_mask), the nodes that a node sees: node n is row lengths[b] + n; nodes
    int32 [B] or None, nodes of each sequence.  Strides are free but for a contiguous last dimension and multiples of 8.  -> out bf16 [B, T, H, D]; rows of nodes
    that a sequence does not have stay as they were (`out` given; its rows share no memory, and its span meets none of q, k and v) or are unspecified.  A node that sees nothing is zeros."""
    try:
        B, T, H, D = q.shape
        P, S, KVH, Dk = k.shape
        dev, words = q.device, (T + 63) >> 6
        fine = (q.is_cuda and q.dtype is _BF16 and k.dtype is _BF16 and v.dtype is _BF16 and Dk == D and v.shape == k.shape and k.device == dev and v.device == dev
                and mask.dtype is _I64 and mask.device == dev and mask.shape == (B, T, words) and lengths.dtype is _I32 and lengths.device == dev
                and lengths.shape == (B,) and lengths.is_contiguous())
        qs, ks, vs, ms = q.stride(), k.stride(), v.stride(), mask.stride()
        fine = fine and qs[3] == ks[3] == vs[3] == 1 and (ms[2] == 1 or words == 1)
        if nodes is not None:
            fine = fine and nodes.dtype is _I32 and nodes.device == dev and nodes.shape == (B,) and nodes.is_contiguous()
        if page_table is not None:
            max_pages = page_table.shape[1]
            fine = (fine and page_table.dtype is _I32 and page_table.device == dev and page_table.shape == (B, max_pages)
                    and (page_table.stride(1) == 1 or max_pages <= 1) and (page_table.stride(0) >= max_pages or B == 1))
            table, ld = page_table.data_ptr(), max(page_table.stride(0), max_pages)
        else:
            fine, max_pages, table, ld = fine and P >= B, 1, None, 0
        if out is not None:
            fine = fine and out.dtype is _BF16 and out.device == dev and out.shape == q.shape and out.stride(3) == 1
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _tree_refusals(q, k, v, lengths, mask, nodes, page_table, out)
        raise ValueError("tree_attention: heads must be contiguous")
    if out is None:
        out = torch.empty((B, T, H, D), dtype=_BF16, device=dev)
    elif _overlaps(out, q) or _overlaps(out, k) or _overlaps(out, v):
        raise ValueError("out must not share memory with q, k or v")
    if B == 0 or T == 0:
        return out
    os_ = out.stride()
    d = _lib.TreeAttnDesc(q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], out.data_ptr(), os_[0], os_[1], os_[2],
                          table, ld, max_pages, P, S, lengths.data_ptr(), None if nodes is None else nodes.data_ptr(), mask.data_ptr(), ms[0], ms[1], B, T, H, KVH, D,
                          D ** -0.5 if scale is None else float(scale))
    L, ref = _lib.lib(), C.byref(d)
    need = L.lp_tree_attention_workspace_bytes(ref)
    if need == 0:
        _lib.check(-1, "lp_tree_attention")
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(dev, L, "lp_tree_attention", L.lp_tree_attention, ref, ws.data_ptr(), need)
    return out


def _verify_refusals(target, tokens, parents, uniform, draft, nodes):
    _need(target, "target", (_F32,), 3, rows=True)
    B, T, _ = target.shape
    for t, n, kind in ((tokens, "tokens", _I64), (parents, "parents", _I32), (uniform, "uniform", _F32)):
        _need(t, n, (kind,), 2, (B, T), target.device, contiguous=True)
    if draft is not None:
        _need(draft, "draft", (_F32,), 3, target.shape, target.device, rows=True)
    if nodes is not None:
        _need(nodes, "nodes", (_I32,), 1, (B,), target.device, contiguous=True)


def verify_draft(target, tokens, parents, uniform, draft=None, nodes=None):
    """Which drafted nodes the target accepts, and the token after them (lp_verify_draft): target fp32 [B, T, V], row i the target's probabilities after node i;
    draft of the same shape, what the children of node i were drawn from, each independently of the others and with replacement, which is what keeps the target's distribution
    (children drawn without replacement do not); None: drafts that were not drawn, such as the best of a list; tokens
    int64, parents int32, uniform fp32 (numbers in [0, 1): [b, c] tries node c, [b, 0] takes the next token) [B, T]; nodes int32 [B] or None.
    -> (path int32 [B, T]: the accepted nodes from node 0 on, then -1; count int32 [B]; next token int64 [B])."""
    try:
        B, T, V = target.shape
        dev, shape, ts = target.device, (B, T), target.stride()
        fine = (target.is_cuda and target.dtype is _F32 and ts[2] == 1 and tokens.dtype is _I64 and parents.dtype is _I32 and uniform.dtype is _F32
                and tokens.shape == shape and parents.shape == shape and uniform.shape == shape and tokens.device == dev and parents.device == dev
                and uniform.device == dev and tokens.is_contiguous() and parents.is_contiguous() and uniform.is_contiguous())
        ds = (0, 0, 1) if draft is None else draft.stride()
        fine = fine and (draft is None or (draft.dtype is _F32 and draft.shape == target.shape and draft.device == dev and ds[2] == 1))
        fine = fine and (nodes is None or (nodes.dtype is _I32 and nodes.shape == (B,) and nodes.device == dev and nodes.is_contiguous()))
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _verify_refusals(target, tokens, parents, uniform, draft, nodes)
        if target.shape[2] != 1:
            raise ValueError("verify_draft: rows must be contiguous")
        ts, ds = target.stride(), (0, 0, 1) if draft is None else draft.stride()
    path = torch.empty((B, T), dtype=_I32, device=dev)
    count = torch.empty((B,), dtype=_I32, device=dev)
    token = torch.empty((B,), dtype=_I64, device=dev)
    if B:
        L = _lib.lib()
        _call(dev, L, "lp_verify_draft", L.lp_verify_draft, target.data_ptr(), ts[0], ts[1], None if draft is None else draft.data_ptr(), ds[0], ds[1], tokens.data_ptr(),
              parents.data_ptr(), uniform.data_ptr(), None if nodes is None else nodes.data_ptr(), B, T, V, path.data_ptr(), count.data_ptr(), token.data_ptr())
    return path, count, token


def _pools(pools):
    """one tensor [n, pages, page_size, width] or a list of [pages, page_size, width] alike -> (their pointers or the first one's, bytes between them, their number,
    shape, strides, bytes of an element, device)"""
    if isinstance(pools, torch.Tensor):
        if not pools.is_cuda or pools.dim() != 4:
            _need(pools, "pools", (pools.dtype,), 4)
        n, st, e = pools.shape[0], pools.stride(), pools.element_size()
        if n > 1 and st[0] == 0:
            raise ValueError("pools must not share their memory")
        return (C.c_void_p * 1)(pools.data_ptr()), st[0] * e if n > 1 else 0, n, pools.shape[1:], st[1:], e, pools.device
    pools = list(pools)
    if not pools:
        return None, 0, 0, (0, 0, 0), (0, 0, 0), 0, None
    first = pools[0]
    _need(first, "pools[0]", (first.dtype if isinstance(first, torch.Tensor) else _BF16,), 3)
    for i, t in enumerate(pools):
        if not isinstance(t, torch.Tensor) or t.shape != first.shape or t.stride() != first.stride() or t.device != first.device or t.dtype != first.dtype:
            raise ValueError(f"pools[{i}] is not like pools[0], {tuple(first.shape)} {first.dtype} on {first.device}: shapes, strides and types have to be the same")
    return (C.c_void_p * len(pools))(*[t.data_ptr() for t in pools]), 0, len(pools), first.shape, first.stride(), first.element_size(), first.device


def cache_compact(pools, lengths, path, count, page_table=None):
    """The accepted nodes' rows become the last rows of their sequences, in every pool, in place (lp_cache_compact): row lengths[b] + path[b, j] moves to row
    lengths[b] + j, j < count[b] (path and count as verify_draft gives them; path rises).  pools: one tensor [n, pages, page_size, width] or a list of [pages, page_size,
    width] of equal shapes, any type (the decoder's cache [layers, 2, rows, width]: kv.flatten(0, 1).unsqueeze(1)); page_table int32 [B, max_pages], or None: sequence b
    is page b.  lengths, count int32 [B], path int32 [B, T].  Rows that are not there move nothing.  Pools, pages and rows share no memory, and a page whose rows move stands
    in no other sequence's table (copy what several hold first: cache_copy_pages).  Returns pools."""
    ptrs, step, n, shape, st, e, dev = _pools(pools)
    if not n or not path.numel():
        return pools
    P, S, W = shape
    try:
        B, T = path.shape
        fine = (path.dtype is _I32 and path.device == dev and (path.stride(1) == 1 or T == 1) and (path.stride(0) >= T or B == 1) and lengths.dtype is _I32 and lengths.device == dev and lengths.shape == (B,)
                and lengths.is_contiguous() and count.dtype is _I32 and count.device == dev and count.shape == (B,) and count.is_contiguous() and (st[2] == 1 or W == 1))
        if page_table is not None:
            max_pages = page_table.shape[1]
            fine = (fine and page_table.dtype is _I32 and page_table.device == dev and page_table.shape == (B, max_pages)
                    and (page_table.stride(1) == 1 or max_pages <= 1) and (page_table.stride(0) >= max_pages or B == 1))
            table, ld = page_table.data_ptr(), max(page_table.stride(0), max_pages)
        else:
            max_pages, table, ld = 1, None, 0
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _need(path, "path", (_I32,), 2, device=dev, rows=True)
        _need(lengths, "lengths", (_I32,), 1, (path.shape[0],), dev, contiguous=True)
        _need(count, "count", (_I32,), 1, (path.shape[0],), dev, contiguous=True)
        if page_table is not None:
            _need(page_table, "page_table", (_I32,), 2, (path.shape[0], page_table.shape[-1]), dev, rows=True)
        raise ValueError("rows must be contiguous")
    L = _lib.stream32_lib()
    _call(dev, L, "lp_cache_compact", L.lp_cache_compact, ptrs, step, n, st[0] * e, (st[1] if S > 1 else W) * e, W * e, P, S, table, ld, max_pages, lengths.data_ptr(),
          path.data_ptr(), max(path.stride(0), T), count.data_ptr(), B, T)
    return pools


def cache_copy_pages(pools, src, dst):
    """Page src[i] of every pool is copied to page dst[i] (lp_cache_copy_pages): src, dst int32 [n] on the device; no page may be in both, nor twice in dst; entries
    that are not pages copy nothing.  pools as in cache_compact, contiguous within a page.  Returns pools."""
    ptrs, step, n, shape, st, e, dev = _pools(pools)
    _need(src, "src", (_I32,), 1)
    if not n or not src.numel():
        return pools
    _need(src, "src", (_I32,), device=dev, contiguous=True)
    _need(dst, "dst", (_I32,), 1, src.shape, dev, contiguous=True)
    P, S, W = shape
    if (W > 1 and st[2] != 1) or (S > 1 and st[1] != W):
        raise ValueError("pages must be contiguous")
    L = _lib.stream32_lib()
    _call(dev, L, "lp_cache_copy_pages", L.lp_cache_copy_pages, ptrs, step, n, (st[0] if P > 1 else S * W) * e, S * W * e, P, src.data_ptr(), dst.data_ptr(), src.numel())
    return pools


def _distill_refusals(logits, ids, teacher, weight, vocab, target):
    _need(logits, "logits", (_F32, _BF16), 2, rows=True)
    R, Vp = logits.shape
    dev = logits.device
    _need(ids, "ids", (_I64, _I32), 2, device=dev, rows=True)
    _need(teacher, "teacher", (_F32, _BF16), 2, ids.shape, dev, rows=True)
    _need(weight, "weight", (_F32,), 1, (R,), dev, rows=True)
    if ids.shape[0] != R:
        raise ValueError(f"logits {tuple(logits.shape)} and ids {tuple(ids.shape)} do not fit together")
    if target is not None:
        _need(target, "target", (_I64,), 1, (R,), dev, rows=True)
    if not 0 < vocab <= Vp:
        raise ValueError(f"vocab {vocab} must lie in [1, {Vp}], the logits' columns")


def distill_fwd_bwd(logits, ids, teacher, weight, vocab, temperature=1.0, target=None, hard=0.0):
    """Loss against a teacher's top logits, and its gradient, beside ce_fwd_bwd (lp_distill_fwd_bwd): logits [R, Vp] (fp32 or bf16; columns >= vocab are padding), ids
    int64 or int32 [R, K] and teacher fp32 or bf16 [R, K] the teacher's best tokens and their logits (ids outside [0, vocab): missing entries; K <= 1024), weight fp32
    [R] (rows of weight 0 are skipped), temperature from 1e-6 to 1e6, target int64 [R] labels for the share `hard` of the loss.
    loss = (1 - hard) temperature^2 KL(softmax(teacher / temperature) || softmax(logits / temperature)) + hard CE(target)
    -> (loss [R] fp32, dlogits bf16 [R, Vp], weighted as in ce_fwd_bwd)."""
    try:
        R, Vp = logits.shape
        K, dev = ids.shape[1], logits.device
        fine = (logits.is_cuda and (logits.dtype is _F32 or logits.dtype is _BF16) and logits.stride(1) == 1 and (ids.dtype is _I64 or ids.dtype is _I32)
                and (teacher.dtype is _F32 or teacher.dtype is _BF16) and ids.shape == (R, K) and teacher.shape == (R, K) and ids.device == dev and teacher.device == dev
                and (K <= 1 or (ids.stride(1) == 1 and teacher.stride(1) == 1))
                and (R <= 1 or (logits.stride(0) >= Vp and ids.stride(0) >= K and teacher.stride(0) >= K)) and weight.dtype is _F32 and weight.shape == (R,) and weight.device == dev
                and weight.is_contiguous() and 0 < vocab <= Vp
                and (target is None or (target.dtype is _I64 and target.shape == (R,) and target.device == dev and target.is_contiguous())))
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _distill_refusals(logits, ids, teacher, weight, vocab, target)
        if logits.shape[1] != 1:
            raise ValueError("distill_fwd_bwd: rows must be contiguous")
    loss = torch.empty((R,), device=dev, dtype=_F32)
    d = torch.empty((R, Vp), device=dev, dtype=_BF16) if Vp % 2 == 0 else torch.empty((R, Vp + 1), device=dev, dtype=_BF16)[:, :Vp]
    if R:
        L, ld = _lib.lib(), Vp + (Vp & 1)
        _call(dev, L, "lp_distill_fwd_bwd", L.lp_distill_fwd_bwd, logits.data_ptr(), 1 if logits.dtype is _F32 else 0, max(logits.stride(0), Vp), ids.data_ptr(),
              1 if ids.dtype is _I64 else 0, max(ids.stride(0), K), teacher.data_ptr(), 1 if teacher.dtype is _F32 else 0, max(teacher.stride(0), K), K, weight.data_ptr(),
              None if target is None else target.data_ptr(), float(temperature), float(hard), loss.data_ptr(), d.data_ptr(), ld, R, vocab, ld)
    return loss, d


# ---- serving many continuations of one prompt (csrc/lp_serve.cu, lp_sample.cu, lp_prefixattn.cu): a step's tables and pages, rotary positions and cache rows, attention over a prefix
# that the batch shares, the next tokens ----------------------------------------------------------------------------------------------------------------------------------------------
_MOST = 2 ** 31 - 1      # the entry points' whole numbers have 32 bits, of which ctypes would take the low ones of a larger one


def _whole(x, name):
    x = int(x)
    if not -_MOST <= x <= _MOST:
        raise ValueError(f"{name} must be a whole number of 32 bits, got {x}")
    return x


def step_tables(lengths, new, page_table, free, used, page_size, rows):
    """The index tables of a step whose requests bring tokens, and the cache pages that these need (lp_step_tables): lengths int32 [B], cached rows; new int32 [B], tokens that each
    brings (0: none); page_table int32 [B, max_pages] (negative: no page yet), which gets pages for the new rows, in place, from free int32 [n], of which used int32 [1] have been given
    before (it grows; when the list is over, entries stay negative); rows: how many rows the step has room for.
    Entries that are pages already stay, whoever else holds them: a page that a shared prompt ends in has to be copied for each request before its first step (cache_copy_pages), or the requests get the
    same slots.
    -> (row_seq int32 [rows], row_pos int32 [rows], slots int64 [rows] = page * page_size + row of the page; row0 int32 [B + 1], each request's first row).  Rows that no request has are -1 in all
    three, rows without a page in slots."""
    try:
        (B,), dev, max_pages = lengths.shape, lengths.device, page_table.shape[1]
        fine = (lengths.is_cuda and lengths.dtype is _I32 and new.dtype is _I32 and page_table.dtype is _I32 and free.dtype is _I32 and used.dtype is _I32 and new.device == dev
                and page_table.device == dev and free.device == dev and used.device == dev and new.shape == (B,) and lengths.is_contiguous() and new.is_contiguous()
                and page_table.shape == (B, max_pages) and (page_table.stride(1) == 1 or max_pages <= 1) and (page_table.stride(0) >= max_pages or B <= 1) and free.dim() == 1 and free.is_contiguous()
                and used.shape == (1,))
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _need(lengths, "lengths", (_I32,), 1, contiguous=True)
        for t, n, shape in ((new, "new", lengths.shape), (used, "used", (1,)), (free, "free", None)):
            _need(t, n, (_I32,), 1, shape, lengths.device, contiguous=True)
        _need(page_table, "page_table", (_I32,), 2, (lengths.shape[0], page_table.shape[-1]), lengths.device, rows=True)
        raise ValueError("step_tables: the tables must be contiguous in their rows")
    rows, page_size, n_free, ld = _whole(rows, "rows"), _whole(page_size, "page_size"), free.shape[0], page_table.stride(0)
    if rows < 0:
        raise ValueError(f"rows must not be negative, got {rows}")
    slots, seq, pos, row0 = torch.empty((4 * rows + B + 1,), dtype=_I32, device=dev).split((2 * rows, rows, rows, B + 1))      # (one allocation: four take 2.4 us longer)
    slots = slots.view(_I64)
    if B == 0:
        return seq.fill_(-1), pos.fill_(-1), slots.fill_(-1), row0.zero_()
    L = _lib.lib()
    _call(dev, L, "lp_step_tables", L.lp_step_tables, lengths.data_ptr(), new.data_ptr(), page_table.data_ptr(), ld, max_pages, page_size, free.data_ptr(), n_free, used.data_ptr(), B, rows,
          seq.data_ptr(), pos.data_ptr(), slots.data_ptr(), row0.data_ptr())
    return seq, pos, slots, row0


def _rotary_check(x, name, dtypes, dim, device=None):
    _need(x, name, dtypes, dim, device=device)
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")


def _rotary_layout(layout):
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    return layout == "interleaved"


def _rotary_rows(positions, inv_freq, rows, D, dev):
    _whole(rows, "the number of rows")
    _need(positions, "positions", (_I32, _I64), 1, (rows,), dev, contiguous=True)
    _need(inv_freq, "inv_freq", (_F32,), 1, device=dev, contiguous=True)
    if 2 * inv_freq.numel() > D:
        raise ValueError(f"{inv_freq.numel()} frequencies turn {2 * inv_freq.numel()} dimensions, heads have {D}")


def rotary(x, positions, inv_freq, layout="half", scale=1.0, inverse=False, out=None):
    """Rotary positions (lp_rotary): x bf16 or fp32 [rows, heads, D]; positions int32 or int64 [rows]; inv_freq fp32 [n] (seqlm.rotary_table has the scaled ones and their `scale`): the first
    2 n dimensions of each head are turned, pairs (i, i + n) for layout "half" and (2 i, 2 i + 1) for "interleaved", and multiplied by `scale`.  inverse: turned back, which takes the gradient of the result to
    that of x.  Angles are formed in 64 bits from the position.  out: x itself, or memory apart from it.  -> out."""
    try:
        rows, heads, D = x.shape
        dev, kind, n = x.device, x.dtype, inv_freq.shape[0]
        xs = x.stride()
        fine = (x.is_cuda and rows <= _MOST and (kind is _BF16 or kind is _F32) and (xs[2] == 1 or D <= 1) and (positions.dtype is _I32 or positions.dtype is _I64) and positions.shape == (rows,)
                and positions.is_contiguous() and positions.device == dev and inv_freq.dtype is _F32 and inv_freq.dim() == 1 and inv_freq.is_contiguous() and inv_freq.device == dev and 2 * n <= D
                and (out is None or (out.dtype is kind and out.shape == x.shape and out.device == dev and (out.stride(2) == 1 or D <= 1))))
    except (AttributeError, ValueError, IndexError):
        fine = False
    inter = _rotary_layout(layout)
    if not fine:
        _rotary_check(x, "x", (_BF16, _F32), 3)
        rows, heads, D = x.shape
        dev, kind, xs = x.device, x.dtype, x.stride()
        _rotary_rows(positions, inv_freq, rows, D, dev)
        n = inv_freq.numel()
        if out is not None:
            _rotary_check(out, "out", (kind,), 3, dev)
            if out.shape != x.shape:
                raise ValueError(f"out must be {tuple(x.shape)}, got {tuple(out.shape)}")
    if out is None:
        out = torch.empty((rows, heads, D), dtype=kind, device=dev)
    if rows == 0 or heads == 0 or D == 0:
        return out
    ys = out.stride()
    L = _lib.lib()
    _call(dev, L, "lp_rotary", L.lp_rotary, x.data_ptr(), xs[0], xs[1], out.data_ptr(), ys[0], ys[1], 1 if kind is _F32 else 0, rows, heads, D, positions.data_ptr(),
          1 if positions.dtype is _I64 else 0, inv_freq.data_ptr(), n, int(inter), float(scale), int(bool(inverse)))
    return out


def rotary_append(q, k, v, positions, inv_freq, k_pool, v_pool, slots, layout="half", scale=1.0, q_out=None):
    """A step's queries and keys turned as by `rotary`, keys and values written to their cache rows in the same pass (lp_rotary_append): q [rows, H, D], k, v [rows, KVH, D] bf16 or fp32 (views of
    one product, say); k_pool, v_pool of the same type [pages, page_size, KVH, D]; slots int64 [rows] (step_tables): page * page_size + row of the page, rows whose slot is no row of the pool are
    left out; no slot comes twice.  -> q_out (q itself, if given so)."""
    try:
        rows, H, D = q.shape
        dev, kind, n, G = q.device, q.dtype, inv_freq.shape[0], k.shape[1]
        s, ks, vs, kp, vp = q.stride(), k.stride(), v.stride(), k_pool.stride(), v_pool.stride()
        fine = (q.is_cuda and rows <= _MOST and (kind is _BF16 or kind is _F32) and k.dtype is kind and v.dtype is kind and k_pool.dtype is kind and v_pool.dtype is kind and s[2] == ks[2] == vs[2] == kp[3] == vp[3] == 1
                and k.shape == (rows, G, D) and v.shape == (rows, G, D) and k_pool.shape[2:] == (G, D) and v_pool.shape == k_pool.shape and k.device == dev and v.device == dev and k_pool.device == dev
                and v_pool.device == dev and (positions.dtype is _I32 or positions.dtype is _I64) and positions.shape == (rows,) and positions.is_contiguous() and positions.device == dev
                and inv_freq.dtype is _F32 and inv_freq.dim() == 1 and inv_freq.is_contiguous() and inv_freq.device == dev and 2 * n <= D and slots.dtype is _I64 and slots.shape == (rows,)
                and slots.is_contiguous() and slots.device == dev
                and (q_out is None or (q_out.dtype is kind and q_out.shape == (rows, H, D) and q_out.device == dev and q_out.stride(2) == 1)))
    except (AttributeError, ValueError, IndexError):
        fine = False
    inter = _rotary_layout(layout)
    if not fine:
        _rotary_check(q, "q", (_BF16, _F32), 3)
        rows, H, D = q.shape
        dev, kind = q.device, q.dtype
        for t, name, dim in ((k, "k", 3), (v, "v", 3), (k_pool, "k_pool", 4), (v_pool, "v_pool", 4)):
            _rotary_check(t, name, (kind,), dim, dev)
        G = k.shape[1]
        if k.shape != (rows, G, D) or v.shape != k.shape or k_pool.shape[2:] != (G, D) or v_pool.shape != k_pool.shape:
            raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, k_pool {tuple(k_pool.shape)} and v_pool {tuple(v_pool.shape)} do not fit together")
        _rotary_rows(positions, inv_freq, rows, D, dev)
        _need(slots, "slots", (_I64,), 1, (rows,), dev, contiguous=True)
        n, s, ks, vs, kp, vp = inv_freq.numel(), q.stride(), k.stride(), v.stride(), k_pool.stride(), v_pool.stride()
        if q_out is not None:
            _rotary_check(q_out, "q_out", (kind,), 3, dev)
            if q_out.shape != q.shape:
                raise ValueError(f"q_out must be {tuple(q.shape)}, got {tuple(q_out.shape)}")
    if q_out is None:
        q_out = torch.empty((rows, H, D), dtype=kind, device=dev)
    if rows == 0 or D == 0:
        return q_out
    if k_pool.numel() == 0:      # no slot is one of its rows: the queries are turned all the same
        return rotary(q, positions, inv_freq, layout, scale, out=q_out)
    o = q_out.stride()
    d = _lib.RotaryAppendDesc(q.data_ptr(), s[0], s[1], q_out.data_ptr(), o[0], o[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], k_pool.data_ptr(), kp[0], kp[1], kp[2],
                              v_pool.data_ptr(), vp[0], vp[1], vp[2], positions.data_ptr(), inv_freq.data_ptr(), slots.data_ptr(), 1 if positions.dtype is _I64 else 0, n,
                              int(inter), 1 if kind is _F32 else 0, rows, H, G, D, k_pool.shape[0], k_pool.shape[1], float(scale))
    L = _lib.lib()
    _call(dev, L, "lp_rotary_append", L.lp_rotary_append, C.byref(d))
    return q_out


def _prefix_refusals(q, k, v, lengths, prefix, new, page_table, prefix_k, prefix_v, out):
    for t, n, dim in ((q, "q", 4), (k, "k", 4), (v, "v", 4), (out, "out", 4), (prefix_k, "prefix_k", 3), (prefix_v, "prefix_v", 3)):
        if t is not None:
            _rotary_check(t, n, (_BF16,), dim, q.device if t is not q else None)
    B, T, H, D = q.shape
    G, dev = k.shape[2], q.device
    if k.shape[3] != D or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    if out is not None and out.shape != q.shape:
        raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    _need(lengths, "lengths", (_I32,), 1, (B,), dev, contiguous=True)
    if new is not None:
        _need(new, "new", (_I32,), 1, (B,), dev, contiguous=True)
    if page_table is not None:
        _need(page_table, "page_table", (_I32,), 2, (B, page_table.shape[-1]), dev, rows=True)
        if prefix_k is not None or prefix_v is not None:
            raise ValueError("the prefix lies in the pages of the table, or in prefix_k and prefix_v: not both")
    else:
        if k.shape[0] < B:
            raise ValueError(f"{B} requests need a page table or a cache of their own each, k holds {k.shape[0]}")
        if prefix and (prefix_k is None or prefix_v is None):
            raise ValueError("without a page table the prefix is prefix_k and prefix_v")
        for t, n in ((prefix_k, "prefix_k"), (prefix_v, "prefix_v")):
            if prefix and t.shape != (prefix, G, D):
                raise ValueError(f"{n} must be {(prefix, G, D)}, got {tuple(t.shape)}")
    raise ValueError("prefix_attention: heads must be contiguous")


def prefix_attention(q, k, v, lengths, prefix, new=None, page_table=None, prefix_k=None, prefix_v=None, scale=None, out=None):
    """Attention of a batch whose requests share their first `prefix` rows, which are read once for all of them (lp_prefix_attention): q bf16 [B, T, H, D], the requests' new tokens; lengths int32 [B], rows
    of each before these, the prefix among them; new int32 [B] or None (T), tokens that each brings, whose keys and values are the cache's next rows already (rotary_append): token t sees the prefix and its
    request's rows up to its own.  With page_table int32 [B, max_pages]: k, v bf16 [pages, page_size, KVH, D] and each request's whole sequence in its pages (tables that begin with the same pages share
    them; a page that the prefix ends in is each request's own), the prefix read from those of request 0.  Without: own rows in k, v [B, rows, KVH, D], from row 0 on, the prefix in prefix_k, prefix_v [prefix, KVH, D].  Strides are free but for a contiguous last
    dimension and multiples of 8.  -> out bf16 [B, T, H, D]; rows of tokens that a request does not bring stay as they were (`out` given; its rows share no memory, and its span meets none of the
    inputs) or are unspecified.  A token that sees nothing is zeros.  T <= 256."""
    prefix = _whole(prefix, "prefix")
    try:
        B, T, H, D = q.shape
        P, S, G, Dk = k.shape
        dev = q.device
        fine = (q.is_cuda and q.dtype is _BF16 and k.dtype is _BF16 and v.dtype is _BF16 and Dk == D and v.shape == k.shape and k.device == dev and v.device == dev
                and lengths.dtype is _I32 and lengths.device == dev and lengths.shape == (B,) and lengths.is_contiguous())
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        fine = fine and qs[3] == ks[3] == vs[3] == 1 and (new is None or (new.dtype is _I32 and new.device == dev and new.shape == (B,) and new.is_contiguous()))
        pk = pv = None
        pks = pvs = (0, 0)
        if page_table is not None:
            max_pages = page_table.shape[1]
            fine = (fine and page_table.dtype is _I32 and page_table.device == dev and page_table.shape == (B, max_pages) and (page_table.stride(1) == 1 or max_pages <= 1)
                    and (page_table.stride(0) >= max_pages or B == 1) and prefix_k is None and prefix_v is None)
            table, ld = page_table.data_ptr(), page_table.stride(0)
        else:
            fine, max_pages, table, ld = fine and P >= B, 1, None, 0
            if prefix:
                fine = (fine and prefix_k.dtype is _BF16 and prefix_v.dtype is _BF16 and prefix_k.shape == (prefix, G, D) and prefix_v.shape == (prefix, G, D) and prefix_k.device == dev
                        and prefix_v.device == dev and prefix_k.stride(2) == 1 and prefix_v.stride(2) == 1)
                pk, pv, pks, pvs = prefix_k.data_ptr(), prefix_v.data_ptr(), prefix_k.stride(), prefix_v.stride()
        if out is not None:
            fine = fine and out.dtype is _BF16 and out.device == dev and out.shape == q.shape and out.stride(3) == 1
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _prefix_refusals(q, k, v, lengths, prefix, new, page_table, prefix_k, prefix_v, out)
    if out is None:
        out = torch.empty((B, T, H, D), dtype=_BF16, device=dev)
    if B == 0 or T == 0:
        return out
    os_ = out.stride()
    d = _lib.PrefixAttnDesc(q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], pk, pks[0], pks[1], pv, pvs[0], pvs[1],
                            out.data_ptr(), os_[0], os_[1], os_[2], table, ld, max_pages, P, S, lengths.data_ptr(), None if new is None else new.data_ptr(), prefix, B, T, H, G, D,
                            D ** -0.5 if scale is None else float(scale))
    L, ref = _lib.lib(), C.byref(d)
    need = L.lp_prefix_attention_workspace_bytes(ref)
    if need == 0:
        _lib.check(-1, "lp_prefix_attention")
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(dev, L, "lp_prefix_attention", L.lp_prefix_attention, ref, ws.data_ptr(), need)
    return out


def _setting(x, name, dtype, rows, dev):
    """a number for all rows, or a tensor of one each -> (its address or None, the number)"""
    if isinstance(x, torch.Tensor):
        _need(x, name, (dtype,), 1, (rows,), dev, contiguous=True)
        return x.data_ptr(), 0
    return None, max(-1, min(int(x), _MOST)) if dtype is _I32 else float(x)      # (top_k: more words than any row has)


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The next token of each row from given random numbers (lp_sample_tokens): logits fp32 or bf16 [rows, V]; uniform fp32 [rows] in [0, 1).  temperature, top_p, min_p (numbers or fp32 [rows]) and
    top_k (a number or int32 [rows]): of the words in the order of their logits, equal ones by index, the first top_k are kept (0: all), of them those before which less than top_p of their mass
    lies, of them those at least min_p times as likely as the likeliest; drawn is the first kept word, by index, up to which more than `uniform` of the kept mass lies.  temperature 0 takes the largest
    logit, the first of equal ones.  -> int64 [rows]; -1 for a row of -inf and NaN alone, which are never drawn.  Weights are held in units
    of 2^-43 of the largest, for top_p of 2^-35 (V > 131072: 2^-32).  V <= 376832."""
    try:
        R, V = logits.shape
        dev, kind, ld = logits.device, logits.dtype, logits.stride(0)
        fine = (logits.is_cuda and max(R, V) <= _MOST and (kind is _F32 or kind is _BF16) and (logits.stride(1) == 1 or V <= 1) and (R <= 1 or ld >= V) and uniform.dtype is _F32 and uniform.shape == (R,)
                and uniform.is_contiguous() and uniform.device == dev)
    except (AttributeError, ValueError, IndexError):
        fine = False
    if not fine:
        _need(logits, "logits", (_F32, _BF16), 2, rows=True)
        _whole(max(logits.shape), "a size of logits")
        _need(uniform, "uniform", (_F32,), 1, logits.shape[:1], logits.device, contiguous=True)
        raise ValueError("sample_tokens: rows must be contiguous")
    settings = [*_setting(temperature, "temperature", _F32, R, dev), *_setting(top_k, "top_k", _I32, R, dev), *_setting(top_p, "top_p", _F32, R, dev), *_setting(min_p, "min_p", _F32, R, dev)]
    out = torch.empty((R,), dtype=_I64, device=dev)
    L = _lib.stream32_lib()
    _call(dev, L, "lp_sample_tokens", L.lp_sample_tokens, logits.data_ptr(), 1 if kind is _F32 else 0, max(ld, V), uniform.data_ptr(), *settings, R, V, out.data_ptr())
    return out
