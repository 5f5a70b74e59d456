"""Rows of a weight that have neither teacher entries nor a label have no loss and no gradient, whatever their logits are; their neighbours are as without them."""
import pytest
import torch

import test_draft_ops as D
from leopard_b200 import ops


@D.gpu
@pytest.mark.parametrize("V, K, dtype, pad", [
    (900, 5, torch.float32, 0), (900, 5, D.BF16, 4), (6000, 30, torch.float32, 0), (40000, 30, torch.float32, 3), (40000, 30, D.BF16, 0),      # the persistent kernel
    (900, 300, torch.float32, 0), (32003, 9, torch.float32, 0), (32003, 9, D.BF16, 0), (40000, 300, D.BF16, 0),                                # rows off 16 bytes, many entries
    (140001, 9, torch.float32, 1),                                                                                                             # long rows
])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=2.0), dict(temperature=0.5, hard=0.25), dict(hard=0.5), dict(hard=1.0)])
def test_rows_without_terms(V, K, dtype, pad, kw):
    c = D.distill_case(9, V, K, V + K, dtype, pad, share=2.0)
    none = [1, 3, 4, 6, 8]
    c["ids"][none] = -1
    c["ids"][3] = torch.arange(K, device="cuda")
    c["teacher"][3] = -float("inf")                        # entries that have no mass
    c["target"][none] = -100
    want = ops.distill_fwd_bwd(vocab=V, **c, **kw)
    odd = c["logits"].clone()
    odd[1] = float("nan")
    odd[3, 7] = float("inf")
    odd[4] = -float("inf")
    odd[6, V // 2] = float("nan")
    odd[8] = float("inf")
    loss, d = ops.distill_fwd_bwd(vocab=V, **{**c, "logits": odd}, **kw)
    assert bool((loss[none] == 0).all()) and bool((d[none] == 0).all())
    assert torch.equal(loss, want[0]) and torch.equal(d, want[1])
    rest = [r for r in range(9) if r not in none]
    D.distill_close({k: v[rest] for k, v in c.items()}, V, got=(loss[rest], d[rest]), **kw)


@D.gpu
@pytest.mark.parametrize("V, K, dtype", [(900, 5, torch.float32), (40000, 30, D.BF16), (32003, 9, torch.float32), (140001, 9, torch.float32)])
@pytest.mark.parametrize("temperature", [1e-6, 1e6])
@pytest.mark.parametrize("size", [1.0, 1e9, 1e30, 3e38])
def test_the_ends_of_the_temperatures(V, K, dtype, temperature, size):
    """finite logits of any size: no gradient is infinite and nothing is NaN (a loss may pass fp32's range); the largest logit stands alone at the low end, and small ones are all equal at
    the high end"""
    c = D.distill_case(6, V, K, V, dtype, V % 2, share=2.0)
    c["logits"] = (c["logits"].float() / c["logits"].float().abs().amax() * size).to(dtype)
    loss, d = ops.distill_fwd_bwd(vocab=V, **c, temperature=temperature)
    assert not bool(loss.isnan().any()) and bool(d.isfinite().all())
    p = torch.softmax(c["logits"][:, :V].double() / temperature, -1)
    t = torch.zeros_like(p).scatter_add_(1, c["ids"], torch.softmax(c["teacher"].double() / temperature, -1))
    want = c["weight"].double()[:, None] * temperature * (p - t)
    # what counts in p has an exponent x within 64 of the largest, off by |x| 2^-23 of itself but for what all have in common; sums of up to 140,001 exponentials in parts of 256 and their
    # tree 2^-15, two-instruction exponentials 2^-21: 2^-12 of p and t is ample.  An exponential below 2^-126 is 0, and every one is at most its sum: p is off by
    # less than 2^-126 more, and the gradient by that times weight and temperature.  The gradient is rounded to bf16 once.
    tol = 2.0 ** -8 * want.abs() + c["weight"].double()[:, None] * temperature * (2.0 ** -12 * (p + t) + 2.0 ** -126) + 2.0 ** -133
    assert bool(((d[:, :V].double() - want).abs() <= tol).all())
