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
