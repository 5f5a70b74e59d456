"""Calls of the serving operators and of the sampler at the edges of what they say of themselves: pools without a page."""
import pytest
import torch

from leopard_b200 import _lib, ops
from oracle import serve as O

gpu = pytest.mark.gpu
BF16, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------ rotary positions and cache rows
@gpu
@pytest.mark.parametrize("pages, size, G", [(0, 16, 2), (3, 0, 2), (3, 16, 0)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_queries_are_turned_though_the_pool_has_no_rows(pages, size, G, dtype, layout):
    """no slot is a row of the pool, so that no key goes anywhere; the queries are those of `rotary`, to the last bit, as a new tensor, into one given and in place"""
    rows, H, D = 7, 3, 32
    q = torch.randn(rows, H, D, generator=gen(1), device="cuda").to(dtype)
    k, v = (torch.randn(rows, G, D, generator=gen(s), device="cuda").to(dtype) for s in (2, 3))
    pos = torch.arange(5, 5 + rows, device="cuda", dtype=I32)
    freq = (1000.0 ** (-torch.arange(8, dtype=torch.float64) / 8)).float().cuda()
    slots = torch.arange(rows, device="cuda")
    pools = [torch.zeros(pages, size, G, D, dtype=dtype, device="cuda") for _ in range(2)]
    want = ops.rotary(q, pos, freq, layout=layout, scale=1.5)
    assert not torch.equal(want, q)
    rest = (pos, freq, *pools, slots)
    given, mine = torch.full_like(q, 7.0), q.clone()
    got = ops.rotary_append(q, k, v, *rest, layout=layout, scale=1.5)
    assert torch.equal(got, want)
    assert ops.rotary_append(q, k, v, *rest, layout=layout, scale=1.5, q_out=given) is given and torch.equal(given, want)
    assert ops.rotary_append(mine, k, v, *rest, layout=layout, scale=1.5, q_out=mine) is mine and torch.equal(mine, want)
    with pytest.raises(ValueError, match="layout"):
        ops.rotary_append(q, k, v, *rest, layout="pairs")
    assert ops.rotary_append(q[:0], k[:0], v[:0], pos[:0], freq, *pools, slots[:0]).shape == (0, H, D)
