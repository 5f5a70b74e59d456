"""A step whose teacher is refused is none: nothing of it counts, and the next one is as if it had not been asked for.  On the CPU with every native op restated (oracle)."""
import ctypes as C

import pytest
import torch

from leopard_b200 import train as T
from test_distill_step import cpu, labels_as_teacher  # noqa: F401 (cpu: a fixture)
from test_train_glue import _batch


def test_a_refused_teacher_is_no_step(cpu):  # noqa: F811
    cfg, make, restated = cpu
    one, two = _batch(cfg, b=1, n_text=15, seed=3), _batch(cfg, b=1, n_text=15, seed=4)
    both = [list(p) for p in zip(one, two)]
    ids, values = labels_as_teacher(one[1], cfg.dec.vocab)
    good = (ids, values)
    wide = torch.zeros(*ids.shape[:2], 1025)
    hp = dict(lr=1e-2, decay_iters=10, warmup_iters=2)
    tr, fresh = T.SFTTrainer(make(), **hp), T.SFTTrainer(make(), **hp)
    logits = []
    gemm, restated.gemm = restated.gemm, lambda *a, **kw: logits.append(1) or gemm(*a, **kw)
    for bad in ((ids,), (ids, values[:, :-1]), (ids, values[..., :1]), (ids[0], values[0]), (ids, None), 3, (ids.short(), values), (ids, values.double()), (ids, values.half()),
                (wide.long(), wide), (ids[..., :0], values[..., :0]), (values, ids)):
        with pytest.raises((ValueError, TypeError), match="teacher"):
            tr.step(*one, teacher=bad)
        with pytest.raises((ValueError, TypeError), match="teacher"):
            tr.step(*both, teacher=[good, bad])
    for bad in ([good], good, 3):                          # as many as there are micro-batches, each a pair
        with pytest.raises((ValueError, TypeError), match="teacher"):
            tr.step(*both, teacher=bad)
    assert tr.iteration == 0 and not logits
    for _ in range(3):
        assert tr.step(*both, teacher=[good, None]) == fresh.step(*both, teacher=[good, None])
    assert tr.iteration == 3


@pytest.mark.parametrize("temperature", [1e-30, 9e-7, 1.1e6, 1e20, float("inf"), float("nan"), -1.0])
def test_temperatures_that_products_or_squares_do_not_hold(native_lib, cpu, temperature):  # noqa: F811
    with pytest.raises(ValueError, match="distill_temperature"):
        T.SFTTrainer(cpu[1](), distill_temperature=temperature)
    L, p = native_lib, C.c_void_p(1 << 20)
    assert L.lp_distill_fwd_bwd(p, 1, 16, p, 1, 2000, p, 1, 2000, 4, p, None, temperature, 0.0, p, p, 10, 2, 10, 10, None) == -1
    assert b"temperature" in L.lp_last_error()
