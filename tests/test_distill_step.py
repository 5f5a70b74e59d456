"""The SFT step on a teacher's top logits.  A teacher that names one token a row is the label, so such a step has to be the ordinary one; with several tokens the step's loss and
the head's gradient are those of the loss over the step's own logits.  On the CPU with every native op restated (oracle), and marked gpu on the kernels."""
import types

import pytest
import torch

from leopard_b200 import train as T
from leopard_b200.config import leopard_llava, reduced
from leopard_b200.native_weights import load_hf
from leopard_b200.weights import SyntheticCheckpoint
from oracle import draft as OD
from oracle import native_ops
from test_train_glue import _batch, _FakeEngine, _narrow


def distill_restated(logits, ids, teacher, weight, vocab, temperature=1.0, target=None, hard=0.0):
    loss, d = OD.distill(logits, ids, teacher, weight, vocab, temperature, target, hard)
    return loss.float(), d.to(torch.bfloat16)


@pytest.fixture
def cpu(monkeypatch):
    cfg = _narrow(reduced(leopard_llava(), vit_layers=1, dec_layers=1, vocab=324))
    ck = SyntheticCheckpoint(cfg, seed=5)
    restated = types.SimpleNamespace(**{k: getattr(native_ops, k) for k in dir(native_ops) if not k.startswith("__")}, distill_fwd_bwd=distill_restated)
    monkeypatch.setattr(T, "ops", restated)
    monkeypatch.setattr(T._lib, "lib", lambda: types.SimpleNamespace(lp_grad_norm_workspace_bytes=lambda: 4096))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    return cfg, lambda: _FakeEngine(cfg, ck, load_hf(cfg, lambda n: ck[n], device="cpu")), restated


def labels_as_teacher(labels, vocab):
    """one token a row: the next label; where there is none (weight 0) nothing"""
    ids = torch.full((*labels.shape, 2), -1, dtype=torch.int64)
    ids[:, :-1, 1] = torch.where(labels[:, 1:] >= 0, labels[:, 1:], vocab + 7)
    return ids, torch.randn(ids.shape, generator=torch.Generator().manual_seed(1))


def steps(make, batch, teacher, rate=1e-3, **kw):
    plain, taught = (T.SFTTrainer(make(), lr=rate, clip_grad=0.0, **k) for k in ({}, kw))
    return plain, plain.step(*batch), taught, taught.step(*batch, teacher=teacher)


@pytest.mark.parametrize("kw", [{}, dict(distill_hard=0.25), dict(distill_hard=1.0)])
def test_a_teacher_of_one_token_is_the_label(cpu, kw):
    cfg, make, _ = cpu
    batch = _batch(cfg, b=2, n_text=15, seed=3)
    plain, a, taught, b = steps(make, batch, labels_as_teacher(batch[1], cfg.dec.vocab), **kw)
    assert abs(a[0] - b[0]) < 1e-4 * abs(a[0]) and abs(a[1] - b[1]) < 2e-2 * a[1]
    for n in ("dec.lm_head", "dec.0.qkv_w", "embed"):
        g, h = plain.grad(n).float(), taught.grad(n).float()
        assert float((g - h).norm() / g.norm()) < 2e-2, n      # (both from dlogits rounded to bf16)


def test_several_tokens_and_micro_batches(cpu):
    cfg, make, restated = cpu
    seen = []

    def spy(*a, **kw):
        seen.append((a, kw))
        return distill_restated(*a, **kw)
    restated.distill_fwd_bwd = spy
    one, two = _batch(cfg, b=1, n_text=15, seed=4), _batch(cfg, b=1, n_text=15, seed=5)
    g = torch.Generator().manual_seed(2)
    teachers = [(torch.randint(-1, cfg.dec.vocab, (*x[0].shape, 5), generator=g), torch.randn(*x[0].shape, 5, generator=g)) for x in (one, two)]
    tr = T.SFTTrainer(make(), distill_temperature=2.0, distill_hard=0.5)
    loss, _ = tr.step(*[list(p) for p in zip(one, two)], teacher=teachers)
    assert len(seen) == 2
    parts = []
    for (a, kw), t, batch in zip(seen, teachers, (one, two)):
        logits, ids, values, weight, vocab = a
        assert vocab == cfg.dec.vocab and kw["temperature"] == 2.0 and kw["hard"] == 0.5
        assert torch.equal(ids, t[0].reshape(-1, 5)) and torch.equal(values, t[1].reshape(-1, 5))
        assert torch.equal(kw["target"][:-1], batch[1].reshape(-1)[1:])
        parts.append(float((OD.distill(logits, ids, values, weight, vocab, 2.0, kw["target"], 0.5)[0] * weight.double()).sum()) * 2)
    assert abs(loss - sum(parts) / 2) < 1e-4 * abs(loss)


def test_refusals(cpu):
    cfg, make, _ = cpu
    batch = _batch(cfg, b=1, n_text=15, seed=3)
    tr = T.SFTTrainer(make())
    ids, values = labels_as_teacher(batch[1], cfg.dec.vocab)
    for bad in ((ids,), (ids, values[:, :-1]), (ids, values[..., :1]), (ids[0], values[0])):
        with pytest.raises(ValueError, match="teacher"):
            tr.step(*batch, teacher=bad)
    with pytest.raises(ValueError):
        tr.step([batch[0]], [batch[1]], [batch[2]], [batch[3]], teacher=[])
    for kw in (dict(distill_temperature=0.0), dict(distill_hard=1.5)):
        with pytest.raises(ValueError, match="distill"):
            T.SFTTrainer(make(), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(distill_hard=0.25)])
def test_a_teacher_of_one_token_is_the_label_on_the_gpu(native_lib, kw):
    from leopard_b200.engine import PrefillEngine
    cfg = reduced(leopard_llava(), vit_layers=1, dec_layers=1, vocab=2048)
    ck = SyntheticCheckpoint(cfg, seed=5)
    batch = _batch(cfg, b=1, n_text=23, seed=3)
    plain, a, taught, b = steps(lambda: PrefillEngine(cfg, load_hf(cfg, lambda n: ck[n], "cuda")), batch, labels_as_teacher(batch[1], cfg.dec.vocab), **kw)
    assert abs(a[0] - b[0]) < 1e-4 * abs(a[0]) and abs(a[1] - b[1]) < 2e-2 * a[1]
    for n in ("dec.lm_head", "dec.0.qkv_w", "embed"):
        g, h = plain.grad(n).float(), taught.grad(n).float()
        assert float((g - h).norm() / g.norm()) < 2e-2, n
