"""Token selection from a step's logits.  Greedy arg-max is what the reference's evaluation uses (generate(..., do_sample=False),
evaluations/models/llava_multiimg_siglip_anyres.py:448-452); temperature / top-k sampling is offered for the language models,
with top-p and min-p by the native draw (ops.sample_tokens).
Selection runs on the device; only the chosen ids come back to the host (the stopping criterion needs them)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import ops


@dataclass
class SamplingParams:
    temperature: float = 0.0       # 0: greedy
    top_k: int = 0                 # the likeliest words, and all that are equal to the last of them (0: the whole vocabulary)
    seed: Optional[int] = None
    top_p: float = 1.0             # of these the likeliest, before which less than this share of the mass lies (1: all)
    min_p: float = 0.0             # of these words at least this many times as likely as the likeliest (0: all)

    def __post_init__(self):
        # before a prompt has run and holds pages (what is not a number fails both)
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError(f"top_p must be above 0 and 1 at most, got {self.top_p}")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError(f"min_p must be from 0 to 1, got {self.min_p}")


def _draw(logits, u, temperature, top_p, min_p):
    """What ops.sample_tokens draws, for logits that are not on a GPU (the engines of the CPU backend): in 64 bits, from the words in their order."""
    t, top_p, min_p = torch.tensor([temperature, top_p, min_p], dtype=torch.float32).double()      # (settings come in 32 bits)
    z = logits.double()
    z = torch.where(z.isnan(), -torch.inf, z)
    z, order = torch.sort(z, dim=-1, descending=True, stable=True)
    top = z[:, :1]
    w = torch.where(z == top, 1.0, torch.exp((z - top) / t)).masked_fill(z == -torch.inf, 0.0)     # (beside an infinite one nothing counts)
    keep = (w.cumsum(-1) - w < top_p * w.sum(-1, keepdim=True)) & (w >= min_p)
    upto = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0)).cumsum(-1)
    return torch.where(top[:, 0] > -torch.inf, (upto > u.double()[:, None] * upto[:, -1:]).int().argmax(-1), -1)


class Sampler:
    def __init__(self, params: Optional[SamplingParams] = None):
        self.p = params or SamplingParams()
        self._gen = None

    def __call__(self, logits: torch.Tensor) -> torch.Tensor:
        """logits fp32 [n, vocab] -> ids int64 [n] (on the logits' device)."""
        p = self.p
        if p.temperature <= 0.0:
            return logits.argmax(-1)
        if self._gen is None:
            self._gen = torch.Generator(device=logits.device)
            if p.seed is not None:
                self._gen.manual_seed(p.seed)
        if 0 < p.top_k < logits.shape[-1]:
            # All words equal to the k-th stay, whatever else is set; ops.sample_tokens takes them by index, exactly top_k (and 20 us for a row of 128,256 where this takes 137, 42 and 270 for 64).
            z = logits / p.temperature
            logits = logits.masked_fill(z < z.topk(p.top_k, -1).values[:, -1:], float("-inf"))
        if p.top_p < 1.0 or p.min_p > 0.0:
            u = torch.rand(logits.shape[0], device=logits.device, generator=self._gen)
            draw = ops.sample_tokens if logits.is_cuda else _draw
            return draw(logits, u, temperature=p.temperature, top_p=max(p.top_p, 1e-30), min_p=p.min_p)      # (top_p goes there in 32 bits)
        return torch.multinomial(torch.softmax(logits / p.temperature, -1), 1, generator=self._gen).squeeze(-1)
