"""Token sampling: temperature, top-k, top-p (nucleus), min-p, repetition penalty, multinomial draw, and a draw from given
random numbers in one kernel (``Sampler.draw``)
(example-cli/src/model/sampling.rs:8-300; the reference's ``sample_token`` is a placeholder returning
``vocab/2`` and its repetition penalty is a TODO)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch


@dataclass
class SamplingConfig:
    temperature: float = 1.0
    top_k: int = 0            # 0 = disabled
    top_p: float = 1.0        # 1.0 = disabled
    repetition_penalty: float = 1.0
    seed: Optional[int] = None
    min_p: float = 0.0        # 0.0 = disabled

    def validate(self) -> None:
        if self.temperature < 0:
            raise ValueError("temperature must be >= 0")
        if self.top_k < 0:
            raise ValueError("top_k must be >= 0")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError("top_p must be in (0, 1]")
        if self.repetition_penalty <= 0:
            raise ValueError("repetition_penalty must be > 0")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError("min_p must be in [0, 1]")

    @staticmethod
    def greedy() -> "SamplingConfig":
        return SamplingConfig(temperature=0.0)


def softmax(logits: torch.Tensor) -> torch.Tensor:
    return torch.softmax(logits.float(), -1)


def apply_repetition_penalty(logits: torch.Tensor, history: torch.Tensor, penalty: float) -> torch.Tensor:
    """Divide positive / multiply negative logits of already generated tokens by ``penalty``.  Entries below zero stand for steps that
    had no token (``Sampler.draw``) and change nothing."""
    if penalty == 1.0 or history.numel() == 0:
        return logits
    out = logits.clone()
    token = history.clamp_min(0)
    g = out.gather(-1, token)
    # a missing token is sent to place 0 with what that place gets anyway, so that all writers of a place agree
    keep = (history < 0) & ~(history == 0).any(-1, keepdim=True)
    out.scatter_(-1, token, torch.where(keep, g, torch.where(g > 0, g / penalty, g * penalty)))
    return out


def apply_top_k_to_probs(probs: torch.Tensor, k: int) -> torch.Tensor:
    if k <= 0 or k >= probs.shape[-1]:
        return probs
    kth = probs.topk(k, -1).values[..., -1:]
    p = torch.where(probs < kth, torch.zeros_like(probs), probs)
    return p / p.sum(-1, keepdim=True)


def apply_top_p_to_probs(probs: torch.Tensor, top_p: float) -> torch.Tensor:
    if top_p >= 1.0:
        return probs
    sp, si = probs.sort(-1, descending=True)
    cum = sp.cumsum(-1)
    keep = cum - sp < top_p                   # always keeps the most probable token
    sp = torch.where(keep, sp, torch.zeros_like(sp))
    p = torch.zeros_like(probs).scatter_(-1, si, sp)
    return p / p.sum(-1, keepdim=True)


def apply_min_p_to_probs(probs: torch.Tensor, min_p: float) -> torch.Tensor:
    """Drop tokens of less than ``min_p`` times the largest probability."""
    if min_p <= 0.0:
        return probs
    p = torch.where(probs < min_p * probs.amax(-1, keepdim=True), torch.zeros_like(probs), probs)
    return p / p.sum(-1, keepdim=True)


def multinomial_sample(probs: torch.Tensor, generator: Optional[torch.Generator] = None) -> torch.Tensor:
    return torch.multinomial(probs, 1, generator=generator).squeeze(-1)


class Sampler:
    """Callable ``logits [B, V] -> tokens [B]`` carrying the configuration and the generated history."""

    def __init__(self, config: Optional[SamplingConfig] = None, device=None):
        self.config = config or SamplingConfig()
        self.config.validate()
        self.history: Optional[torch.Tensor] = None
        self._gen = None
        if self.config.seed is not None:
            self._gen = torch.Generator(device=device or "cpu").manual_seed(self.config.seed)

    def __call__(self, logits: torch.Tensor) -> torch.Tensor:
        c = self.config
        logits = logits.float()
        if self.history is not None:
            logits = apply_repetition_penalty(logits, self.history, c.repetition_penalty)
        if c.temperature == 0.0:
            tok = logits.argmax(-1)
        else:
            probs = softmax(logits / c.temperature)
            probs = apply_min_p_to_probs(apply_top_p_to_probs(apply_top_k_to_probs(probs, c.top_k), c.top_p), c.min_p)
            gen = self._gen if (self._gen is not None and self._gen.device == probs.device) else None
            tok = multinomial_sample(probs, gen)
        t = tok.view(-1, 1)
        self.history = t if self.history is None else torch.cat([self.history, t], 1)
        return tok

    def draw(self, logits: torch.Tensor, uniform: torch.Tensor) -> torch.Tensor:
        """``logits [B, V]`` and numbers ``uniform [B]`` in ``[0, 1)`` -> tokens ``[B]`` by the same settings: one kernel on CUDA
        (``ops.sampling.sample_tokens``), a function of its arguments and the history alone.  Of tokens that tie at ``top_k`` it keeps
        the first (``__call__`` keeps them all); a row without a possible token gives -1."""
        from ..ops.sampling import sample_tokens
        c = self.config
        if self.history is not None and c.repetition_penalty != 1.0:
            logits = apply_repetition_penalty(logits.float(), self.history, c.repetition_penalty)
        tok = sample_tokens(logits, uniform, temperature=c.temperature, top_k=c.top_k, top_p=c.top_p, min_p=c.min_p)
        t = tok.view(-1, 1)
        self.history = t if self.history is None else torch.cat([self.history, t], 1)
        return tok

    def reset(self) -> None:
        self.history = None


def sample_token(logits: torch.Tensor, config: Optional[SamplingConfig] = None) -> int:
    return int(Sampler(config)(logits.view(1, -1))[0])
