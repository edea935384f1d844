"""What a model answers, and how near a quantised model stays to its teacher.

The reference judges a quantised model by the argmax and the five best of its last logits
(bsi_ops/benchmarks/benchmark_performance_bsi.py:209-217). This module adds, over all positions and in one pass over the logits:

* ``token_logprobs``: log probability, rank and entropy for given tokens, with the top alternatives (rank 0 is the argmax, a rank
  below 5 the reference's top-5 hit);
* ``distillation_loss`` / ``distillation_loss_and_grad``: the divergence from a teacher's top entries, which is what
  ``token_logprobs(..., top_k)`` of the dense model leaves, and its gradient for the parameters that stay in full precision.

Logits are float32, float16 or bfloat16 CUDA tensors [..., vocabulary]; slices such as ``logits[:, :-1]`` are read where they lie.
Statistics are float32. There is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .linear import _ops


class TokenLogprobs(NamedTuple):
    """Tensors of the logits' leading shape; the last two with ``top_k`` behind it."""
    logprobs: torch.Tensor       # float32
    ranks: torch.Tensor          # int64: entries ahead of the token, 0 = the argmax; -1 where the token is not scored
    entropy: torch.Tensor        # float32, nats
    top_logprobs: torch.Tensor   # float32, descending
    top_ids: torch.Tensor        # int64; equal logits by ascending id


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of ``tokens`` (int64 or int32, the logits' leading shape) under ``softmax(logits)``.

    A token outside the vocabulary, such as an ignore index of -100, is not scored: logprob 0, rank -1; its row still has an entropy
    and alternatives. ``tokens=None`` scores none. ``top_k`` is at most 128. A row that holds a NaN or +inf, or nothing but -inf, has
    NaN log probabilities and entropy. The five tensors share one allocation: one that is kept keeps all. Nothing is recorded for
    gradients."""
    return TokenLogprobs(*_ops().token_logprobs(logits, tokens, int(top_k)))


_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _reduction(name: str) -> int:
    if name not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {name!r}")
    return _REDUCTIONS[name]


def distillation_loss(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, temperature: float = 1.0, tail: bool = False,
                      weights: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """Kullback-Leibler divergence of the student's ``softmax(logits / temperature)`` from a teacher's top entries, times
    ``temperature ** 2``; differentiable for ``logits``.

    ids, teacher: [..., entries] with the logits' leading shape, 1 to 512 entries a row. ``tail=False``: ``teacher`` holds logits (or
    log probabilities), renormalised over the listed entries at the temperature. ``tail=True``: it holds log probabilities at the
    temperature, and what they leave of 1 is compared with the student's mass outside the list (also what rounding leaves: where the
    list holds all that the teacher gives anything to and the student masks everything else, ``tail=False`` is the loss). Entries with an id outside the
    vocabulary are not there; an id listed twice counts with the sum of its probabilities.
    weights: a factor per row, 0 for padding: such a row is not read, its loss and gradient are 0. ``mean`` divides by their sum.
    Vocabularies of up to 2 ** 30; with the tail about 11 million, and a RuntimeError beyond."""
    return _ops().distill_loss(logits, ids, teacher, float(temperature), bool(tail), weights, _reduction(reduction))


def distillation_loss_and_grad(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, temperature: float = 1.0, tail: bool = False,
                               weights: Optional[torch.Tensor] = None, reduction: str = "mean"):
    """(distillation_loss(...), its gradient for ``logits``) from one pass: the logits come from memory once, so a loop that drives its
    backward pass by hand (``logits.backward(grad)``) moves a third less than through autograd. ``none``: one loss per row, the gradient
    of their sum."""
    return _ops().distill_fused(logits, ids, teacher, float(temperature), bool(tail), weights, _reduction(reduction))
