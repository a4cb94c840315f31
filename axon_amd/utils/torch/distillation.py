"""Distillation from a teacher's top logits, on the HIP path.

A teacher stores, for every position, the log-probabilities of its best tokens (``top_logprobs_from_logits``,
``linear_top_logprobs``); a student is trained to agree with them (the reference has no such operator).  With ``q`` the
teacher's probabilities of the given tokens and ``p`` the student's, ``softmax(logits / temperature)`` over the whole
vocabulary, a position's loss is one of

    "forward"   sum q log(q / p)
    "reverse"   sum p log(p / q)
    "jsd"       beta sum q log(q / m) + (1 - beta) sum p log(p / m),   m = beta q + (1 - beta) p

over

    "rest"         the given tokens and, as one more outcome, all others: 1 - sum q, and the student's probability of them
    "drop"         the given tokens alone, their probabilities as they are
    "renormalize"  the given tokens alone, the teacher's probabilities divided by their sum (any logits will do then; where it
                   gives all of them none, they stay at 0)

What the teacher has left is known to the rounding of its log-probabilities only, ``e = sum q (2^-21 (1 + |log q|) + s |log q|)`` (``s``
for those stored in fewer bits: 2^-7 for bf16, 2^-10 for fp16): a list of all tokens that there are, or of a teacher that is sure.
So ``"rest"`` counts 0 in ``"forward"`` where neither teacher nor student has more than ``e`` left (the teacher ``8 e`` where the
student has none), and the teacher has at least ``e`` left in ``"reverse"``: neither loss is infinite for a rounding.

A row is read once for its softmax statistics; the outcomes and their gradients are formed in 64 bits.  What the student has left
is a sum over the tokens that are not given, so that it is right where almost nothing is.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from axon_amd import _lib

__all__ = ["Distillation", "distillation_from_logits", "distillation_loss_from_logits"]

_DIVERGENCES = {"forward": 0, "reverse": 1, "jsd": 2}
_TAILS = {"drop": 0, "rest": 1, "renormalize": 2}


class Distillation(NamedTuple):
    """``loss``: the weighted sum, 0-d fp32, differentiable; ``losses`` and ``covered`` ``[...]`` fp32: every position's loss and
    the student's probability of the given tokens, constants."""

    loss: torch.Tensor
    losses: torch.Tensor
    covered: torch.Tensor


def _how(what, divergence, tail, beta, temperature):
    if divergence not in _DIVERGENCES:
        raise ValueError(f"{what}: divergence must be one of {sorted(_DIVERGENCES)}, got {divergence!r}")
    if tail not in _TAILS:
        raise ValueError(f"{what}: tail must be one of {sorted(_TAILS)}, got {tail!r}")
    beta, temperature = float(beta), float(temperature)
    if divergence == "jsd" and not 0.0 < beta < 1.0:
        raise ValueError(f"{what}: beta must be between 0 and 1, got {beta}")
    if not 2.0 ** -126 <= temperature <= torch.finfo(torch.float32).max:  # as a number of 32 bits that has a reciprocal
        raise ValueError(f"{what}: temperature must be positive (2^-126 or more, finite in 32 bits), got {temperature}")
    return _DIVERGENCES[divergence], _TAILS[tail], beta, temperature


def distillation_from_logits(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                             divergence: str = "forward", tail: str = "rest", beta: float = 0.5, temperature: float = 1.0,
                             inplace_backward: bool = False):
    """``(losses [...], covered [...])``: every position's loss, differentiable with respect to ``logits`` ``[..., vocab]`` (fp32
    or bf16), and the student's probability of the given tokens (a constant).

    ``teacher_ids`` (int32 or int64) and ``teacher_logprobs`` (floating point, constants): ``[..., k]``, at most 512 per
    position.  An id outside the vocabulary is a filler; one that comes twice is two outcomes.  A position without a token has
    loss 0 and no gradient; one whose logits hold a NaN, or nothing but -inf, is NaN.  A token that the student gives no
    probability at all has an infinite forward divergence, and so has ``"rest"`` where it leaves nothing and the teacher more than
    the rounding named above; a token that the teacher gives none (``-inf``) and the student some has an infinite reverse one, whose
    gradient is no number.  A position whose upstream gradient is 0 is not read by the backward:
    its gradient is 0, whatever it holds.  With ``inplace_backward`` the backward writes d loss / d logits over the logits'
    storage, and can run once.

    Where the weights of the losses are known beforehand, ``distillation_loss_from_logits`` reads the logits once less."""
    how = _how("distillation_from_logits", divergence, tail, beta, temperature)
    _, losses, covered = _lib.native().distill(logits, teacher_ids, teacher_logprobs, None, *how, bool(inplace_backward))
    return losses, covered


def distillation_loss_from_logits(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor,
                                  token_weights: torch.Tensor, *, divergence: str = "forward", tail: str = "rest",
                                  beta: float = 0.5, temperature: float = 1.0) -> Distillation:
    """``sum token_weights * losses`` of what ``distillation_from_logits`` returns, with the gradient formed in the forward, while
    a row's logits are at hand.  ``token_weights`` ``[...]``: mask, mean and coefficient of every position in one number; a
    position of weight 0 is not looked at, whatever it holds (loss, ``covered`` and gradient 0).

    The backward hands that gradient on where the upstream gradient is 1, as in ``loss.backward()``, and forms it anew
    from the saved logits where it is not (a factor that is known belongs into the weights)."""
    if not isinstance(token_weights, torch.Tensor):
        raise TypeError("distillation_loss_from_logits: token_weights must be a tensor")
    how = _how("distillation_loss_from_logits", divergence, tail, beta, temperature)
    return Distillation(*_lib.native().distill(logits, teacher_ids, teacher_logprobs, token_weights, *how, False))
