"""What a sampler does to the logits before it draws a token, on the HIP path.

A rollout that was sampled under penalties for repeated tokens, biases or a grammar was drawn from another distribution
than ``softmax(logits)``, and has to be scored under the one that it was drawn from: otherwise the importance ratio of the
sampler correction and of the policy loss compares two different things (the reference scores the raw logits and has no
such operator).  ``LogitControls`` says what is done, for the next token of every sequence (a decoder) or for every position
of a batch (a trainer):

    y  = z / r where z > 0, z * r elsewhere     the ids that the row's history holds (repetition_penalty r)
    y -= f * count + a                          the ids that count > 0 of its own tokens are (frequency_penalty f,
                                                presence_penalty a)
    y += bias                                   the given ids
    y  = -inf                                   what the row's mask forbids, whatever the logit is
    out = y / temperature

in this order.  Samplers differ in it: one that adds its biases before the penalties draws from another distribution, for ids
that are both biased and in the history, and its rollouts are not scored by this (biases added to the logits beforehand are).

``controlled_logits`` writes this out, ``controlled_logprobs_from_logits`` returns ``log softmax(out)[label]`` and the entropy of
``softmax(out)`` from one read of the logits.  Both are differentiable with respect to the logits; an id that is out
(``-inf``) has no gradient.
"""

from __future__ import annotations

import torch

from axon_amd import _lib

__all__ = ["LogitControls", "controlled_logits", "controlled_logprobs_from_logits"]


def _value(x, name):
    """A number for all sequences, or a tensor with one for each."""
    if isinstance(x, torch.Tensor):
        return 1.0, x  # a number that every check lets pass: the tensor is what counts
    if isinstance(x, bool) or not isinstance(x, (int, float)):
        raise TypeError(f"LogitControls: {name} must be a number or a tensor, got {type(x).__name__}")
    return float(x), None


class LogitControls:
    """Controls of logits.

    * ``token_ids``: the sequences' tokens (int32 or int64), ``[sequences, length]``, or packed ``[tokens]`` (also ``[1,
      tokens]``) with ``cu_seqlens`` ``[sequences + 1]``; needed for penalties.  An id outside the vocabulary counts for
      nothing, as does a token whose ``attention_mask`` (same arrangement) is 0: padding.
    * ``positions``: ``"all"``: the logits have a row for every token, whose history is its sequence up to and with that token
      (the row scores the token behind it); ``"last"``: a row for every sequence, whose history is all of it.
    * ``response_mask`` (same arrangement as the tokens): which of them the model has generated, for ``frequency_penalty``
      and ``presence_penalty``; None: all.  ``repetition_penalty`` counts the prompt too.
    * penalties and ``temperature``: a number, or a float tensor with one for each sequence (whose values are not looked at:
      a repetition penalty and a temperature have to be positive, 2^-126 or more).
    * ``bias_ids`` and ``bias``: ``[k]`` for all rows, or ``[sequences, k]``; an id outside the vocabulary is a filler, one
      that comes twice gets both; ``-inf`` takes an id out.
    * ``allowed``: int32 bit masks ``[words]`` (for all rows) or ``[masks, words]``, bit i of word w for token ``32 w + i``, 1
      where it may be sampled; the mask of every row is ``allowed_index`` (one per row, outside ``[0, masks)``: anything may
      be sampled), or its own.

    The tensors are held, not copied where their layout allows it, and read by every call."""

    def __init__(self, token_ids=None, cu_seqlens=None, *, positions: str = "all", response_mask=None, attention_mask=None,
                 repetition_penalty=1.0, frequency_penalty=0.0, presence_penalty=0.0, bias_ids=None, bias=None, allowed=None,
                 allowed_index=None, temperature=1.0):
        if positions not in ("all", "last"):
            raise ValueError(f"LogitControls: positions must be 'all' or 'last', got {positions!r}")
        if attention_mask is not None:
            if token_ids is None or attention_mask.shape != token_ids.shape:
                raise ValueError("LogitControls: attention_mask does not lie beside token_ids")
            token_ids = token_ids.masked_fill(attention_mask == 0, -1)
        self.positions = positions
        self._native = _lib.native().Controls(
            token_ids, cu_seqlens, positions == "all", response_mask, _value(repetition_penalty, "repetition_penalty"),
            _value(frequency_penalty, "frequency_penalty"), _value(presence_penalty, "presence_penalty"), bias_ids, bias, allowed,
            allowed_index, _value(temperature, "temperature"))


def _native(controls):
    if not isinstance(controls, LogitControls):
        raise TypeError(f"controls must be LogitControls, got {type(controls).__name__}")
    return controls._native


def controlled_logits(logits: torch.Tensor, controls: LogitControls, inplace: bool = False) -> torch.Tensor:
    """``logits`` ``[..., vocab]`` (fp32 or bf16) under ``controls``, in the logits' type, computed in fp32 and rounded once.
    ``inplace`` writes over them (not where they require a gradient)."""
    return _lib.native().controlled_logits(logits, _native(controls), bool(inplace))


def controlled_logprobs_from_logits(logits: torch.Tensor, labels: torch.Tensor, controls: LogitControls,
                                    inplace_backward: bool = False):
    """``(logprobs, entropy)`` of shape ``logits.shape[:-1]``, fp32: the log-probability of ``labels`` (``-inf`` where the
    controls take it out, 0 for a label outside the vocabulary) and the entropy under ``controls``.  A row that they leave nothing
    of has log-probability ``-inf``, entropy 0 and a zero gradient; one that holds a NaN that is not masked is NaN.  A row whose
    upstream gradients are 0 (a prompt's, say) is not read by the backward: its gradient is 0, whatever it holds.  With
    ``inplace_backward`` the backward writes d loss / d logits over the logits' storage, and can run once."""
    return _lib.native().controlled_logprobs(logits, labels, _native(controls), bool(inplace_backward))
