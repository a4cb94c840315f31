"""Several tokens per position through the LM head: the best alternatives, or given ones, without the logits.

``linear_cross_entropy`` scores one label per position.  A teacher that stores its alternatives, a scorer that reports
them and a student that is trained on them need more (the reference has no such op):

    r = linear_top_logprobs(hidden, weight, k, labels, temperature)             # TopLogprobs
    logprobs, entropy = linear_token_logprobs(hidden, weight, r.top_ids, temperature)

* ``hidden`` ``[..., H]`` and ``weight`` ``[V, H]`` as ``linear_cross_entropy`` takes them (computed in bf16 with fp32
  accumulation; fp16 and fp32 operands are rounded first and receive their gradients in their own dtype), ``H`` a multiple
  of 32; outputs are fp32 in the shape of ``hidden`` without its last dimension (and with ``k`` behind it);
* both are differentiable with respect to ``hidden`` and ``weight`` through log-probabilities and entropy; the ids of the
  alternatives are constants.  The backward takes the fp32 logits that the forward has kept for it where those of all
  tokens take at most 2.5 GB (and memory has room for as much again), and recomputes them else: to the same gradients of
  alternatives, bit for bit, while the log-probabilities of given tokens, which come from the kept logits or from a dot per
  token, and their gradients may differ in the last bits;
* the alternatives (at most 128) are ordered by the product's fp32 result, before temperature and soft cap (which keep that
  order, but may round different logits to one), equal ones by ascending id; a position's fp32 logits are held while its
  block of tokens is selected from (2.5 GB whatever the number of tokens), never all of them.  A label that is one of them
  has its log-probability from a dot of its own, which may differ from the alternative's in the last bits;
* given tokens (at most 512 per position): an id outside the vocabulary is a filler, with log-probability 0 and no gradient;
  an id may occur more than once.
"""

from __future__ import annotations

import torch

from axon_amd import _lib, _ops
from axon_amd.utils.kernel.linear_cross_entropy import _warn_rounded_to_bf16
from axon_amd.utils.torch.ops import TopLogprobs

__all__ = ["linear_top_logprobs", "linear_token_logprobs"]

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _operands(what, hidden, weight, temperature, logit_softcapping):
    """Checked operands as rows in bf16, and the kernels' scalars."""
    if hidden.dtype not in _FLOATS or weight.dtype not in _FLOATS:
        raise ValueError(f"{what}: hidden and weight must be bf16, fp16 or fp32")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not match")
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"{what}: temperature must be positive, got {temperature}")
    cap = 0.0 if logit_softcapping is None else float(logit_softcapping)
    if not 0.0 <= cap < float("inf"):
        raise ValueError(f"{what}: logit_softcapping must be positive, got {logit_softcapping}")
    _lib.require_device(hidden, what)
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        _warn_rounded_to_bf16(hidden.dtype, weight.dtype, what)
    rows = hidden.reshape(-1, hidden.shape[-1]).to(torch.bfloat16)
    return _ops.on_16_bytes(rows.contiguous()), _ops.on_16_bytes(weight.to(torch.bfloat16).contiguous()), 1.0 / temperature, cap


class _LinearAlternatives(torch.autograd.Function):
    """The k best tokens of every row (``ids`` None) or given ones, and a label: their log-probabilities."""

    @staticmethod
    def forward(ctx, hidden, weight, k, ids, labels, temperature, logit_softcapping, what, grad_enabled):
        ctx.set_materialize_grads(False)
        rows, w, inv_t, cap = _operands(what, hidden, weight, temperature, logit_softcapping)
        batch, n = hidden.shape[:-1], rows.shape[0]
        top_ids = label_lp = None
        # needs_input_grad is true of a trainable weight under no_grad too, where no backward can come
        want_grad = grad_enabled and (ctx.needs_input_grad[0] or ctx.needs_input_grad[1])
        if ids is None:
            lab = labels.reshape(-1).contiguous() if labels is not None else None
            label_lp, entropy, lse, mean, lp, at, logits = _ops.lmhead_top(rows, w, k, lab, inv_t, cap, want_grad)
            top_ids = at.view(*batch, k)
            ctx.mark_non_differentiable(top_ids)
        else:
            lab, at = None, ids.reshape(n, ids.shape[-1])
            lp, entropy, lse, mean, logits = _ops.lmhead_tokens(rows, w, at, inv_t, cap, want_grad)
        ctx.save_for_backward(rows, w, at, lp, lab, label_lp, lse, mean, logits)
        ctx.shape, ctx.in_dtypes, ctx.scalars = hidden.shape, (hidden.dtype, weight.dtype), (inv_t, cap)
        return (label_lp.view(batch) if label_lp is not None else None, entropy.view(batch),
                lp.view(*batch, lp.shape[1]), top_ids)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_label, g_entropy, g_lp, _g_ids):
        if g_label is None and g_entropy is None and g_lp is None:
            return (None,) * 9
        rows, w, at, lp, lab, label_lp, lse, mean, logits = ctx.saved_tensors
        n, k = lp.shape
        g = torch.zeros_like(lp) if g_lp is None else g_lp.reshape(n, k)
        if g_label is not None:  # the label is one more token of its position
            at = torch.cat([lab[:, None].to(at.dtype), at], 1)
            lp = torch.cat([label_lp[:, None], lp], 1)
            g = torch.cat([g_label.reshape(n, 1), g], 1)
        g_en = None if g_entropy is None else g_entropy.reshape(n)
        d_hidden, d_weight = _ops.lmhead_tokens_backward(g, g_en, rows, w, at, lp, lse, mean, *ctx.scalars, logits)
        return d_hidden.view(ctx.shape).to(ctx.in_dtypes[0]), d_weight.to(ctx.in_dtypes[1]), *(None,) * 7


def linear_top_logprobs(hidden, weight, k, labels=None, temperature=1.0, logit_softcapping=None) -> TopLogprobs:
    """The ``k`` best tokens of every position with their log-probabilities, the entropy and, with ``labels`` (int32 or
    int64, one per position; outside the vocabulary: log-probability 0 and no gradient), the labels' log-probabilities."""
    if labels is not None and labels.shape != hidden.shape[:-1]:
        raise ValueError(f"linear_top_logprobs: labels {tuple(labels.shape)} do not lie beside hidden {tuple(hidden.shape)}")
    return TopLogprobs(*_LinearAlternatives.apply(hidden, weight, k, None, labels, temperature, logit_softcapping,
                                                  "linear_top_logprobs", torch.is_grad_enabled()))


def linear_token_logprobs(hidden, weight, token_ids, temperature=1.0, logit_softcapping=None):
    """``(logprobs [..., k], entropy [...])`` of the ``k`` given tokens of every position."""
    if token_ids.dim() != hidden.dim() or token_ids.shape[:-1] != hidden.shape[:-1]:
        raise ValueError(f"linear_token_logprobs: token_ids {tuple(token_ids.shape)} do not lie beside hidden "
                         f"{tuple(hidden.shape)}")
    _, entropy, logprobs, _ = _LinearAlternatives.apply(hidden, weight, 0, token_ids, None, temperature, logit_softcapping,
                                                        "linear_token_logprobs", torch.is_grad_enabled())
    return logprobs, entropy
