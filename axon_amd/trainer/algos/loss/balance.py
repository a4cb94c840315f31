"""Balance loss of a mixture of experts and the experts' loads, with the gradient of the router logits.

The term that a trainer adds to the policy loss of a model with routed experts, beside the entropy bonus and the KL penalty
(the reference leaves it to the model's own code, and has no operator for it).  For a layer and T unmasked tokens

    loss = sum_e (experts / (k T)) c_e * (1 / T) sum_t p_te

with ``p`` the router's scores of a token (softmax, or sigmoids divided by their sum) and ``c_e`` how often expert ``e`` was
chosen, which is a constant for the gradient: 1 where scores and choices are uniform.  The mean over the layers is returned;
with ``cu_seqlens`` the loss is formed for every sequence by itself and averaged over the sequences that have unmasked tokens.
"""

from __future__ import annotations

import torch

from axon_amd import _lib

__all__ = ["router_balance_loss"]

_SCORES = {"softmax": 0, "sigmoid": 1}


def router_balance_loss(router_logits, top_k: int, *, token_mask=None, cu_seqlens=None, expert_ids=None,
                        score_fn: str = "softmax"):
    """``(loss, counts)``: the balance loss (0-d fp32) and how often every expert was chosen (int64 ``[layers, experts]``).

    * ``router_logits``: one ``[..., experts]`` tensor per layer in a list or tuple (as a model returns them), one tensor
      ``[layers, tokens, experts]``, or ``[tokens, experts]`` of a single layer (``counts`` is then ``[experts]``); fp32 or
      bf16, at most 1024 experts, the same shape in all layers.  The gradient comes back in the logits' type.
    * ``top_k``: experts per token.  The choices are the ``top_k`` largest logits, equal ones by ascending expert and a NaN as
      -inf (the loss of a batch that has one is NaN), or ``expert_ids`` (int32 or int64, ``[..., top_k]`` per layer in the
      same arrangement): what the router chose, where that is not the order of these logits (a selection bias, replayed
      routes).  An id outside the experts chooses nothing.
    * ``token_mask``: as many entries as tokens, shared by the layers; a token counts where it is not zero (what its
      row holds does not matter otherwise).
    * ``cu_seqlens``: int32 ``[sequences + 1]``: the loss per sequence, averaged.  Tokens of no sequence count nowhere.
    * ``score_fn``: ``"softmax"`` or ``"sigmoid"``.

    A batch without unmasked tokens has loss 0 and a zero gradient.  Nothing is read back; sums repeat bit for bit."""
    what = "router_balance_loss"
    if isinstance(top_k, bool) or not isinstance(top_k, int):
        raise TypeError(f"{what}: top_k must be an int, got {type(top_k).__name__}")
    single = isinstance(router_logits, torch.Tensor) and router_logits.dim() == 2
    stacked = isinstance(router_logits, torch.Tensor) and not single
    if stacked and router_logits.dim() != 3:
        raise ValueError(f"{what}: a tensor of router logits must be [tokens, experts] or [layers, tokens, experts], got "
                         f"{tuple(router_logits.shape)}")
    tensors = [router_logits] if isinstance(router_logits, torch.Tensor) else list(router_logits)
    if not tensors or (stacked and router_logits.shape[0] == 0):
        raise ValueError(f"{what}: no layers")
    if any(t.dim() < 2 or t.shape[-1] < 1 for t in tensors):
        raise ValueError(f"{what}: every layer's logits must be [..., experts]")
    experts = int(tensors[0].shape[-1])
    if not 1 <= top_k <= experts:
        raise ValueError(f"{what}: top_k must be between 1 and the {experts} experts, got {top_k}")
    if score_fn not in _SCORES:
        raise ValueError(f"{what}: score_fn must be one of {sorted(_SCORES)}, got {score_fn!r}")
    if isinstance(expert_ids, torch.Tensor):
        expert_ids = list(expert_ids.unbind(0)) if expert_ids.dim() == 3 else [expert_ids]
    loss, counts = _lib.native().router_balance(tensors, stacked, top_k, token_mask, cu_seqlens, expert_ids, _SCORES[score_fn])
    return loss, counts[0] if single else counts
