"""The per-micro-batch loss assembly of the FSDP actor on the HIP path.

``CausalLM.forward_backward_fn`` keeps the contract of
axon/models/fsdp_models.py:183-279: run the model forward, evaluate the registry loss
(with the sampler correction hook), subtract the entropy bonus, add the KL penalty, scale by
``dp_replicas`` and report the same metrics.  The model forward itself is the caller's: ``module`` is
any callable ``module(model_inputs, meta_info) -> {"log_probs": ..., "entropys": ...}`` (in the
reference that is ``CausalLM.forward_fn`` around the HF model and the fused LM head).

The two side terms and the two entropy metrics come out of ONE kernel pass
(``axon_side_terms``) instead of three ``agg_loss`` calls and an elementwise KL chain.

A model with routed experts may return its ``router_logits`` too: their balance loss (``router_balance_loss``) is then one
more term (the reference has none here).  So are the ``distill_losses`` of a model that compares itself with a teacher.
"""

from __future__ import annotations

import numpy as np
import torch

from axon_amd import _lib, _ops
from axon_amd.trainer.algos.loss import compute_loss_fn, router_balance_loss
from axon_amd.utils.rl.sampler import compute_sampler_corr_metrics_from_logprobs


class _SideTerms(torch.autograd.Function):
    """(aggregated entropy, aggregated KL penalty, raw sums) with gradients to entropy / log_probs."""

    @staticmethod
    def forward(ctx, entropy, log_probs, ref_log_probs, mask, rows, kl_type, kl_plus, agg):
        acc, agg_w, grad_kl = _ops.side_terms(entropy, log_probs, ref_log_probs, mask, rows, kl_type=kl_type,
                                              kl_plus=kl_plus, **agg)
        ctx.save_for_backward(agg_w, grad_kl, acc)
        ctx.dtypes = (entropy.dtype if entropy is not None else None, log_probs.dtype if log_probs is not None else None)
        ctx.mark_non_differentiable(acc)
        return acc[0].clone(), acc[1].clone(), acc

    @staticmethod
    def backward(ctx, g_ent, g_kl, _g_acc):
        agg_w, grad_kl, acc = ctx.saved_tensors
        d_ent = d_lp = None
        if agg_w is not None and ctx.needs_input_grad[0]:
            d_ent = _ops.scale_f32(agg_w, g_ent, acc[5]).to(ctx.dtypes[0])
        if grad_kl is not None and ctx.needs_input_grad[1]:
            d_lp = _ops.scale_f32(grad_kl, g_kl, acc[5]).to(ctx.dtypes[1])
        return d_ent, d_lp, None, None, None, None, None, None


def _router_term(b, cu, entropy, args, router_logits, router_expert_ids):
    """``(balance loss, largest load of an expert relative to the mean of its layer, misfit)``, all on the device.  All tokens of
    a packed batch count, in a padded one those of ``attention_mask`` (where the batch has it).  Routers that saw fewer tokens
    than a padded batch has entries saw them packed (remove-padding): the mask's tokens, row after row; ``misfit`` (else None)
    is how many tokens too many the mask has for that."""
    if router_logits is None:
        raise ValueError("router_aux_loss_coef is set, but the model returned no router_logits")
    if "router_top_k" not in args:
        raise ValueError("router_aux_loss_coef needs router_top_k, the experts per token")
    mask, seqs, misfit = (b.get("attention_mask", None) if cu is None else None), None, None
    if isinstance(router_logits, torch.Tensor):  # [layers, tokens, experts] or [tokens, experts]
        tokens = router_logits.shape[max(router_logits.dim() - 2, 0)]
    else:
        tokens = sum(t.numel() // max(t.shape[-1], 1) for t in router_logits[:1])
    per_sequence = args.get("router_balance_per_sequence", False)
    if mask is not None and tokens < mask.numel():
        ends = (mask != 0).reshape(-1, mask.shape[-1]).sum(-1).cumsum(0)
        seqs = torch.nn.functional.pad(ends if per_sequence else ends[-1:], (1, 0)).to(torch.int32)
        mask, misfit = None, (ends[-1] - tokens).float()
    elif per_sequence:
        seqs = cu
        if seqs is None:  # padded: a row is a sequence
            rows = entropy.shape[0]
            length, odd = divmod(tokens, max(rows, 1))
            if odd:
                raise ValueError(f"router_logits of {tokens} tokens do not belong to {rows} rows of one length")
            seqs = torch.arange(rows + 1, device=entropy.device, dtype=torch.int32) * length
    balance, counts = router_balance_loss(router_logits, args["router_top_k"], token_mask=mask, cu_seqlens=seqs,
                                          expert_ids=router_expert_ids, score_fn=args.get("router_score_fn", "softmax"))
    counts = counts.view(-1, counts.shape[-1]).float()
    load = counts.amax(1) * counts.shape[1] / counts.sum(1).clamp(min=1)
    return balance, load.max(), misfit


def loss_from_outputs(data, log_prob, entropy, meta_info, router_logits=None, router_expert_ids=None, distill_losses=None):
    """Everything of ``forward_backward_fn`` after the model forward (fsdp_models.py:224-278).

    With ``loss_fn_args["router_aux_loss_coef"]`` the balance loss of ``router_logits`` times that coefficient is added, as
    the mean over the micro-batches of a step and the data-parallel replicas (the other terms are their sums: they are
    divided by counts over all of these), with ``router_top_k``, ``router_score_fn`` ("softmax") and
    ``router_balance_per_sequence`` (False) from the same arguments.  Routers that saw a padded batch packed (remove-padding)
    are recognised by their number of tokens, which has to be that of ``attention_mask``.

    With ``loss_fn_args["distill_coef"]`` the ``distill_losses`` of the tokens (``distillation_from_logits``, in the shape of
    ``entropy``; the reference has no such term), aggregated over ``response_mask`` as the KL penalty is, are added times that
    coefficient.

    Returns ``(scaled_loss, metrics)``.  ``data.batch["log_probs"]`` is set; ``response_mask`` may be
    overwritten by the sampler correction hook, while the side terms keep the mask they were given
    (the reference captures it before the hook, :197-211).
    """
    loss_fn = meta_info["loss_fn"]
    loss_fn_args = meta_info["loss_fn_args"]
    dp_replicas = meta_info["dp_replicas"]
    n_micro_batches = meta_info.get("n_micro_batches", 1)

    b = data.batch
    response_mask = b["response_mask"]  # before compute_loss_fn can replace it
    cu = data.meta_info.get("cu_seqlens", None) if data.meta_info else None
    nps = data.non_tensor_batch.get("num_program_steps", None) if data.non_tensor_batch else None
    if nps is None:
        nps = b.get("num_program_steps", None)
    elif isinstance(nps, np.ndarray):
        nps = torch.from_numpy(nps.astype(np.int64))
    token_reduce = loss_fn_args.get("token_reduce", "sum")
    batch_reduce = loss_fn_args.get("batch_reduce", "token-mean")
    valid = {"token-mean": b.get("valid_token_count", None), "step-mean": b.get("valid_batch_size", None),
             "program-mean": b.get("valid_program_count", None)}[batch_reduce]
    agg = dict(token_reduce=token_reduce, batch_reduce=batch_reduce,
               num_program_tokens=b.get("num_program_tokens", None), num_program_steps=nps, valid_count=valid)

    b["log_probs"] = log_prob
    pg_loss, pg_metrics = compute_loss_fn(data, loss_fn=loss_fn, loss_fn_args=loss_fn_args)
    metrics = dict(pg_metrics)
    loss = pg_loss

    sampler_log_prob = b.get("sampler_log_probs", None)
    if loss_fn != "bypass_mode" and sampler_log_prob is not None:
        metrics.update(compute_sampler_corr_metrics_from_logprobs(log_prob=log_prob, sampler_log_prob=sampler_log_prob,
                                                                  response_mask=response_mask, cu_seqlens=cu))

    entropy_coef = loss_fn_args.get("entropy_coef", 0)
    kl_coef = loss_fn_args.get("kl_coef", 0)
    kl_type, kl_plus = (0, 0)
    ref = None
    if kl_coef != 0:
        assert "ref_log_prob" in b, "ref_log_prob is required for KL loss"
        ref = b["ref_log_prob"]
        kl_type, kl_plus = _ops.kl_type_of(loss_fn_args.get("kl_type", "low_var_kl"))
    _lib.require_device(entropy, "forward_backward_fn")
    rows = _ops.rows_of(entropy, cu)
    ent_in = entropy if entropy_coef != 0 else entropy.detach()
    ent_agg, kl_agg, acc = _SideTerms.apply(ent_in, log_prob if kl_type else None, ref, response_mask, rows, kl_type,
                                            kl_plus, agg)
    if entropy_coef != 0:
        loss = loss - ent_agg * entropy_coef
    if kl_coef != 0:
        loss = loss + kl_agg * kl_coef
    distill_coef = loss_fn_args.get("distill_coef", 0)
    distill_vals = []
    if distill_coef != 0:
        if distill_losses is None:
            raise ValueError("distill_coef is set, but the model returned no distill_losses")
        if distill_losses.shape != entropy.shape:
            raise ValueError(f"distill_losses {tuple(distill_losses.shape)} do not lie beside the tokens {tuple(entropy.shape)}")
        kept = torch.where(response_mask != 0, distill_losses, 0.0)  # what another token's loss is does not matter
        distill, _, _ = _SideTerms.apply(kept, None, None, response_mask, rows, 0, 0, agg)
        loss = loss + distill * distill_coef
        distill_vals = [distill.detach()]
    router_coef = loss_fn_args.get("router_aux_loss_coef", 0)
    router_vals = []
    if router_coef != 0:
        balance, load, misfit = _router_term(b, cu, entropy, loss_fn_args, router_logits, router_expert_ids)
        loss = loss + balance * (router_coef / (n_micro_batches * dp_replicas))
        router_vals = [balance.detach(), load] + ([misfit] if misfit is not None else [])
    # one readback for pg_loss and the side-term metrics
    vals = torch.stack([pg_loss.detach().float(), acc[0], acc[1], acc[2], acc[4], *distill_vals, *router_vals]).tolist()
    distill_val = vals.pop(5) if distill_vals else None
    if vals[7:] and vals[7] != 0:
        raise ValueError("router_logits are neither of the padded batch's tokens nor of those that attention_mask keeps")
    metrics["pg_loss"] = vals[0] * n_micro_batches
    metrics["entropy"] = vals[1] * n_micro_batches
    metrics["entropy_token_mean"] = vals[3] / max(vals[4], 1.0)
    if kl_coef != 0:
        metrics["kl_loss"] = vals[2] * n_micro_batches
        metrics["kl_coef"] = kl_coef
    if distill_vals:
        metrics["distill_loss"] = distill_val * n_micro_batches
        metrics["distill_coef"] = distill_coef
    if router_vals:
        metrics["router_balance_loss"] = vals[5]
        metrics["router_max_load"] = vals[6]
        metrics["router_aux_loss_coef"] = router_coef
    return loss * dp_replicas, metrics


class CausalLM:
    @staticmethod
    def forward_backward_fn(module, data, meta_info):
        """Per micro-batch forward + loss; ``data`` is a DataProto.  Returns ``(scaled_loss, metrics)``."""
        model_inputs = {**data.batch, **data.non_tensor_batch}
        result = module(model_inputs, {**meta_info, "temperature": meta_info["temperature"], "calculate_entropy": True})
        return loss_from_outputs(data, result["log_probs"], result["entropys"], meta_info, result.get("router_logits", None),
                                 result.get("router_expert_ids", None), result.get("distill_losses", None))
