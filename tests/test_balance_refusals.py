"""What the balance loss refuses, on the host: nothing is launched."""

import ctypes

import pytest
import torch

from axon_amd import _lib
from axon_amd.trainer.algos.loss import router_balance_loss

X = torch.zeros(6, 8)
I64 = torch.int64


@pytest.mark.parametrize("k", [0, 9, -1])
def test_a_count_out_of_range_is_refused(k):
    with pytest.raises(ValueError, match="top_k"):
        router_balance_loss(X, k)


@pytest.mark.parametrize("k", [2.0, True, None])
def test_a_count_that_is_no_int_is_refused(k):
    with pytest.raises(TypeError, match="top_k"):
        router_balance_loss(X, k)


@pytest.mark.parametrize("logits", [[], X[0], X[None, None], [X, X[:5]], [X, X.bfloat16()], X.half(), torch.zeros(2, 1025),
                                    torch.zeros(0, 6, 8), [X[0]], torch.zeros(4, 0)])
def test_logits_that_do_not_fit_are_refused(logits):
    with pytest.raises(ValueError):
        router_balance_loss(logits, 1)


@pytest.mark.parametrize("kw", [dict(score_fn="tanh"), dict(token_mask=torch.ones(5)), dict(cu_seqlens=torch.zeros(2, 2, dtype=I64)),
                                dict(cu_seqlens=torch.zeros(0, dtype=I64)), dict(expert_ids=torch.zeros(6, 3, dtype=I64)),
                                dict(expert_ids=torch.zeros(5, 2, dtype=I64)), dict(expert_ids=torch.zeros(6, 2)),
                                dict(expert_ids=[torch.zeros(6, 2, dtype=I64)] * 2), dict(expert_ids=torch.zeros(2, 6, 2, dtype=I64))])
def test_arguments_that_do_not_fit_are_refused(kw):
    with pytest.raises(ValueError):
        router_balance_loss(X, 2, **kw)


def test_tensors_that_are_not_on_a_gpu_are_refused():
    with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
        router_balance_loss([X, X], 2)


def test_the_c_entry_points_check_their_arguments():
    lib = _lib.load()
    p = (ctypes.addressof(ctypes.create_string_buffer(64)) + 15) & ~15
    two = (ctypes.c_void_p * 2)(p, p)
    one = (ctypes.c_void_p * 2)(p, None)
    odd = (ctypes.c_void_p * 2)(p, p + 2)
    ws = lib.axon_router_balance_workspace_bytes(6, 1, 2, 8)
    assert ws > 0 and lib.axon_router_balance_workspace_bytes(6, 1, 0, 8) < 0

    def fwd(x=two, dtype=0, ld=8, layers=2, n=6, e=8, k=2, ids=None, mask=None, kind=0, cu=None, s=1, score=0, loss=p, coef=p,
            scale=p, counts=p, w=p, wb=ws):
        return lib.axon_router_balance_fwd(x, dtype, ld, layers, n, e, k, ids, 1, mask, kind, cu, s, score, loss, coef, scale,
                                           counts, w, wb, None)

    for bad in (dict(x=None), dict(x=one), dict(x=odd), dict(dtype=2), dict(ld=7), dict(layers=0), dict(n=-1), dict(e=0), dict(ids=one),
                dict(mask=p, kind=5), dict(s=2), dict(s=-1), dict(score=2), dict(loss=None), dict(coef=None), dict(scale=None),
                dict(counts=None), dict(w=None), dict(w=p + 4)):
        assert fwd(**bad) == -1, bad
    for bad in (dict(k=0), dict(k=9), dict(e=1025, ld=1025), dict(n=1 << 30), dict(cu=p, s=1 << 24)):
        assert fwd(**bad) == -2, bad
    assert fwd(wb=ws - 1) == -3

    def bwd(x=two, coef=p, scale=p, g=p, d=two, n=6):
        return lib.axon_router_balance_bwd(x, 0, 8, 2, n, 8, None, 0, None, 1, 0, coef, scale, g, d, None)

    assert bwd(n=0) == 0
    for bad in (dict(x=None), dict(x=one), dict(coef=None), dict(scale=None), dict(g=None), dict(d=None), dict(d=odd)):
        assert bwd(**bad) == -1, bad


@pytest.mark.parametrize("per_sequence", [False, True])
def test_a_loss_term_without_layers_or_tokens(per_sequence):
    """The operator's own errors, also where there is no layer or token to ask for its size."""
    from axon_amd.models.fsdp_models import _router_term

    args = {"router_top_k": 2, "router_balance_per_sequence": per_sequence}
    with pytest.raises(ValueError, match="no layers"):
        _router_term({}, None, torch.zeros(2, 3), args, [], None)
    for router in (torch.zeros(0, 4), (torch.zeros(0, 4),), torch.zeros(3, 0, 4)):
        with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
            _router_term({}, None, torch.zeros(2, 0), args, router, None)


def test_an_attention_mask_of_one_dimension_is_one_row():
    """Beside packed routers too: the operator itself refuses what is not on a GPU."""
    from axon_amd.models.fsdp_models import _router_term

    for router in (torch.zeros(4, 8), torch.zeros(6, 8)):
        with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
            _router_term({"attention_mask": torch.ones(6, dtype=I64)}, None, torch.zeros(1, 6), {"router_top_k": 2}, router, None)
