"""What distillation's entry points refuse, on the host: nothing is launched."""

import ctypes

import pytest
import torch

from axon_amd import _lib
from axon_amd.utils.torch.distillation import distillation_from_logits, distillation_loss_from_logits

Z = torch.zeros(4, 50)
IDS = torch.zeros(4, 3, dtype=torch.int64)
LQ = torch.zeros(4, 3)
W = torch.ones(4)


def both(z=Z, ids=IDS, lq=LQ, w=W, **how):
    return [lambda: distillation_from_logits(z, ids, lq, **how), lambda: distillation_loss_from_logits(z, ids, lq, w, **how)]


@pytest.mark.parametrize("kw", [
    dict(divergence="kl"), dict(tail="bucket"), dict(divergence="jsd", beta=0.0), dict(divergence="jsd", beta=1.0),
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
    dict(z=Z.half()), dict(z=Z.double()), dict(z=Z.long()), dict(ids=IDS.float()), dict(ids=IDS.to(torch.int16)), dict(ids=IDS[:3]),
    dict(ids=IDS[:, 0]), dict(ids=IDS[:, :2]), dict(ids=IDS[:, :0], lq=LQ[:, :0]),
    dict(ids=torch.zeros(4, 513, dtype=torch.int64), lq=torch.zeros(4, 513)), dict(lq=LQ.long()), dict(lq=LQ[:, :2]),
    dict(lq=LQ.clone().requires_grad_(True)),
])
def test_operands_that_do_not_fit_are_refused(kw):
    for call in both(**kw):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("w", [torch.ones(3), torch.ones(4, 1), torch.ones(4, requires_grad=True)])
def test_weights_that_do_not_fit_are_refused(w):
    with pytest.raises(ValueError):
        distillation_loss_from_logits(Z, IDS, LQ, w)
    with pytest.raises(TypeError):
        distillation_loss_from_logits(Z, IDS, LQ, None)


def test_tensors_that_are_not_on_a_gpu_are_refused():
    for call in both():
        with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
            call()


def test_the_c_entry_points_check_their_arguments():
    lib = _lib.load()
    p = ctypes.addressof(ctypes.create_string_buffer(64)) & ~15  # any address: nothing is read
    ws = lib.axon_distill_workspace_bytes(0, 2, 100)
    assert ws > 0 and lib.axon_distill_workspace_bytes(0, -1, 100) < 0 and lib.axon_distill_workspace_bytes(5, 2, 100) < 0

    def fwd(z=p, dtype=0, ld=100, n=2, v=100, ids=p, lq=p, k=3, div=0, tail=1, beta=0.5, t=1.0, losses=p, cov=p, grads=p, coef=p, w=p, wb=ws):
        return lib.axon_distill_fwd(z, dtype, ld, n, v, ids, 1, lq, k, None, div, tail, beta, t, losses, cov, grads, coef, w, wb, 0, None)

    assert fwd(n=0) == 0
    for bad in (dict(z=None), dict(z=p + 2), dict(dtype=2), dict(ld=99), dict(n=-1), dict(v=0), dict(ids=None), dict(lq=None), dict(div=3),
                dict(tail=-1), dict(div=2, beta=1.0), dict(t=0.0), dict(t=float("nan")), dict(losses=None), dict(cov=None), dict(grads=None),
                dict(coef=None)):
        assert fwd(**bad) == -1, bad
    for bad in (dict(k=0), dict(k=513), dict(n=1 << 24), dict(v=3145729, ld=3145729)):
        assert fwd(**bad) == -2, bad
    assert fwd(w=None) == fwd(wb=ws - 1) == fwd(w=p + 8) == -3

    def bwd(ids=p, k=3, weights=None, t=1.0, grads=p, coef=p, up=p, ready=0, d=p, ld_d=100, n=2):
        return lib.axon_distill_bwd(p, 0, 100, n, 100, ids, 1, k, weights, t, grads, coef, up, ready, d, ld_d, None)

    assert bwd(n=0) == 0
    for bad in (dict(ids=None), dict(grads=None), dict(coef=None), dict(up=None), dict(d=None), dict(ld_d=99), dict(t=0.0), dict(ready=1),
                dict(ready=1, weights=p, up=None), dict(d=p + 1)):
        assert bwd(**bad) == -1, bad
    assert bwd(k=0) == bwd(k=513) == -2

    def loss(out=p, weights=p, d=None):
        return lib.axon_distill_loss(p, 0, 100, 2, 100, p, 1, p, 3, weights, 0, 1, 0.5, 1.0, out, p, p, p, p, d, 100, p, ws - 1, None)

    assert loss(out=None) == loss(weights=None) == loss(d=p + 1) == -1 and loss() == -3
