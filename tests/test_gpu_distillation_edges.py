"""Distillation where teacher or student have next to nothing left, against its definition in 64 bits, by logarithms throughout."""

import math

import pytest
import torch

from axon_amd.utils.torch.distillation import distillation_from_logits, distillation_loss_from_logits

pytestmark = pytest.mark.gpu

# As derived beside the tests of ordinary rows: a sum of exponentials, its logarithm absolutely, and every probability.
P_REL = 4e-5


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def reference(z, ids, lq, divergence, tail, temperature=1.0, beta=0.5, q_rest=None):
    """(losses, gradient of their sum, size of the losses' terms, size of the gradient's) of ids that differ."""
    z, ids, lq = z.detach().double().cpu(), ids.cpu().long(), lq.double().cpu()
    n, v = z.shape
    ok = (ids >= 0) & (ids < v)
    at = torch.where(ok, ids, torch.zeros_like(ids))
    log_p = torch.log_softmax(z / temperature, 1)
    given = torch.zeros(n, v, dtype=torch.int64).scatter_add_(1, at, ok.long()) > 0
    lq = torch.where(ok, lq, -math.inf)
    lp = torch.where(ok, log_p.gather(1, at), -math.inf)
    left = torch.where(given, -math.inf, log_p)
    if tail == "rest":
        lp_rest = torch.logsumexp(left, 1, keepdim=True)
        q_rest = (1.0 - lq.exp().sum(1)).clamp(min=0.0) if q_rest is None else q_rest
        lq, lp = torch.cat([lq, q_rest.log()[:, None]], 1), torch.cat([lp, lp_rest], 1)
    q, p = lq.exp(), lp.exp()
    zero = torch.zeros_like(p)
    if divergence == "forward":
        terms, G = torch.where(q > 0, q * (lq - lp), zero), -q
        size, gsize = torch.where(q > 0, q * (lq.abs() + lp.abs() + 1), zero), q
    elif divergence == "reverse":
        terms = torch.where(p > 0, p * (lp - lq), zero)
        G = torch.where(p > 0, terms + p, zero)
        size = torch.where(p > 0, p * (lq.abs() + lp.abs() + 1), zero)
        gsize = size
    else:
        lm = (beta * q + (1 - beta) * p).log()
        mine = torch.where(p > 0, (1 - beta) * p * (lp - lm), zero)
        terms, G = torch.where(q > 0, beta * q * (lq - lm), zero) + mine, mine
        gsize = torch.where(p > 0, p * (lp.abs() + lm.abs() + 1), zero)
        size = torch.where(q > 0, q * (lq.abs() + lm.abs() + 1), zero) + gsize
    p_all, k = log_p.exp(), ids.shape[1]
    total, total_size = G.sum(1, keepdim=True), gsize.sum(1, keepdim=True)
    d = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, at, torch.where(ok, G[:, :k], 0.0)) - p_all * total
    dsize = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, at, torch.where(ok, gsize[:, :k], 0.0)) + p_all * total_size
    if tail == "rest":
        # by differences of the logits: beside the type's lowest value 64 bits have no room for the logarithm of a sum
        share = torch.where(lp_rest > -math.inf, torch.softmax(torch.where(given, -math.inf, z / temperature), 1), 0.0)
        d, dsize = d + share * G[:, -1:], dsize + share * gsize[:, -1:]
    return terms.sum(1), d / temperature, size.sum(1), dsize / temperature


def agrees(z, ids, lq, ref, dtype, **how):
    """Both entry points, losses and gradients."""
    losses, grad, size, gsize = ref
    loss_bound = 2 * P_REL * size + 1e-12
    grad_bound = 4 * P_REL * gsize + (2.0 ** -8 * grad.abs() if dtype == torch.bfloat16 else 0.0) + 1e-30
    x = z.clone().requires_grad_(True)
    got, _ = distillation_from_logits(x, ids, lq, **how)
    r = distillation_loss_from_logits(x, ids, lq, torch.ones(len(z), device="cuda"), **how)
    for values, total in ((got, got.sum()), (r.losses, r.loss)):
        assert ((values.detach().double().cpu() - losses).abs() <= loss_bound).all(), how
        d, = torch.autograd.grad(total, x)
        assert ((d.double().cpu() - grad).abs() <= grad_bound).all(), how
    again, = torch.autograd.grad(distillation_loss_from_logits(x, ids, lq, torch.full((len(z),), 0.5, device="cuda"), **how).loss, x,
                                 torch.tensor(2.0, device="cuda"))  # formed anew
    assert ((again.double().cpu() - grad).abs() <= grad_bound).all(), how


@pytest.mark.parametrize("gap", [60.0, 80.0, 95.0, 110.0, 400.0, 720.0, 800.0, 1e5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("many,v", [(1, 5000), (120, 5001), (1, 70000)])
def test_next_to_nothing_left(gap, dtype, many, v):
    """The student has e^-gap left, the teacher a fifth: every token that is not given gets its part of it, -inf gets nothing."""
    n = 4 * many
    z = torch.randn(n, v, generator=gen(v), device="cuda") - gap
    z[::4, 10:] = -math.inf  # a grammar's row: five are left beside the given ones
    z[1::4, torch.rand(v, generator=gen(1), device="cuda") < 0.5] = -math.inf
    ids = torch.tensor([[0, 1, v // 2, v - 1, 4]], device="cuda").repeat(n, 1)
    z.scatter_(1, ids, torch.randn(n, 5, generator=gen(2), device="cuda"))
    z = z.to(dtype)
    lq = torch.log_softmax(torch.randn(n, 5, generator=gen(3), device="cuda"), 1) + math.log(0.8)
    for divergence in ("forward", "reverse", "jsd"):
        agrees(z, ids, lq, reference(z, ids, lq, divergence, "rest"), dtype, divergence=divergence)
    temperature = 0.4
    ref = reference(z, ids, lq, "forward", "rest", temperature)
    agrees(z, ids, lq, ref, dtype, temperature=temperature)


@pytest.mark.parametrize("lowest", [True, False])
def test_what_is_left_at_the_types_lowest(lowest):
    """Tokens that a mask has set to the type's lowest value, or all but one of them to -inf: gradients stay numbers."""
    n, v = 6, 3000
    for dtype in (torch.float32, torch.bfloat16):
        z = torch.full((n, v), torch.finfo(dtype).min if lowest else -math.inf, device="cuda", dtype=dtype)
        if not lowest:
            z[:, 77] = -200.0
        z[:, :4] = torch.randn(n, 4, generator=gen(1), device="cuda").to(dtype)
        ids = torch.arange(4, device="cuda").repeat(n, 1)
        lq = torch.full((n, 4), math.log(0.2), device="cuda")
        for divergence in ("forward", "reverse", "jsd"):
            agrees(z, ids, lq, reference(z, ids, lq, divergence, "rest"), dtype, divergence=divergence)


def error_of(lq, step=0.0):
    """How well 1 - sum q is known."""
    lq = lq.double().cpu()
    return torch.where(lq > -math.inf, lq.exp() * (2.0 ** -21 * (1 + lq.abs()) + step * lq.abs()), 0.0).sum(1)


def stored(z, how):
    """(log-probabilities of all of z's tokens, how far two half steps of their type are apart) as programs compute and store them."""
    lq = z - torch.logsumexp(z, 1, keepdim=True) if how == "difference" else torch.log_softmax(z, 1)
    return {"bf16": (lq.bfloat16(), 2.0 ** -7), "fp16": (lq.half(), 2.0 ** -10), "fp64": (lq.double(), 0.0)}.get(how, (lq, 0.0))


@pytest.mark.parametrize("how", ["fp32", "difference", "bf16", "fp16", "fp64"])
@pytest.mark.parametrize("v,legal,scale", [(10, 10, 1.0), (3000, 10, 3.0), (3000, 2, 8.0), (40001, 300, 3.0)])
@pytest.mark.parametrize("out", [-math.inf, "lowest"])
def test_lists_of_all_tokens_that_there_are(how, v, legal, scale, out):
    """A grammar leaves ``legal`` tokens, the teacher gives all of them, with fillers and impossible ones beside them: what 1 - sum q has
    by rounding is no outcome."""
    n, extra = 300, 3
    allowed = torch.rand(n, v, generator=gen(1), device="cuda").topk(legal, 1).indices
    student = torch.randn(n, legal, generator=gen(2), device="cuda") * scale
    z = torch.full((n, v), torch.finfo(torch.float32).min if out == "lowest" else out, device="cuda").scatter_(1, allowed, student)
    lq, step = stored(torch.randn(n, legal, generator=gen(3), device="cuda") * scale + 15.0, how)
    ids = torch.cat([allowed, torch.tensor([[-1, v + 5, -1]], device="cuda").expand(n, extra)], 1)
    lq = torch.cat([lq, torch.tensor([[-2.0, -math.inf, 0.0]], device="cuda", dtype=lq.dtype).expand(n, extra)], 1)
    left = 1.0 - lq[:, :legal].double().exp().sum(1).cpu()
    assert (left > 0).any() and (left <= 8 * error_of(lq[:, :legal], step)).all()
    ref = reference(z, ids, lq, "forward", "rest", q_rest=torch.zeros(n, dtype=torch.float64))
    assert torch.isfinite(ref[0]).all() and torch.isfinite(ref[1]).all()
    agrees(z, ids, lq, ref, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sure", [17.0, 18.1, 25.0, 60.0])
def test_teachers_that_are_sure(dtype, sure):
    """log p of a sure teacher is rounded to 0, or its list adds up to more than 1: it has at least the rounding left."""
    n, v = 60, 2500
    teacher = torch.randn(n, v, generator=gen(1), device="cuda") * 0.1
    teacher[:, 3] += sure + math.log(v)
    lq = torch.log_softmax(teacher, 1)[:, 3:6]
    ids = torch.arange(3, 6, device="cuda").repeat(n, 1)
    left = 1.0 - lq.double().exp().sum(1).cpu()
    e = error_of(lq)
    assert sure < 25 or (left <= 0).any()
    z = (torch.randn(n, v, generator=gen(2), device="cuda") * 2).to(dtype)
    agrees(z, ids, lq, reference(z, ids, lq, "reverse", "rest", q_rest=torch.maximum(left, e)), dtype, divergence="reverse")
    agrees(z, ids, lq, reference(z, ids, lq, "jsd", "rest"), dtype, divergence="jsd")
    agrees(z, ids, lq, reference(z, ids, lq, "forward", "rest"), dtype)


def test_what_a_teacher_has_left_in_earnest():
    """More than a rounding, where the student has none: the forward divergence is infinite, as it is for a given token."""
    n, v = 4, 900
    z = torch.full((n, v), -math.inf, device="cuda")
    z[:, :5] = torch.randn(n, 5, generator=gen(1), device="cuda")
    ids = torch.arange(5, device="cuda").repeat(n, 1)
    lq = torch.log_softmax(torch.randn(n, 5, generator=gen(2), device="cuda"), 1) - 1e-4
    losses, _ = distillation_from_logits(z, ids, lq)
    assert (losses == math.inf).all()
    reverse, _ = distillation_from_logits(z, ids, lq, divergence="reverse")
    assert torch.isfinite(reverse).all()


@pytest.mark.parametrize("v", [700, 70000])
@pytest.mark.parametrize("tail", ["renormalize", "drop"])
def test_a_teacher_that_rules_out_all_that_is_given(tail, v):
    """q = 0 for each of them: nothing of a forward divergence, p log(p / m) of the third, and against 0 an infinite reverse one."""
    n, k = 8, 5
    z = torch.randn(n, v, generator=gen(v), device="cuda")
    ids = torch.randperm(v, generator=gen(1), device="cuda")[:k].repeat(n, 1)
    lq = torch.log_softmax(torch.randn(n, k, generator=gen(2), device="cuda"), 1)
    lq[::2] = -math.inf
    ids[4, 1:] = -1
    sums = torch.logsumexp(lq.double(), 1, keepdim=True) if tail == "renormalize" else torch.zeros(n, 1, device="cuda")
    ref_lq = torch.where(lq > -math.inf, lq.double() - sums, -math.inf)
    for divergence in ("forward", "jsd"):
        ref = reference(z, ids, ref_lq, divergence, "drop")
        assert torch.isfinite(ref[0]).all() and (divergence == "jsd" or (ref[0][::2] == 0).all() and (ref[1][::2] == 0).all())
        agrees(z, ids, lq, ref, torch.float32, divergence=divergence, tail=tail)
    losses, _ = distillation_from_logits(z, ids, lq, divergence="reverse", tail=tail)
    assert (losses[::2] == math.inf).all() and torch.isfinite(losses[1::2]).all()


@pytest.mark.parametrize("temperature", [1e-37, 1e-20, 1e20, 1e30, 1e37, 2e38])
@pytest.mark.parametrize("v,n", [(900, 3), (70001, 2), (600, 2000)])
def test_temperatures_at_both_ends_of_the_range(temperature, v, n):
    """Logits of the temperature's size, and logits that are all alike beside it."""
    k = 6
    ids = torch.stack([torch.randperm(v, generator=gen(i), device="cuda")[:k] for i in range(min(n, 5))]).repeat(-(-n // 5), 1)[:n]
    lq = torch.log_softmax(torch.randn(n, k + 1, generator=gen(1), device="cuda"), 1)[:, :k]
    w = torch.rand(n, generator=gen(2), device="cuda") + 0.5
    for scale in (min(temperature, 1e37), 1.0) if temperature > 1 else (temperature,):
        z = torch.randn(n, v, generator=gen(3), device="cuda") * scale
        for divergence, tail in (("forward", "rest"), ("jsd", "drop"), ("reverse", "renormalize")):
            ref_lq = lq.double() - (torch.logsumexp(lq.double(), 1, keepdim=True) if tail == "renormalize" else 0.0)
            losses, grad, size, gsize = reference(z, ids, ref_lq, divergence, "rest" if tail == "rest" else "drop", temperature)
            x = z.clone().requires_grad_(True)
            how = dict(divergence=divergence, tail=tail, temperature=temperature)
            got, _ = distillation_from_logits(x, ids, lq, **how)
            r = distillation_loss_from_logits(x, ids, lq, w, **how)
            for values in (got, r.losses):
                assert ((values.detach().double().cpu() - losses).abs() <= 2 * P_REL * size + 1e-12).all(), how
            each, = torch.autograd.grad(got, x, w)
            once, = torch.autograd.grad(r.loss, x)
            up = w.double().cpu()[:, None]
            # a gradient and 1 / T may be numbers that 32 bits hold in steps of 2^-149
            bound = 4 * P_REL * gsize * up + 2.0 ** -149 * (4 + 4 * temperature * gsize)
            for d in (each, once):
                assert ((d.double().cpu() - up * grad).abs() <= bound).all(), (how, scale)


def test_rows_that_are_read_and_rows_that_are_not():
    """Per position: rows without an upstream gradient get exactly 0 whatever they hold; with one, a row of the type's lowest logits and
    one that gives a given token no probability have the gradient of their definition, though the latter's loss is infinite."""
    v, n, k = 3000, 7, 5
    z = torch.randn(n, v, generator=gen(1), device="cuda") * 3
    ids = torch.stack([torch.randperm(v, generator=gen(i), device="cuda")[:k] for i in range(n)])
    lq = torch.log_softmax(torch.randn(n, k + 1, generator=gen(2), device="cuda"), 1)[:, :k]
    z[0, 77] = math.nan
    z[1] = -math.inf
    z[2, 5] = math.inf
    z[3, ids[3, 2]] = -math.inf
    z[4] = torch.finfo(torch.float32).min
    for divergence in ("forward", "reverse", "jsd"):
        for tail in ("rest", "drop", "renormalize"):
            x = z.clone().requires_grad_(True)
            out, _ = distillation_from_logits(x, ids, lq, divergence=divergence, tail=tail)
            for i in (5, 4, 3):
                up = torch.zeros(n, device="cuda")
                up[i] = 1.0
                d, = torch.autograd.grad(out, x, up, retain_graph=True)
                rest = torch.arange(n) != i
                assert (d[rest.cuda()] == 0).all(), (divergence, tail, i)
                ref_lq = lq.double() - (torch.logsumexp(lq.double(), 1, keepdim=True) if tail == "renormalize" else 0.0)
                _, grad, _, gsize = reference(z[i:i + 1], ids[i:i + 1], ref_lq[i:i + 1], divergence, "rest" if tail == "rest" else "drop")
                assert ((d[i].double().cpu() - grad[0]).abs() <= 4 * P_REL * gsize[0] + 1e-30).all(), (divergence, tail, i)
                w = torch.zeros(n, device="cuda")
                w[i] = 1.0
                r = distillation_loss_from_logits(x, ids, lq, w, divergence=divergence, tail=tail)
                once, = torch.autograd.grad(r.loss, x)
                assert (once[rest.cuda()] == 0).all() and (r.losses[rest.cuda()] == 0).all()
                assert ((once[i].double().cpu() - grad[0]).abs() <= 4 * P_REL * gsize[0] + 1e-30).all(), (divergence, tail, i)
