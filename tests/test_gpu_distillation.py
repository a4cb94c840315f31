"""Distillation from a teacher's top logits, against its definition in 64 bits."""

import math

import pytest
import torch

from axon_amd.utils.torch.controls import LogitControls, controlled_logits
from axon_amd.utils.torch.distillation import distillation_from_logits, distillation_loss_from_logits
from axon_amd.utils.torch.ops import top_logprobs_from_logits

import controls_reference as R

pytestmark = pytest.mark.gpu

# Off by, relative: an exponential's argument of up to 100 in 2^-24 twice (the factor log2(e) / T, the product: 1.2e-5, weighted
# by the term's probability), 2^-22 for itself, and sums in chains of at most 300 roundings of 2^-24 (1.8e-5).  So is a sum of
# exponentials, its logarithm absolutely, and every probability.
P_REL = 4e-5
LP_TOL = P_REL


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def batch(seed, n, v, k, dtype, *, ids=torch.int64, fillers=0.1, repeats=True, peaked=False):
    g = gen(seed)
    z = torch.randn(n, v, generator=g, device="cuda") * 3
    if peaked:
        z[:, v // 2] += 40.0
    z = z.to(dtype)
    # a teacher near the student, whose probabilities of the given tokens add up to less than 1
    t = torch.log_softmax(z.float() + torch.randn(n, v, generator=g, device="cuda"), 1)
    at = t.topk(min(k, v), 1).indices
    if k > v:
        at = torch.cat([at, torch.randint(0, v, (n, k - v), generator=g, device="cuda")], 1)
    lq = t.gather(1, at)
    at = torch.where(torch.rand(n, k, generator=g, device="cuda") < fillers, torch.randint(-2, 1, (n, k), generator=g, device="cuda") * v - 1, at)
    at[at == -1] = v  # fillers on either side of the vocabulary
    if repeats and k > 2:
        at[:, -1] = at[:, 0]
        lq[:, -1], lq[:, 0] = lq[:, 0] - 0.7, lq[:, 0] - 0.7
    if k > 3:
        lq[0, 1] = -math.inf  # the teacher has never seen it
    return z, at.to(ids), lq


def reference(z, ids, lq, divergence, tail, beta, temperature, up=None):
    """(losses, covered, gradient of sum up * losses, size of its terms, size of the losses' terms)."""
    z = z.detach().double().cpu()
    ids, lq = ids.cpu().long(), lq.double().cpu()
    n, v = z.shape
    ok = (ids >= 0) & (ids < v)
    at = torch.where(ok, ids, torch.zeros_like(ids))
    log_p = torch.log_softmax(z / temperature, 1)
    p_all = log_p.exp()
    lp = log_p.gather(1, at)
    lq = torch.where(ok, lq, torch.full_like(lq, -math.inf))
    if tail == "renormalize":
        total = torch.logsumexp(lq, 1, keepdim=True)
        lq = torch.where(ok, lq - total, lq)
    given = torch.zeros(n, v, dtype=torch.int64).scatter_add_(1, at, ok.long()) > 0
    p_rest = torch.where(given, 0.0, p_all).sum(1)
    if tail == "rest":
        q_rest = (1.0 - lq.exp().sum(1)).clamp(min=0.0)
        lq = torch.cat([lq, q_rest.log()[:, None]], 1)
        lp = torch.cat([lp, p_rest.log()[:, None]], 1)
        ok = torch.cat([ok, torch.ones(n, 1, dtype=torch.bool)], 1)
    q, p = lq.exp(), torch.where(ok, lp.exp(), 0.0)
    zero = torch.zeros_like(p)
    if divergence == "forward":
        terms, G = torch.where(q > 0, q * (lq - lp), zero), -q
        size, gsize = torch.where(q > 0, q * (lq.abs() + lp.abs() + 1), zero), q
    elif divergence == "reverse":
        terms = torch.where(p > 0, p * (lp - lq), zero)
        G = terms + p
        size = torch.where(p > 0, p * (lq.abs() + lp.abs() + 1), zero)
        gsize = size + p
    else:
        lm = (beta * q + (1 - beta) * p).log()
        mine = torch.where(p > 0, (1 - beta) * p * (lp - lm), zero)
        terms, G = torch.where(q > 0, beta * q * (lq - lm), zero) + mine, mine
        gsize = torch.where(p > 0, p * (lp.abs() + lm.abs() + 1), zero)
        size = torch.where(q > 0, q * (lq.abs() + lm.abs() + 1), zero) + gsize
    losses, covered = terms.sum(1), p[:, : ids.shape[1]].sum(1)
    up = torch.ones(n, dtype=torch.float64) if up is None else up.double().cpu()
    G_given = G[:, : ids.shape[1]]
    hit = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, at, torch.where(ok[:, : ids.shape[1]], G_given, 0.0))
    hit_size = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, at, torch.where(ok[:, : ids.shape[1]], gsize[:, : ids.shape[1]], 0.0))
    total, total_size = G.sum(1, keepdim=True), gsize.sum(1, keepdim=True)
    d, dsize = hit - p_all * total, hit_size + p_all * total_size
    if tail == "rest":
        share = torch.where(given, 0.0, p_all) / torch.where(p_rest > 0, p_rest, 1.0)[:, None]
        d = d + share * G[:, -1:]
        dsize = dsize + share * gsize[:, -1:]
    scale = (up / temperature)[:, None]
    return losses, covered, d * scale, dsize * scale.abs(), size.sum(1)


def check(got, want, bound):
    off = (got.detach().double().cpu() - want).abs() / bound
    assert off.max().item() <= 1.0, off.max().item()


# k-term sums are in 64 bits: only the probabilities and the last rounding count.  A loss term q |lq - lp| moves by q LP_TOL, p |..| by
# p P_REL (|..| + 1): both within P_REL of `size`; its gradients likewise, with the probability that multiplies them: twice that.
def loss_bound(size):
    return 2 * P_REL * size + 1e-12


def grad_bound(want, size, dtype):
    return 4 * P_REL * size + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0.0) + 1e-30


CASES = [
    # n, vocab, k, dtype, divergence, tail, beta, temperature, options
    (1, 1, 1, torch.float32, "forward", "rest", 0.5, 1.0, dict(fillers=0.0)),
    (3, 2, 5, torch.bfloat16, "reverse", "drop", 0.5, 1.0, dict()),
    (5, 7, 3, torch.float32, "jsd", "rest", 0.3, 2.0, dict()),
    (4, 33, 16, torch.bfloat16, "forward", "rest", 0.5, 1.0, dict(ids=torch.int32)),
    (6, 1000, 128, torch.float32, "reverse", "rest", 0.5, 0.7, dict(repeats=False)),
    (70, 1003, 40, torch.bfloat16, "jsd", "renormalize", 0.9, 1.0, dict()),
    (9, 4099, 512, torch.float32, "forward", "rest", 0.5, 1.0, dict()),
    (9, 4099, 300, torch.bfloat16, "reverse", "rest", 0.5, 1.0, dict(repeats=False)),
    (600, 2051, 8, torch.bfloat16, "forward", "rest", 0.5, 1.0, dict()),
    (1700, 515, 20, torch.float32, "jsd", "rest", 0.5, 1.0, dict(repeats=False)),
    (3, 50257, 64, torch.bfloat16, "forward", "renormalize", 0.5, 1.0, dict(ids=torch.int32)),
    (300, 50257, 20, torch.bfloat16, "forward", "rest", 0.5, 1.0, dict()),
    (260, 40000, 9, torch.float32, "reverse", "drop", 0.5, 1.0, dict()),
    (2, 151936, 64, torch.float32, "forward", "rest", 0.5, 1.0, dict()),
    (258, 151936, 20, torch.bfloat16, "jsd", "rest", 0.5, 1.5, dict(repeats=False)),
    (5, 201088, 20, torch.bfloat16, "reverse", "rest", 0.5, 1.0, dict(repeats=False)),
    (5, 3001, 4, torch.float32, "forward", "drop", 0.5, 1.0, dict(fillers=1.0, repeats=False)),
    (5, 3001, 4, torch.float32, "reverse", "rest", 0.5, 1.0, dict(fillers=1.0, repeats=False)),
    (12, 9000, 5, torch.float32, "forward", "rest", 0.5, 1.0, dict(peaked=True)),
    (12, 9000, 5, torch.bfloat16, "jsd", "rest", 0.5, 1.0, dict(peaked=True)),
]


@pytest.mark.parametrize("n,v,k,dtype,divergence,tail,beta,temperature,options", CASES)
def test_losses_of_positions(n, v, k, dtype, divergence, tail, beta, temperature, options):
    z, ids, lq = batch(n + v, n, v, k, dtype, **options)
    if divergence == "reverse":
        lq = lq.clamp(min=-60.0)  # what the teacher rules out has an infinite reverse divergence
    how = dict(divergence=divergence, tail=tail, beta=beta, temperature=temperature)
    up = torch.randn(n, generator=gen(7), device="cuda")
    losses, covered, grad, gsize, size = reference(z, ids, lq, divergence, tail, beta, temperature, up)
    z.requires_grad_(True)
    got, cov = distillation_from_logits(z, ids, lq, **how)
    assert got.dtype == cov.dtype == torch.float32 and got.shape == cov.shape == (n,) and not cov.requires_grad
    check(got, losses, loss_bound(size))
    check(cov, covered, 2 * P_REL * covered + 1e-30)
    d, = torch.autograd.grad(got, z, up)
    assert d.dtype == dtype
    check(d, grad, grad_bound(grad, gsize, dtype))
    twin = z.detach().clone().requires_grad_(True)
    over, _ = distillation_from_logits(twin * 1.0, ids, lq, inplace_backward=True, **how)
    assert torch.equal(torch.autograd.grad(over, twin, up)[0], d) and torch.equal(over, got)


@pytest.mark.parametrize("n,v,k,dtype,divergence,tail,beta,temperature,options", CASES)
@pytest.mark.parametrize("masked", [0.0, 0.5])
def test_weighted_sum_of_losses(n, v, k, dtype, divergence, tail, beta, temperature, options, masked):
    z, ids, lq = batch(n + v, n, v, k, dtype, **options)
    if divergence == "reverse":
        lq = lq.clamp(min=-60.0)
    how = dict(divergence=divergence, tail=tail, beta=beta, temperature=temperature)
    w = torch.randn(n, generator=gen(8), device="cuda")
    w[torch.rand(n, generator=gen(9), device="cuda") < masked] = 0.0
    on = w.cpu() != 0
    losses, covered, grad, gsize, size = reference(z, ids, lq, divergence, tail, beta, temperature, w)
    if masked:
        z[w == 0] = math.nan  # positions of weight 0 are not looked at
    z.requires_grad_(True)
    r = distillation_loss_from_logits(z, ids, lq, w, **how)
    assert not r.losses.requires_grad and not r.covered.requires_grad and r.loss.shape == ()
    check(r.losses[on.cuda()], losses[on], loss_bound(size[on]))
    assert (r.losses.cpu()[~on] == 0).all() and (r.covered.cpu()[~on] == 0).all()
    wd = w.double().cpu()
    check(r.loss[None], (wd * losses)[on].sum()[None], (wd.abs() * loss_bound(size))[on].sum()[None] + 2.0 ** -24 * (wd * losses)[on].sum().abs() + 1e-30)
    grad[~on], gsize[~on] = 0.0, 0.0
    d, = torch.autograd.grad(r.loss, z, retain_graph=True)
    check(d, grad, grad_bound(grad, gsize, dtype))
    d.fill_(5.0)  # what the caller does to a gradient does not come back
    again, = torch.autograd.grad(r.loss, z, retain_graph=True)
    check(again, grad, grad_bound(grad, gsize, dtype))
    twice, = torch.autograd.grad(r.loss, z, torch.tensor(-2.5, device="cuda"))
    check(twice, -2.5 * grad, grad_bound(2.5 * grad, 2.5 * gsize, dtype))
    with torch.no_grad():
        quiet = distillation_loss_from_logits(z, ids, lq, w, **how)
    assert torch.equal(quiet.loss, r.loss) or (quiet.loss - r.loss).abs() <= 2 * (wd.abs() * loss_bound(size))[on].sum()
    check(quiet.losses[on.cuda()], losses[on], loss_bound(size[on]))
    other = distillation_loss_from_logits(z, ids, lq, w, **how)  # an upstream gradient that is not 1 at the first backward
    half, = torch.autograd.grad(other.loss, z, torch.tensor(0.5, device="cuda"))
    check(half, 0.5 * grad, grad_bound(0.5 * grad, 0.5 * gsize, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("many", [1, 120])
def test_what_a_student_has_left_is_right_where_it_is_little(dtype, many):
    """All but 1e-13 of the student's probability on the given tokens: the rest is summed by itself."""
    v, n = 5000, 3 * many
    z = torch.full((n, v), -20.0, device="cuda", dtype=dtype)
    z[:, :4] = 18.0
    ids = torch.tensor([[0, 1, 2, 3]], device="cuda").repeat(n, 1)
    lq = torch.full((n, 4), math.log(0.2), device="cuda")
    w = torch.ones(n, device="cuda")
    for divergence in ("forward", "reverse", "jsd"):
        losses, _, grad, gsize, size = reference(z, ids, lq, divergence, "rest", 0.5, 1.0)
        x = z.clone().requires_grad_(True)
        got, _ = distillation_from_logits(x, ids, lq, divergence=divergence)
        check(got, losses, loss_bound(size))
        d, = torch.autograd.grad(got.sum(), x)
        check(d, grad, grad_bound(grad, gsize, dtype))
        r = distillation_loss_from_logits(x, ids, lq, w, divergence=divergence)
        check(r.losses, losses, loss_bound(size))
        check(torch.autograd.grad(r.loss, x)[0], grad, grad_bound(grad, gsize, dtype))


def test_rows_without_a_softmax_and_infinities():
    v = 3000
    z, ids, lq = batch(5, 6, v, 5, torch.float32, fillers=0.0, repeats=False)
    lq = lq.clamp(min=-30)
    clean, _ = distillation_from_logits(z, ids, lq)
    z[0, 77] = math.nan
    z[1] = -math.inf
    z[2, 5] = math.inf
    z[3, ids[3, 2]] = -math.inf  # the student rules out what the teacher has
    z[4] = torch.finfo(torch.float32).min  # all the same
    for tail in ("rest", "drop", "renormalize"):
        x = z.clone().requires_grad_(True)
        f, cov = distillation_from_logits(x, ids, lq, divergence="forward", tail=tail)
        assert torch.isnan(f[:3]).all() and f[3] == math.inf and torch.isfinite(f[4:]).all()
        assert abs(cov[4].item() - 5 / v) <= 5 / v * 1e-5
        r, _ = distillation_from_logits(x, ids, lq, divergence="reverse", tail=tail)
        j, _ = distillation_from_logits(x, ids, lq, divergence="jsd", tail=tail)
        assert torch.isnan(r[:3]).all() and torch.isfinite(r[3:]).all() and torch.isnan(j[:3]).all() and torch.isfinite(j[3:]).all()
        for out in (f, r, j):
            d, = torch.autograd.grad(out[5], x, retain_graph=True)
            assert (d[:5] == 0).logical_or(torch.isnan(d[:5])).all() and torch.isfinite(d[5]).all()
        w = torch.tensor([0.0, 0.0, 0.0, 0.0, 1.0, 1.0], device="cuda")
        s = distillation_loss_from_logits(x, ids, lq, w, tail=tail)
        assert torch.isfinite(s.loss) and (torch.autograd.grad(s.loss, x)[0][:4] == 0).all()
    assert torch.equal(distillation_from_logits(z, ids, lq)[0][5], clean[5])
    never = lq.clone()
    never[:, 1] = -math.inf  # the teacher rules out what the student has
    r, _ = distillation_from_logits(z, ids, never, divergence="reverse")
    assert r[5] == math.inf and torch.isfinite(distillation_from_logits(z, ids, never)[0][5])


def test_rows_that_lie_elsewhere():
    n, v, k = 37, 4003, 6
    z, ids, lq = batch(11, n, v, k, torch.bfloat16)
    up = torch.randn(n, generator=gen(1), device="cuda")
    x = z.requires_grad_(True)
    want, _ = distillation_from_logits(x, ids, lq)
    d_want, = torch.autograd.grad(want, x, up)
    wide = torch.full((n * 3, 2 * k), -1, device="cuda", dtype=ids.dtype)
    wide[::3, ::2] = ids
    lq_half = lq.double()
    for off in (1, 5):
        buf = torch.full((n * (v + 9) + off,), 99.0, device="cuda", dtype=z.dtype)
        view = buf[off:].view(n, v + 9)[:, :v]
        with torch.no_grad():
            view.copy_(z)
        view.requires_grad_(True)
        got, _ = distillation_from_logits(view, wide[::3, ::2], lq_half)
        d, = torch.autograd.grad(got, view, up)
        assert torch.allclose(got, want, rtol=0, atol=1e-4) and (d - d_want).abs().max() <= 2.0 ** -7 * d_want.abs().max()
        r = distillation_loss_from_logits(view, ids, lq, up)
        d, = torch.autograd.grad(r.loss, view)
        assert (d - d_want).abs().max() <= 2.0 ** -7 * d_want.abs().max()
    many = z.detach().view(1, n, v).requires_grad_(True)
    got, cov = distillation_from_logits(many, ids[None], lq[None])
    assert got.shape == cov.shape == (1, n) and torch.equal(got[0], want)
    none, cov = distillation_from_logits(z[:0], ids[:0], lq[:0])
    assert none.shape == (0,) and cov.shape == (0,)
    r = distillation_loss_from_logits(z[:0], ids[:0], lq[:0], up[:0])
    assert r.loss.item() == 0.0 and torch.autograd.grad(r.loss, z)[0].abs().sum() == 0


def test_gradients_against_differences():
    z, ids, lq = batch(21, 9, 400, 7, torch.float32, repeats=False)
    lq = lq.clamp(min=-30)
    for divergence in ("forward", "reverse", "jsd"):
        for tail in ("rest", "drop", "renormalize"):
            f = lambda x: distillation_from_logits(x, ids, lq, divergence=divergence, tail=tail, temperature=1.3)[0].double().sum()
            x = z.clone().requires_grad_(True)
            f(x).backward()
            g = x.grad
            step = 0.02 / g.norm()
            numeric = (f(z + step * g) - f(z - step * g)).item() / (2 * step.item())
            exact = g.double().square().sum().item()
            # third derivatives: step^2 of 10 |g|^3; nine losses of about 1, off by 1e-6 each
            assert abs(numeric - exact) <= 0.01 * exact + 9e-6 / step.item(), (divergence, tail)


def test_results_repeat_bit_for_bit():
    for n in (20, 700):
        z, ids, lq = batch(31, n, 20000, 30, torch.bfloat16)
        w = torch.rand(n, generator=gen(1), device="cuda")
        x = z.requires_grad_(True)
        runs = []
        for _ in range(3):
            r = distillation_loss_from_logits(x, ids, lq, w)
            losses, cov = distillation_from_logits(x, ids, lq)
            runs.append([*r, losses, cov, *torch.autograd.grad(r.loss, x), *torch.autograd.grad(losses, x, w)])
        assert all(torch.equal(a, b) for other in runs[1:] for a, b in zip(runs[0], other))


def test_offsets_beyond_32_bits():
    v, n = 151936, 15000  # 4.5 GB of bf16
    z = torch.zeros(n, v, device="cuda", dtype=torch.bfloat16)
    z[-4:] = torch.randn(4, v, generator=gen(1), device="cuda").bfloat16()
    ids = torch.randint(0, v, (n, 5), generator=gen(2), device="cuda")
    lq = torch.full((n, 5), -2.0, device="cuda")
    w = torch.rand(n, generator=gen(3), device="cuda")
    w[: n - 600] = 0.0
    x = z.requires_grad_(True)
    r = distillation_loss_from_logits(x, ids, lq, w)
    d, = torch.autograd.grad(r.loss, x)
    losses, _, grad, gsize, size = reference(z[-4:], ids[-4:], lq[-4:], "forward", "rest", 0.5, 1.0, w[-4:])
    check(r.losses[-4:], losses, loss_bound(size))
    check(d[-4:], grad, grad_bound(grad, gsize, torch.bfloat16))
    assert (d[: n - 600] == 0).all()


@pytest.mark.parametrize("n,v", [(20, 7001), (600, 9000)])
def test_another_stream_and_a_captured_graph(n, v):
    z, ids, lq = batch(41, n, v, 9, torch.bfloat16)
    w = torch.rand(n, generator=gen(1), device="cuda")
    want = distillation_loss_from_logits(z, ids, lq, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = distillation_loss_from_logits(z, ids, lq, w)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = z.clone().requires_grad_(True)
    scale = torch.ones((), device="cuda")

    def step():
        r = distillation_loss_from_logits(x, ids, lq, w)
        d, = torch.autograd.grad(r.loss, x, scale)
        losses, cov = distillation_from_logits(x, ids, lq, divergence="jsd")
        return [r.loss.detach(), r.losses, d, losses.detach(), cov, *torch.autograd.grad(losses, x, w)]

    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i, factor in enumerate((1.0, 3.0, 1.0, 0.5)):
        with torch.no_grad():
            x.copy_(torch.randn(n, v, generator=gen(50 + i), device="cuda"))
            scale.fill_(factor)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(replayed, step()))
        torch.cuda.synchronize()


def test_a_backward_captured_by_itself():
    """Its replays form the gradient anew: none of them stands behind a forward.  (What the node has saved has to live as long as the
    graph that reads it: retain_graph.)"""
    z, ids, lq = batch(61, 40, 6000, 9, torch.bfloat16)
    w = torch.rand(40, generator=gen(1), device="cuda")
    x = z.requires_grad_(True)
    stream = torch.cuda.Stream()
    one = torch.ones((), device="cuda")
    with torch.cuda.stream(stream):
        torch.cuda.synchronize()
        want, = torch.autograd.grad(distillation_loss_from_logits(x, ids, lq, w).loss, x, one)
        r = distillation_loss_from_logits(x, ids, lq, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            d, = torch.autograd.grad(r.loss, x, one, retain_graph=True)
        for _ in range(3):
            d.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert (d - want).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_saved_tensors_and_second_derivatives():
    z, ids, lq = batch(71, 12, 900, 5, torch.float32)
    w = torch.rand(12, generator=gen(1), device="cuda")
    for changed in ("logits", "weights", "ids"):
        y = (z * 1.0).requires_grad_(True) * 1.0
        at, ww = ids.clone(), w.clone()
        r = distillation_loss_from_logits(y, at, lq, ww)
        with torch.no_grad():
            {"logits": y, "weights": ww, "ids": at}[changed].add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            r.loss.backward()
    x = z.clone().requires_grad_(True)
    losses, _ = distillation_from_logits(x, ids, lq)
    d, = torch.autograd.grad(losses.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        d.sum().backward()
    r = distillation_loss_from_logits(x, ids, lq, w)
    r.loss.backward()
    with pytest.raises(RuntimeError):
        r.loss.backward()


def test_a_student_under_a_grammar_learns_from_a_teacher_under_it():
    """The teacher's alternatives and the student's logits under the same controls, and the loss's gradient through them."""
    n, v, k = 14, 2500, 6
    g = gen(81)
    keep = torch.rand(n, v, generator=g, device="cuda") < 0.2
    tokens = torch.randint(0, v, (n,), generator=g, device="cuda")
    kw = dict(token_ids=tokens, cu_seqlens=torch.tensor([0, 9, 14], dtype=torch.int32, device="cuda"), repetition_penalty=1.2,
              temperature=0.9, allowed=R.pack(keep))
    ctl = LogitControls(**kw)
    teacher = torch.randn(n, v, generator=g, device="cuda") * 3
    student = (torch.randn(n, v, generator=g, device="cuda") * 3).requires_grad_(True)
    with torch.no_grad():
        top = top_logprobs_from_logits(controlled_logits(teacher, ctl), k)
    w = torch.rand(n, generator=g, device="cuda")
    r = distillation_loss_from_logits(controlled_logits(student, ctl), top.top_ids, top.top_logprobs, w)
    d, = torch.autograd.grad(r.loss, student)
    spans = R.spans_of([9, 5], "all")
    out, slope, _ = R.controlled(student, spans, tokens, repetition=1.2, keep=list(keep), temperature=0.9)
    t_out, _, _ = R.controlled(teacher, spans, tokens, repetition=1.2, keep=list(keep), temperature=0.9)
    lq = torch.log_softmax(t_out, 1).gather(1, top.top_ids.cpu())
    losses, covered, grad, gsize, size = reference(out, top.top_ids, lq, "forward", "rest", 0.5, 1.0, w)
    # both sets of logits are off by seven roundings of at most 20 (8e-6), the teacher's log-probabilities by twice that
    check(r.losses, losses, loss_bound(size) + 4e-5 * size)
    check(d, grad * slope, (grad_bound(grad, gsize, torch.float32) + 8e-5 * gsize) * slope + 1e-30)
    assert (d[~keep] == 0).all()


@pytest.mark.parametrize("n,v,dtype,on_share", [
    (50000, 40, torch.float32, 0.5),     # more rows than the workgroups' lists hold at once
    (100001, 24, torch.bfloat16, 1.0),
    (100001, 24, torch.bfloat16, 0.01),
    (530, 34001, torch.bfloat16, 0.9),   # rows of 68 KB: more than there are workgroups
    (3, 500003, torch.bfloat16, 1.0),    # longer rows than are held
    (2, 250001, torch.float32, 1.0),
])
def test_weighted_rows_that_go_round(n, v, dtype, on_share):
    z, ids, lq = batch(n + v, n, v, 3, dtype)
    w = torch.rand(n, generator=gen(1), device="cuda") + 0.5
    w[torch.rand(n, generator=gen(2), device="cuda") >= on_share] = 0.0
    losses, covered, grad, gsize, size = reference(z, ids, lq, "forward", "rest", 0.5, 1.0, w)
    on = w.cpu() != 0
    z[w == 0] = math.nan
    z.requires_grad_(True)
    r = distillation_loss_from_logits(z, ids, lq, w)
    d, = torch.autograd.grad(r.loss, z)
    check(r.losses[on.cuda()], losses[on], loss_bound(size[on]))
    check(r.covered[on.cuda()], covered[on], 2 * P_REL * covered[on] + 1e-30)
    assert (r.losses.cpu()[~on] == 0).all() and (r.covered.cpu()[~on] == 0).all() and (d.cpu()[~on] == 0).all()
    check(d[on.cuda()], grad[on], grad_bound(grad[on], gsize[on], dtype))


@pytest.mark.parametrize("n,v", [(5, 900), (1000, 50257)])
def test_weights_that_are_all_zero(n, v):
    z = torch.full((n, v), math.nan, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ids, lq = torch.zeros(n, 4, dtype=torch.int64, device="cuda"), torch.zeros(n, 4, device="cuda")
    r = distillation_loss_from_logits(z, ids, lq, torch.zeros(n, device="cuda"))
    d, = torch.autograd.grad(r.loss, z)
    assert r.loss == 0 and (r.losses == 0).all() and (r.covered == 0).all() and (d == 0).all()


@pytest.mark.parametrize("k", [1, 2, 257, 512])
@pytest.mark.parametrize("v", [9, 4099, 70001])
def test_one_token_given_many_times(k, v):
    """Outcomes of one token: the teacher's probabilities differ, the student's is the same for all."""
    n = 5
    z = torch.randn(n, v, generator=gen(k), device="cuda") * 3
    ids = torch.full((n, k), v // 2, dtype=torch.int64, device="cuda")
    lq = torch.log_softmax(torch.randn(n, k + 1, generator=gen(k + 1), device="cuda"), 1)[:, :k]
    w = torch.rand(n, generator=gen(3), device="cuda") + 0.5
    losses, covered, grad, gsize, size = reference(z, ids, lq, "forward", "rest", 0.5, 1.0, w)
    z.requires_grad_(True)
    r = distillation_loss_from_logits(z, ids, lq, w)
    check(r.losses, losses, loss_bound(size))
    check(torch.autograd.grad(r.loss, z)[0], grad, grad_bound(grad, gsize, torch.float32))
    each, _ = distillation_from_logits(z, ids, lq)
    check(each, losses, loss_bound(size))
    check(torch.autograd.grad(each, z, w)[0], grad, grad_bound(grad, gsize, torch.float32))


@pytest.mark.parametrize("base,step", [(-2.0 ** 31, 256.0), (2.0 ** 31, 256.0), (-1e9, 64.0), (-3e38, 2.0 ** 104)])
@pytest.mark.parametrize("v", [700, 20011])
def test_logits_far_from_zero(base, step, v):
    """Logits whose reference in units of log2 leaves no room for differences: they are formed first."""
    n, k = 6, 8
    z = base + step * torch.randint(0, 3, (n, v), generator=gen(v), device="cuda").float()
    ids = torch.randint(0, v, (n, k), generator=gen(v + 1), device="cuda")
    lq = torch.log_softmax(torch.randn(n, k + 1, generator=gen(3), device="cuda"), 1)[:, :k]
    w = torch.rand(n, generator=gen(4), device="cuda") + 0.5
    for divergence, how in (("forward", dict(tail="rest")), ("jsd", dict(tail="drop"))):
        losses, covered, grad, gsize, size = reference(z, ids, lq, divergence, how["tail"], 0.5, 1.0, w)
        x = z.clone().requires_grad_(True)
        r = distillation_loss_from_logits(x, ids, lq, w, divergence=divergence, **how)
        check(r.losses, losses, loss_bound(size))
        check(r.covered, covered, 2 * P_REL * covered + 1e-30)
        check(torch.autograd.grad(r.loss, x)[0], grad, grad_bound(grad, gsize, torch.float32))
        each, _ = distillation_from_logits(x, ids, lq, divergence=divergence, **how)
        check(each, losses, loss_bound(size))
        check(torch.autograd.grad(each, x, w)[0], grad, grad_bound(grad, gsize, torch.float32))


@pytest.mark.parametrize("padded", [False, True])
def test_as_a_term_of_the_trainers_loss(padded):
    from axon_amd.models.fsdp_models import CausalLM
    from axon_amd.protocol import DataProto
    from axon_amd.trainer.algos.loss import agg_loss

    n, v = 120, 500
    z, ids, lq = batch(9, n, v, 8, torch.float32)
    shape = (4, 30) if padded else (n,)
    g = gen(4)
    rand = lambda: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    lp, ent, old, adv = rand(), rand().abs(), rand(), rand()
    mask = (torch.rand(*shape, generator=g, device="cuda") < 0.7).float()
    cu = None if padded else torch.tensor([0, 50, 90, 120], dtype=torch.int32, device="cuda")
    z[mask.reshape(-1) == 0] = math.nan  # what is no response has a loss that does not count
    x = z.clone().requires_grad_(True)

    def run(args, losses):
        data = DataProto.from_dict(tensors={"old_log_probs": old, "advantages": adv, "response_mask": mask},
                                   meta_info={} if padded else {"cu_seqlens": cu})
        meta = {"loss_fn": "ppo", "loss_fn_args": args, "dp_replicas": 2, "n_micro_batches": 4, "temperature": 1.0}
        module = lambda inputs, m: {"log_probs": lp, "entropys": ent, **({} if losses is None else {"distill_losses": losses})}  # noqa: E731
        return CausalLM.forward_backward_fn(module, data, meta)

    plain, metrics = run({}, None)
    assert not any("distill" in key for key in metrics)
    losses = distillation_from_logits(x, ids, lq)[0].view(shape)
    loss, metrics = run({"distill_coef": 0.25}, losses)
    want = agg_loss(torch.where(mask != 0, losses, 0.0), mask, cu_seqlens=cu)
    # three roundings of fp32 numbers of the losses' size; both replicas count
    assert abs(loss.item() - plain.item() - 2 * 0.25 * want.item()) <= 4 * 2.0 ** -24 * 2 * (abs(plain.item()) + abs(loss.item()) + 1)
    assert metrics["distill_loss"] == 4 * want.item() and metrics["distill_coef"] == 0.25
    d, = torch.autograd.grad(loss, x, retain_graph=True)
    ref, = torch.autograd.grad(want, x)
    keep = mask.reshape(-1) != 0
    assert ((d - 0.5 * ref).abs()[keep] <= 4 * 2.0 ** -24 * ref.abs()[keep] + 1e-30).all() and (d[~keep] == 0).all()
    with pytest.raises(ValueError, match="distill_losses"):
        run({"distill_coef": 0.25}, None)
    with pytest.raises(ValueError, match="do not lie beside"):
        run({"distill_coef": 0.25}, losses.reshape(-1)[:-1])


@pytest.mark.parametrize("n,v", [(40, 9001), (6, 151937), (700, 515)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_without_an_upstream_gradient(n, v, dtype):
    """Their gradient is 0, whatever they hold."""
    z, ids, lq = batch(n + v, n, v, 12, dtype)
    up = torch.randn(n, generator=gen(7), device="cuda")
    up[torch.rand(n, generator=gen(8), device="cuda") < 0.5] = 0.0
    up[0], up[1] = 0.0, -0.0
    on = up != 0
    losses, _, grad, gsize, size = reference(z, ids, lq, "forward", "rest", 0.5, 1.0, up)
    z[~on] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=dtype)[torch.arange(n, device="cuda")[~on] % 3, None]
    z.requires_grad_(True)
    got, _ = distillation_from_logits(z, ids, lq)
    d, = torch.autograd.grad(got, z, up)
    assert (d[~on] == 0).all()
    check(got[on], losses[on.cpu()], loss_bound(size[on.cpu()]))
    check(d[on], grad[on.cpu()], grad_bound(grad[on.cpu()], gsize[on.cpu()], dtype))
    twin = z.detach().clone().requires_grad_(True)
    over, _ = distillation_from_logits(twin * 1.0, ids, lq, inplace_backward=True)
    assert torch.equal(torch.autograd.grad(over, twin, up)[0], d)
    r = distillation_loss_from_logits(z, ids, lq, on.float())
    assert (torch.autograd.grad(r.loss, z, torch.tensor(0.0, device="cuda"))[0] == 0).all()


def test_batches_of_nothing():
    z = torch.zeros(2, 0, 50, device="cuda", requires_grad=True)
    ids, lq = torch.zeros(2, 0, 4, dtype=torch.int64, device="cuda"), torch.zeros(2, 0, 4, device="cuda")
    losses, covered = distillation_from_logits(z, ids, lq)
    assert losses.shape == covered.shape == (2, 0)
    assert torch.autograd.grad(losses.sum(), z)[0].shape == z.shape
    r = distillation_loss_from_logits(z, ids, lq, torch.zeros(2, 0, device="cuda"))
    assert r.loss == 0 and torch.autograd.grad(r.loss, z)[0].shape == z.shape


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("v", [5000, 151936])
def test_likely_tokens_are_exact_to_single_precision(v, weighted):
    """Rows with a likely token that the teacher knows: beside its term all others' additions would round at its size.  What is off in the
    sum: the others' share by the roundings of z - M and of its product with log2(e), 2^-24 of up to 30 each, that of log2(e), 1.4e-8 of
    it, and 2^-23 of the exponential (3.6e-6); the likely one's exponential and the factor that takes its reference's rounding back, 2^-23
    each; the three additions within its vector, 2^-24 each (all other additions are in 64 bits)."""
    n, k = 40, 6
    z = torch.randn(n, v, generator=gen(v), device="cuda") * 2
    at = torch.randint(0, v, (n,), generator=gen(1), device="cuda")
    z[torch.arange(n, device="cuda"), at] += 14.0 + 4.0 * torch.rand(n, generator=gen(3), device="cuda")
    t = torch.log_softmax(z + torch.randn(n, v, generator=gen(4), device="cuda"), 1)
    ids = t.topk(k, 1).indices
    lq = t.gather(1, ids)
    z.requires_grad_(True)
    if weighted:
        r = distillation_loss_from_logits(z, ids, lq, torch.ones(n, device="cuda"), tail="drop")
        got, total = r.losses, r.loss
    else:
        got, _ = distillation_from_logits(z, ids, lq, tail="drop")
        total = got.sum()
    log_p = torch.log_softmax(z.detach().double(), 1)
    q = lq.double().exp()
    want = (q * (lq.double() - log_p.gather(1, ids))).sum(1)
    share = 1.0 - log_p.exp().amax(1)
    lse_bound = 3.6e-6 * share + 7 * 2.0 ** -24
    assert ((got.double() - want).abs() <= q.sum(1) * lse_bound + 2.0 ** -24 * want.abs()).all()
    d, = torch.autograd.grad(total, z)
    p = log_p.exp()
    grad = p * q.sum(1, keepdim=True) - torch.zeros_like(p).scatter_(1, ids, q)
    # a probability: z - lse, its product with log2(e) and log2(e) itself, 2.5 2^-24 of the logarithm, and 2^-23; its factor and the product
    # with it, three roundings; a given token's own q: three as well
    bound = p * (lse_bound[:, None] + 5 * 2.0 ** -24 + 2.5 * 2.0 ** -24 * log_p.abs())
    bound = bound + 3 * 2.0 ** -24 * (p + torch.zeros_like(p).scatter_(1, ids, q)) + 1e-30
    assert ((d.double() - grad).abs() <= bound).all()
