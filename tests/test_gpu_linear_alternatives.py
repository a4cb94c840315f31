"""Top alternatives and log-probabilities of given tokens through the LM head, against the same in 64 bits."""

import math

import pytest
import torch

from axon_amd import _ops
from axon_amd.utils.kernel.linear_cross_entropy import linear_cross_entropy
from axon_amd.utils.kernel.linear_top_logprobs import linear_token_logprobs, linear_top_logprobs

pytestmark = pytest.mark.gpu

# Operands lie on a grid on which every sum of products is exact in 32 bits, so the logits are exact.  A log-probability is
# then off by the sums of exponentials (as for materialised logits, 4e-5 for |logit| <= 32) and, with a soft cap, by the
# hyperbolic tangent's 2^-21 (an exponential of 2^-22, a reciprocal of 2^-23, two roundings) times the cap and the inverse
# temperature, once for the token and once for the sum.
LP_TOL = 4e-5
ENT_TOL = 12 * 2e-5


def lp_tol(cap, inv_t):
    return LP_TOL + 2 * cap * inv_t * 2.0 ** -21


def operands(n, h, v, seed, peak=0.08, values=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shift = 2.0 ** -round(math.log2(math.sqrt(h)) - 1.0)
    w = (torch.randn(v, h, generator=g, device="cuda") * 4).round().clamp(-12, 12) / 4
    if values:  # few different rows: equal logits all over the vocabulary
        w = w[torch.randint(0, min(values, v), (v,), generator=g, device="cuda")]
    at = torch.randint(0, v, (n,), generator=g, device="cuda")
    hid = torch.randn(n, h, generator=g, device="cuda") + peak * w[at]
    hid = (hid * 32).round().clamp(-128, 128) / 32
    return hid.bfloat16(), (w * shift).bfloat16(), at


class Reference:
    def __init__(self, hid, w, inv_t, cap):
        self.h, self.w, self.inv_t, self.cap = hid.double(), w.double(), inv_t, cap
        self.raw = self.h @ self.w.t()
        z = cap * torch.tanh(self.raw / cap) if cap else self.raw
        self.slope = (1 - (z / cap) ** 2) * inv_t if cap else torch.full_like(z, inv_t)
        self.log_p = torch.log_softmax(z * inv_t, 1)
        self.p = self.log_p.exp()
        self.entropy = -(self.p * self.log_p).sum(1)

    def order(self, k):
        return torch.sort(self.raw, dim=1, descending=True, stable=True).indices[:, :k]

    def pick(self, ids):
        ok = (ids >= 0) & (ids < self.raw.shape[1])
        return torch.where(ok, self.log_p.gather(1, torch.where(ok, ids, torch.zeros_like(ids)).long()),
                           torch.zeros((), dtype=torch.float64, device=ids.device))

    def check_grads(self, ids, g_ids, g_en, d_hidden, d_weight):
        """A dlogit is off by its probability's error and rounded to bf16 (2^-8), a sum of them is rounded once more."""
        ok = (ids >= 0) & (ids < self.raw.shape[1])
        at = torch.where(ok, ids, torch.zeros_like(ids)).long()
        up = torch.where(ok, g_ids.double(), torch.zeros((), dtype=torch.float64, device=ids.device))
        ge = g_en.double()[:, None]
        zero = torch.zeros_like(self.p)
        d = zero.scatter_add(1, at, up) - self.p * (up.sum(1, keepdim=True) + ge * (self.log_p + self.entropy[:, None]))
        size = zero.scatter_add(1, at, up.abs()) + self.p * (
            up.abs().sum(1, keepdim=True) + ge.abs() * (self.log_p.abs() + self.entropy[:, None] + 1))
        d, size = d * self.slope, size * self.inv_t
        off = 2.0 ** -8 * d.abs() + (2 * ENT_TOL + 2 * (self.cap or 0) * self.inv_t * 2.0 ** -21) * size
        for got, ref, bound in ((d_hidden, d @ self.w, off @ self.w.abs()), (d_weight, d.t() @ self.h, off.t() @ self.h.abs())):
            worst = ((got.double() - ref).abs() / (bound + 2.0 ** -8 * ref.abs() + 1e-30)).max().item()
            assert worst <= 1.0, worst


SHAPES = [
    # tokens, hidden, vocabulary, k, temperature, cap, different weight rows
    (1, 32, 5, 5, 1.0, None, None),
    (3, 96, 300, 20, 1.0, None, None),
    (1, 896, 5003, 20, 1.0, None, None),
    (8, 64, 1000, 128, 0.7, 30.0, None),
    (130, 128, 2049, 7, 1.0, None, 9),
    (192, 64, 777, 64, 1.3, 5.0, None),
    (200, 64, 50257, 20, 1.0, None, None),
    (257, 64, 40000, 1, 1.0, 30.0, 300),
    (300, 96, 20000, 33, 0.7, 30.0, None),
    (515, 256, 4096, 16, 1.0, None, 3),
    (3, 32, 1400000, 5, 1.0, None, None),  # 10938 parts: their maxima are read where they lie
]


@pytest.mark.parametrize("n,h,v,k,temperature,cap,values", SHAPES)
def test_top_alternatives_through_the_head(n, h, v, k, temperature, cap, values):
    hid, w, lab = operands(n, h, v, 3 * n + v, values=values)
    lab = lab.clone()
    if n > 1:
        lab[-1] = v
    ref = Reference(hid, w, 1 / temperature, cap)
    ids = ref.order(k)
    hid.requires_grad_(True)
    w.requires_grad_(True)
    r = linear_top_logprobs(hid, w, k, lab, temperature, cap)
    assert torch.equal(r.top_ids, ids)
    tol = lp_tol(cap or 0, 1 / temperature)
    assert (r.top_logprobs.double() - ref.pick(ids)).abs().max() <= tol
    assert (r.logprobs.double() - ref.pick(lab[:, None])[:, 0]).abs().max() <= tol
    assert (r.entropy.double() - ref.entropy).abs().max() <= ENT_TOL + 12 * tol
    g = torch.Generator(device="cuda").manual_seed(n)
    g_top, g_lp, g_en = (torch.randn(*s, generator=g, device="cuda") for s in ((n, k), (n,), (n,)))
    got = torch.autograd.grad([r.top_logprobs, r.logprobs, r.entropy], [hid, w], [g_top, g_lp, g_en])
    ref.check_grads(torch.cat([lab[:, None], ids], 1), torch.cat([g_lp[:, None], g_top], 1), g_en, *got)


@pytest.mark.parametrize("n,h,v,k,temperature,cap", [
    (1, 32, 9, 2, 1.0, None),
    (5, 96, 300, 40, 0.7, 30.0),
    (61, 896, 5003, 512, 1.0, None),  # an odd vocabulary: a second, vocabulary-major copy of the dlogits
    (300, 256, 33024, 8, 1.0, 30.0),
    (700, 320, 2056, 64, 1.3, None),
])
@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_given_tokens_through_the_head(n, h, v, k, temperature, cap, ids_dtype):
    hid, w, lab = operands(n, h, v, n + v)
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.randint(-1, v + 1, (n, k), generator=g, device="cuda")
    ids[:, 0] = lab
    ids[0, -1] = ids[0, 0]  # twice in one position
    ref = Reference(hid, w, 1 / temperature, cap)
    hid.requires_grad_(True)
    w.requires_grad_(True)
    lp, ent = linear_token_logprobs(hid, w, ids.to(ids_dtype), temperature, cap)
    tol = lp_tol(cap or 0, 1 / temperature)
    assert (lp.double() - ref.pick(ids)).abs().max() <= tol
    assert (ent.double() - ref.entropy).abs().max() <= ENT_TOL + 12 * tol
    g_ids, g_en = torch.randn(n, k, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    got = torch.autograd.grad([lp, ent], [hid, w], [g_ids, g_en])
    ref.check_grads(ids, g_ids, g_en, *got)


def test_vocabulary_chunks():
    """A backward whose vocabulary goes in pieces writes each id's dlogit in its own piece: as many tokens as make the
    default piece shorter than the vocabulary."""
    n, h, v, k = 16640, 64, 66048, 3
    hid, w, lab = operands(n, h, v, 5)
    ids = torch.stack([lab, (lab + 1) % v, torch.full_like(lab, -1)], 1)
    g = torch.randn(n, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    lp, ent, lse, mean, _ = _ops.lmhead_tokens(hid, w, ids)
    d_h, d_w = _ops.lmhead_tokens_backward(g, None, hid, w, ids, lp, lse, mean)
    part = torch.arange(0, n, 997, device="cuda")
    ref = Reference(hid[part], w, 1.0, None)
    assert (lp[part].double() - ref.pick(ids[part])).abs().max() <= LP_TOL
    up = g[part, :2].double()
    d = torch.zeros_like(ref.p).scatter_add_(1, ids[part, :2], up) - ref.p * up.sum(1, keepdim=True)
    off = 2.0 ** -8 * d.abs() + 2 * ENT_TOL * (ref.p * up.abs().sum(1, keepdim=True))
    bound = off @ ref.w.abs() + 2.0 ** -8 * (d @ ref.w).abs() + 1e-30
    assert ((d_h[part].double() - d @ ref.w).abs() / bound).max() <= 1.0
    # what a row of the weight gets from the ids alone is there: the label's gradient towards its hidden state
    row = int(lab[0])
    same = (ids == row).double() * g.double()
    direct = (same.sum(1)[:, None] * hid.double()).sum(0)
    assert torch.nn.functional.cosine_similarity(direct, d_w[row].double(), 0) > 0.9


def test_blocks_of_tokens_give_the_same(monkeypatch):
    n, h, v, k = 700, 64, 3000, 12
    hid, w, lab = operands(n, h, v, 1)
    whole = linear_top_logprobs(hid, w, k, lab)
    monkeypatch.setattr(_ops, "TOP_LOGITS_BYTES", 1)  # 256 tokens per block
    cut = linear_top_logprobs(hid, w, k, lab)
    for a, b in zip(whole, cut):
        assert torch.equal(a, b)


def test_agrees_with_the_head_for_one_label():
    n, h, v = 300, 128, 5000
    hid, w, lab = operands(n, h, v, 2)
    lp, ent = linear_cross_entropy(hid, w, lab, 0.7, "none", None, 20.0)
    r = linear_top_logprobs(hid, w, 3, lab, 0.7, 20.0)
    t_lp, t_ent = linear_token_logprobs(hid, w, lab[:, None], 0.7, 20.0)
    assert torch.equal(r.logprobs, lp) and torch.equal(r.entropy, ent) and torch.equal(t_ent, ent)
    assert (t_lp[:, 0] - lp).abs().max() <= lp_tol(20.0, 1 / 0.7)


def test_shapes_and_other_types():
    n, h, v = 12, 64, 500
    hid, w, lab = operands(n, h, v, 4)
    h3 = hid.view(3, 4, h).float().requires_grad_(True)
    w16 = w.half().requires_grad_(True)
    with pytest.warns(UserWarning) if not _warned() else _quiet():
        r = linear_top_logprobs(h3, w16, 5, lab.view(3, 4))
    assert r.top_ids.shape == (3, 4, 5) and r.logprobs.shape == (3, 4) and not r.top_ids.requires_grad
    d_h, d_w = torch.autograd.grad(r.top_logprobs.sum(), [h3, w16])
    assert d_h.dtype == torch.float32 and d_h.shape == h3.shape and d_w.dtype == torch.float16
    # operands that are views: strided rows, a start off a 16-byte boundary
    wide = torch.zeros(n, h + 8, device="cuda", dtype=torch.bfloat16)
    wide[:, 4:4 + h] = hid
    flat = torch.zeros(v * h + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = w.reshape(-1)
    got = linear_top_logprobs(wide[:, 4:4 + h], flat[1:].view(v, h), 5, lab)
    want = linear_top_logprobs(hid, w, 5, lab)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = torch.empty(0, h, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    wg = w.clone().requires_grad_(True)
    r = linear_top_logprobs(empty, wg, 5)
    assert r.top_ids.shape == (0, 5) and r.logprobs is None
    lp, _ = linear_token_logprobs(empty, wg, torch.empty(0, 2, dtype=torch.int64, device="cuda"))
    d_h, d_w = torch.autograd.grad(lp.sum() + r.top_logprobs.sum(), [empty, wg])
    assert d_h.shape == (0, h) and not d_w.any()


def _warned():
    from axon_amd.utils.kernel import linear_cross_entropy as m

    return m._warned_rounding


def _quiet():
    import contextlib

    return contextlib.nullcontext()


def test_a_student_on_a_teachers_alternatives():
    """The two together: a teacher stores its alternatives, a student is trained on them; the loss's gradient agrees with
    differences of the loss in 64 bits along a direction."""
    n, h, v, k = 40, 64, 600, 10
    teacher_h, w, _ = operands(n, h, v, 1)
    student_h, _, _ = operands(n, h, v, 2)
    with torch.no_grad():
        t = linear_top_logprobs(teacher_h, w, k)
    x = student_h.clone().requires_grad_(True)
    lp, ent = linear_token_logprobs(x, w, t.top_ids)
    p = t.top_logprobs.exp()
    loss = (p * (t.top_logprobs - lp)).sum(1).mean() - 0.01 * ent.mean()
    grad, = torch.autograd.grad(loss, x)

    def value(hidden):
        log_p = torch.log_softmax(hidden @ w.double().t(), 1)
        kl = (p.double() * (t.top_logprobs.double() - log_p.gather(1, t.top_ids))).sum(1).mean()
        return kl - 0.01 * (-(log_p.exp() * log_p).sum(1)).mean()

    d = torch.randn(n, h, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).double()
    eps = 1e-4
    slope = (value(student_h.double() + eps * d) - value(student_h.double() - eps * d)) / (2 * eps)
    along = (grad.double() * d).sum()
    # every entry of the gradient is off by two roundings of 2^-8 of its terms: half the sum of their sizes at the worst
    assert (slope - along).abs() <= 2.0 ** -7 * (grad.double().abs() * d.abs()).sum() + 1e-6
    assert abs(loss.item() - value(student_h.double()).item()) <= 2 * ENT_TOL


@pytest.mark.parametrize("h", [128, 768])
def test_results_repeat_and_replay(h):
    """Forward and backward repeat bit for bit, eagerly and as a graph replayed on other inputs."""
    n, v, k = 130, 4096, 9
    hid, w, _ = operands(n, h, v, 7)
    ids = torch.randint(0, 5, (n, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    g = torch.randn(n, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))

    hid.requires_grad_(True)
    w.requires_grad_(True)

    def step():
        r = linear_top_logprobs(hid, w, k)
        lp, ent = linear_token_logprobs(hid, w, ids)
        return [r.entropy.detach(), r.top_ids, lp.detach(), *torch.autograd.grad([r.top_logprobs, ent, lp], [hid, w], [g, g[:, 0], g])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (7, 8, 9):
        with torch.no_grad():
            hid.copy_(operands(n, h, v, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(held, step(), step()):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("n,h,v,temperature,cap", [(40, 768, 3000, 1.0, None), (190, 832, 2051, 0.7, 20.0), (300, 768, 5000, 1.0, None),
                                                   (513, 1024, 2048, 1.3, 30.0)])
def test_kept_logits_give_the_same_gradients(monkeypatch, n, h, v, temperature, cap):
    """Bit for bit, whether the backward takes the logits that the forward has kept or recomputes them."""
    hid, w, lab = operands(n, h, v, 6)
    ids = torch.randint(-1, v, (n, 7), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    g = torch.randn(n, 7, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    hid.requires_grad_(True)
    w.requires_grad_(True)

    def step():
        lp, ent = linear_token_logprobs(hid, w, ids, temperature, cap)
        r = linear_top_logprobs(hid, w, 7, lab, temperature, cap)
        saved = [t for t in lp.grad_fn.saved_tensors + r.entropy.grad_fn.saved_tensors if t is not None and t.dtype == torch.uint8]
        a = torch.autograd.grad([lp, ent], [hid, w], [g, g[:, 0]])
        b = torch.autograd.grad([r.top_logprobs, r.logprobs], [hid, w], [g, g[:, 1]])
        return lp.detach(), r.top_ids, [*a, *b], len(saved)

    lp, top, grads, kept = step()
    assert kept == 2
    monkeypatch.setattr(_ops, "TOP_KEEP_LOGITS_MIN_HIDDEN", 1 << 30)
    lp2, top2, grads2, kept = step()
    assert kept == 0 and torch.equal(top, top2) and (lp - lp2).abs().max() <= lp_tol(cap or 0, 1 / temperature)
    # the given tokens' log-probabilities come from the product here and from a dot there: their dlogits, of relative error
    # LP_TOL, may round to the other neighbour in bf16; the alternatives' are the same numbers
    assert all(torch.equal(x, y) for x, y in zip(grads[2:], grads2[2:]))
    ref = Reference(hid.detach(), w.detach(), 1 / temperature, cap)
    for pair in (grads[:2], grads2[:2]):
        ref.check_grads(ids, g, g[:, 0], *pair)


def test_saved_tensors_from_a_hook_are_looked_at_again():
    n, h, v = 20, 768, 600
    hid, w, lab = operands(n, h, v, 3)

    def backward_with(unpack):
        a, b = hid.clone().requires_grad_(True), w.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            r = linear_top_logprobs(a, b, 3, lab)
        return torch.autograd.grad(r.top_logprobs.sum() + r.logprobs.sum(), [a, b])

    want = backward_with(lambda t: t)
    assert all(torch.equal(x, y) for x, y in zip(backward_with(lambda t: t.clone()), want))
    for unpack in (lambda t: t.cpu(), lambda t: t.cpu() if t.dim() == 1 and t.dtype == torch.float32 else t,
                   lambda t: t.cpu() if t.dtype == torch.int64 else t, lambda t: t.cpu() if t.dtype == torch.uint8 else t,
                   lambda t: t[:-16] if t.dtype == torch.uint8 else t, lambda t: t[:5] if t.dim() == 2 and t.dtype == torch.float32 else t):
        with pytest.raises((RuntimeError, ValueError)):
            backward_with(unpack)


@pytest.mark.parametrize("n,v,k", [(3, 500, 4), (300, 2000, 1), (300, 40000, 9)])
def test_a_row_of_nan_has_valid_ids(n, v, k):
    hid, w, lab = operands(n, 64, v, 4)
    want = linear_top_logprobs(hid, w, k, lab)
    hid[1] = math.nan
    r = linear_top_logprobs(hid, w, k, lab)
    assert torch.equal(r.top_ids[1], torch.arange(k, device="cuda")) and torch.isnan(r.top_logprobs[1]).all()
    others = torch.arange(n, device="cuda") != 1
    assert torch.equal(r.top_ids[others], want.top_ids[others]) and torch.equal(r.top_logprobs[others], want.top_logprobs[others])


def test_scoring_without_gradients_keeps_no_logits():
    """Under ``no_grad`` a head that could be trained costs what any other does."""
    n, h, v = 600, 768, 20000
    hid, w, lab = operands(n, h, v, 3)
    trained = w.clone().requires_grad_(True)
    logits = n * v * 4

    def peak_of(op):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = op()
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before, out

    ids = lab[:, None].expand(n, 4)
    with torch.no_grad():
        plain, (lp, ent) = peak_of(lambda: linear_token_logprobs(hid, trained, ids))
    assert plain < logits // 2 and not lp.requires_grad
    frozen, (lp2, ent2) = peak_of(lambda: linear_token_logprobs(hid, w, ids))
    assert frozen == plain and torch.equal(lp, lp2) and torch.equal(ent, ent2)
    held, (lp3, _) = peak_of(lambda: linear_token_logprobs(hid, trained, ids))
    assert held >= logits and lp3.requires_grad


@pytest.mark.parametrize("h", [64, 768])
@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("temperature,cap", [(1.0, None), (0.7, None), (0.7, 30.0)])
def test_positions_with_one_likely_token(n, h, temperature, cap):
    """A probability is at most 1, its logarithm at most 0; without a soft cap, whose argument is formed in another order there, the
    token has the value that the head gives a label with the same exact logit, in every form.

    A likely token's log-probability is off by its sum of exponentials: up to 20 additions in a tile's lane, three among lanes, 24
    merges of two roundings, of 2^-24 each, an exponential and a logarithm of 2^-22 near 1, an argument that is rounded
    once (60 * 2^-24 * what is not 0 of its difference): 71 * 2^-24 + 2 * 2^-22 < 6e-6, with a soft cap lp_tol's term for it more."""
    hid, w, lab = operands(n, h, 5003, n + h, peak=0.0)
    shift = w.float().abs().max() / 3  # entries of w are multiples of a quarter of this
    rows = (w.float() / shift)[lab]
    # label logits of 10 to 46 above the others' centre (|row|^2 shift peak, |row|^2 about h)
    peak = torch.linspace(10, 46, n, device="cuda")[:, None] / (rows.square().sum(1, keepdim=True) * shift)
    step = 2.0 ** -4
    hid = (((hid.float() / 4 + peak * rows) / step).round().clamp(-127, 127) * step).bfloat16()
    ref = Reference(hid, w, 1 / temperature, cap)
    ids = ref.order(3)
    want, best = ref.pick(lab[:, None])[:, 0], ref.pick(ids)
    assert want.max() > -1e-5 and want.min() < -1e-3
    r = linear_top_logprobs(hid, w, 3, lab, temperature, cap)
    wg = w.clone().requires_grad_(True)
    plain = linear_token_logprobs(hid, w, lab[:, None], temperature, cap)[0][:, 0]
    kept = linear_token_logprobs(hid, wg, lab[:, None], temperature, cap)[0].detach()[:, 0]
    assert torch.equal(r.top_ids, ids)
    tol = 6e-6 + (lp_tol(cap, 1 / temperature) - LP_TOL if cap else 0)
    for got, exact in ((plain, want), (kept, want), (r.top_logprobs[:, 0], best[:, 0])):
        assert (got <= 0).all()
        assert (got.double() - exact).abs().max() <= tol
    assert torch.equal(kept, plain)
    at = ids[:, 0] == lab
    assert at.sum() > n // 2 and torch.equal(r.top_logprobs[at, 0], plain[at])
    if not cap:
        assert torch.equal(plain, r.logprobs.clamp(max=0))


def test_weight_gradients_on_both_sides_of_every_chunk_border():
    """A backward in pieces of the vocabulary: rows of d_weight at the ends of every piece, and of ids' own, element by element."""
    n, h, v, k = 16640, 64, 66048, 3
    hid, w, lab = operands(n, h, v, 5)
    ids = torch.stack([lab, (lab + 1) % v, torch.full_like(lab, -1)], 1)
    g = torch.randn(n, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    g_en = torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) * 0.1
    lp, _, lse, mean, _ = _ops.lmhead_tokens(hid, w, ids)
    _, d_w = _ops.lmhead_tokens_backward(g, g_en, hid, w, ids, lp, lse, mean)
    pieces = sorted({c + i for c in range(0, v, 256) for i in (-1, 0)} & set(range(v)))  # whatever the pieces' length
    rows = torch.tensor(sorted({*pieces, 1, v - 2, v - 1, *lab[:8].tolist(), *ids[:8, 1].tolist()}), device="cuda")
    h64, w64 = hid.double(), w.double()
    up, got = g[:, :2].double(), d_w[rows].double()
    ref, off = torch.zeros_like(got), torch.zeros_like(got)
    for a in range(0, n, 1664):
        c = slice(a, a + 1664)
        log_p = torch.log_softmax(h64[c] @ w64.t(), 1)
        entropy = -(log_p.exp() * log_p).sum(1, keepdim=True)
        z = log_p[:, rows]
        p, G, ge = z.exp(), up[c].sum(1, keepdim=True), g_en[c, None].double()
        same = [(ids[c, i, None] == rows).double() * up[c, i, None] for i in (0, 1)]
        d = same[0] + same[1] - p * (G + ge * (z + entropy))
        size = same[0].abs() + same[1].abs() + p * (up[c].abs().sum(1, keepdim=True) + ge.abs() * (z.abs() + entropy + 1))
        ref += d.t() @ h64[c]
        off += (2.0 ** -8 * d.abs() + 2 * ENT_TOL * size).t() @ h64[c].abs()
    assert ((got - ref).abs() <= off + 2.0 ** -8 * ref.abs() + 1e-30).all()
