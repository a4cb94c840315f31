"""Top alternatives and log-probabilities of given tokens from materialised logits, against the same in 64 bits."""

import math

import pytest
import torch

from axon_amd.utils.torch.ops import (logprobs_and_entropy_from_logits, token_logprobs_from_logits,
                                      top_logprobs_from_logits)

pytestmark = pytest.mark.gpu

# How far a log-probability may be off, |logit| <= 32: the sum of exponentials is added up in chains of at most 300
# roundings of 2^-24 (2e-5 at the worst, were they all of one sign: 300 * 6e-8), each exponential is off by the rounding
# of an argument of up to 60 in 2^-24 and by 2^-22 (4e-6, weighted by its probability), the final additions by four
# roundings of a number of up to 46 (1.1e-5).
LP_TOL = 4e-5
# The entropy is formed from the same sums, its terms weighted by up to |log p|, of which 12 is the average at most.
ENT_TOL = 12 * 2e-5


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def logits_of(pattern, n, v, dtype, seed):
    g = gen(seed)
    z = torch.randn(n, v, generator=g, device="cuda") * 3
    if pattern == "constant":
        z = torch.full_like(z, 0.75)
    elif pattern == "few_values":
        z = torch.randint(-1, 2, (n, v), generator=g, device="cuda").float()
    elif pattern == "rising":
        z = torch.arange(v, device="cuda").float().expand(n, v) * (16.0 / v)
    elif pattern == "falling":
        z = torch.arange(v, 0, -1, device="cuda").float().expand(n, v) * (16.0 / v)
    elif pattern == "signed_zero":
        z = torch.where(torch.rand(n, v, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    elif pattern == "banned":
        z[torch.rand(n, v, generator=g, device="cuda") < 0.9] = -math.inf
        z[:, v // 2] = 1.0
    elif pattern == "one_block":  # all that is large lies in one run
        z[:, v // 3: v // 3 + 300] += 20.0
    elif pattern == "peaked":
        z[:, v // 2] += 25.0
    return z.clamp(-math.inf, 31.0).to(dtype).contiguous()


def reference(z, ids, g_ids=None, g_ent=None):
    """Log-probabilities of ids (0 outside the vocabulary), entropy; the gradient and the size of its terms."""
    z = z.double()
    log_p = torch.log_softmax(z, 1)
    p = log_p.exp()
    plogp = torch.where(p > 0, p * log_p, torch.zeros_like(p))
    ent = -plogp.sum(1)
    ok = (ids >= 0) & (ids < z.shape[1])
    at = torch.where(ok, ids, torch.zeros_like(ids)).long()
    lp = torch.where(ok, log_p.gather(1, at), torch.zeros((), dtype=torch.float64, device=z.device))
    if g_ids is None:
        return lp, ent
    up = torch.where(ok, g_ids.double(), torch.zeros((), dtype=torch.float64, device=z.device))
    onehot = torch.zeros_like(z).scatter_add_(1, at, up)
    G, ge = up.sum(1, keepdim=True), g_ent.double()[:, None]
    grad = onehot - p * G - ge * (plogp + p * ent[:, None])
    size = (torch.zeros_like(z).scatter_add_(1, at, up.abs()) + p * up.abs().sum(1, keepdim=True)
            + ge.abs() * (plogp.abs() + p * (ent[:, None] + 1)))
    return lp, ent, grad, size


def order(z, k):
    return torch.sort(z.double() + 0.0, dim=1, descending=True, stable=True).indices[:, :k]


def check_grad(got, ref, size, dtype):
    """A probability's relative error is that of its logarithm (LP_TOL) and of two roundings; a bf16 gradient is rounded
    once more (2^-8)."""
    bound = 2 * ENT_TOL * size + 1e-30
    if dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * ref.abs()
    worst = ((got.double() - ref).abs() / bound).max().item()
    assert worst <= 1.0, worst


def laid_out(z, layout):
    """The same values in another place: rows further apart, off a 16-byte boundary, or with another dimension."""
    n, v = z.shape
    if layout == "plain":
        return z
    if layout == "strided":
        buf = torch.full((n, v + 5), 99.0, device=z.device, dtype=z.dtype)
        buf[:, :v] = z
        return buf[:, :v]
    buf = torch.full((n * v + 3,), 99.0, device=z.device, dtype=z.dtype)
    buf[3:] = z.reshape(-1)
    return buf[3:].view(n, v)


TOP_CASES = [
    # n, vocab, k, dtype, pattern, layout
    (1, 1, 1, torch.float32, "random", "plain"),
    (3, 5, 5, torch.bfloat16, "random", "shifted"),
    (2, 17, 3, torch.float32, "random", "shifted"),
    (5, 127, 64, torch.bfloat16, "few_values", "plain"),
    (4, 129, 128, torch.float32, "random", "strided"),
    (7, 1000, 20, torch.bfloat16, "constant", "plain"),
    (3, 4099, 128, torch.bfloat16, "constant", "shifted"),
    (2, 40000, 128, torch.float32, "constant", "plain"),
    (3, 40000, 128, torch.bfloat16, "few_values", "strided"),
    (6, 4099, 20, torch.float32, "rising", "plain"),
    (6, 4099, 20, torch.float32, "falling", "strided"),
    (3, 50257, 128, torch.bfloat16, "one_block", "plain"),
    (2, 33000, 128, torch.float32, "one_block", "shifted"),
    (5, 3001, 100, torch.float32, "signed_zero", "plain"),
    (9, 2048, 50, torch.bfloat16, "banned", "plain"),
    (3, 600, 128, torch.float32, "banned", "plain"),
    (1, 151936, 20, torch.bfloat16, "random", "plain"),
    (3, 201088, 5, torch.float32, "peaked", "plain"),
    (61, 50257, 7, torch.bfloat16, "random", "plain"),
    (1600, 777, 33, torch.bfloat16, "random", "plain"),
    (1537, 2051, 1, torch.float32, "few_values", "plain"),
]


@pytest.mark.parametrize("n,v,k,dtype,pattern,layout", TOP_CASES)
def test_top_alternatives(n, v, k, dtype, pattern, layout):
    z = logits_of(pattern, n, v, dtype, 11 * n + v)
    ids = order(z, k)
    labels = torch.randint(0, v, (n,), generator=gen(5), device="cuda")
    labels[-1] = v if n > 1 else 0  # a label outside the vocabulary
    lp, ent = reference(z, torch.cat([ids, labels[:, None]], 1))
    r = top_logprobs_from_logits(laid_out(z, layout), k, labels)
    assert r.top_ids.dtype == torch.int64 and torch.equal(r.top_ids, ids)
    both = torch.cat([r.top_logprobs, r.logprobs[:, None]], 1).double()
    finite = torch.isfinite(lp)
    assert torch.equal(torch.isfinite(both), finite)
    assert (both - lp)[finite].abs().max() <= LP_TOL and (both[~finite] == -math.inf).all()
    assert (r.entropy.double() - ent).abs().max() <= ENT_TOL
    bare = top_logprobs_from_logits(z, k)
    assert bare.logprobs is None and torch.equal(bare.top_ids, ids)


def test_rows_without_a_softmax():
    """NaN and infinities stay in their row; ids are valid wherever the values are not."""
    z = logits_of("random", 5, 3000, torch.float32, 3)
    good = top_logprobs_from_logits(z, 9)
    z[0, 77] = math.nan
    z[1] = -math.inf
    z[2, 5] = math.inf
    z[3] = math.nan
    r = top_logprobs_from_logits(z, 9)
    assert torch.isnan(r.top_logprobs[[0, 1, 3]]).all() and torch.isnan(r.entropy[[0, 1, 2, 3]]).all()
    assert torch.isnan(r.top_logprobs[2, 0])
    assert torch.equal(r.top_ids[1], torch.arange(9, device="cuda")) and torch.equal(r.top_ids[3], torch.arange(9, device="cuda"))
    assert r.top_ids[2, 0] == 5 and 77 not in r.top_ids[0].tolist()
    assert torch.equal(r.top_ids[4], good.top_ids[4]) and torch.equal(r.top_logprobs[4], good.top_logprobs[4])


@pytest.mark.parametrize("v,dtype", [(3000, torch.float32), (3000, torch.bfloat16), (12, torch.float32), (151936, torch.bfloat16)])
@pytest.mark.parametrize("k", [1, 7])
def test_ids_are_valid_whatever_the_row_holds(v, dtype, k):
    """NaN counts as -inf for the ids: every row gets k different ids of the vocabulary, the lowest where nothing tells them
    apart.  (The last segment of a row is filled up with -inf, which a row of NaN alone has to reach.)"""
    z = logits_of("random", 4, v, dtype, 3)
    z[0] = math.nan
    z[1, : v - 1] = math.nan
    z[2, ::2] = math.nan
    z[3] = -math.inf
    z[3, v // 2] = math.nan
    for many in (1, 200):  # rows that several workgroups share, and rows that one finishes
        r = top_logprobs_from_logits(z.repeat(many, 1), k)
        for row in range(4):
            want = order(torch.where(torch.isnan(z[row]), torch.tensor(-math.inf, dtype=dtype, device="cuda"), z[row])[None], k)[0]
            assert (r.top_ids[row::4] == want).all()
            assert torch.isnan(r.top_logprobs[row::4]).all() and torch.isnan(r.entropy[row::4]).all()


def test_signaling_nan_hides_nothing():
    """A NaN of any bits beside a row's largest logit."""
    for dtype, ints, bits in ((torch.float32, torch.int32, 0x7f800001), (torch.bfloat16, torch.int16, 0x7f81)):
        z = torch.randn(4, 6000, generator=gen(2), device="cuda").to(dtype)
        z[:, 2048] = 30.0
        for row, at in enumerate((2047, 2049, 2055, 2060)):
            z[row, at] = torch.tensor(bits, dtype=ints, device="cuda").view(dtype)
        clean = torch.where(torch.isnan(z), torch.tensor(-math.inf, dtype=dtype, device="cuda"), z)
        for many in (1, 150):
            r = top_logprobs_from_logits(z.repeat(many, 1), 5)
            assert (r.top_ids.view(many, 4, 5) == order(clean, 5)).all() and torch.isnan(r.top_logprobs).all()


def far_rows(v, dtype, g):
    """Rows whose log-sum-exp is far from 0: what a mask of a large number or of the type's lowest has left nothing of."""
    lowest = torch.finfo(dtype).min
    z = torch.randn(9, v, generator=g, device="cuda") * 3
    z[0] = -1e9
    z[1] = lowest
    z[2] = z[2] * 1000 - 1e9
    z[3] += 20000
    z[4] -= 60000
    z[5, : v // 2] = lowest  # a mask that leaves something
    z[6] = lowest
    z[6, v // 2] = -1e33
    z[7] = torch.finfo(dtype).max
    z[8] = -3e30
    z[8, ::2] = lowest
    return z.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [12, 3001, 151936])
def test_rows_far_from_zero(v, dtype):
    """A log-probability is off by LP_TOL and two roundings of its own size (the difference from the log-sum-exp, and what is
    left of that): the sums of such a row go in chains of at most 600 (3.5e-5), its final additions are of numbers up to 12."""
    g = gen(v)
    z, k = far_rows(v, dtype, g), 5
    for many in (1, 60):  # rows that several workgroups share, and rows that one finishes
        x = z.repeat(many, 1).requires_grad_(True)
        ids = torch.cat([order(z, k), torch.randint(0, v, (9, 3), generator=g, device="cuda")], 1).repeat(many, 1)
        g_ids, g_en = torch.randn(9 * many, 8, generator=g, device="cuda"), torch.randn(9 * many, generator=g, device="cuda")
        lp, ent, ref, size = reference(x.detach(), ids, g_ids, g_en)
        r = top_logprobs_from_logits(x, k, ids[:, 6])
        assert torch.equal(r.top_ids, ids[:, :k])
        got_lp, got_ent = token_logprobs_from_logits(x, ids)
        for got, want in ((r.top_logprobs, lp[:, :k]), (r.logprobs, lp[:, 6]), (got_lp, lp)):
            assert ((got.double() - want).abs() <= LP_TOL + 2.0 ** -23 * want.abs()).all()
        for got in (r.entropy, got_ent):
            assert (got.double() - ent).abs().max() <= ENT_TOL
        grad, = torch.autograd.grad([got_lp, got_ent], x, [g_ids, g_en])
        check_grad(grad, ref, size, dtype)


def test_rows_whose_maxima_do_not_fit_in_lds():
    """700001 fp32 logits are 10938 segments: rows that a workgroup would finish are finished by a second launch."""
    z = logits_of("random", 8, 700001, torch.float32, 6)
    z[3] = 1.0
    r = top_logprobs_from_logits(z.repeat(65, 1), 40)
    assert (r.top_ids.view(65, 8, 40) == order(z, 40)).all()
    few = top_logprobs_from_logits(z, 40)
    lp, ent = reference(z, order(z, 40))
    # chains of 700001 / 256 roundings
    for got, entropy in ((r.top_logprobs[-8:], r.entropy[-8:]), (few.top_logprobs, few.entropy)):
        assert (got.double() - lp).abs().max() <= LP_TOL + 2735 * 2.0 ** -24
        assert (entropy.double() - ent).abs().max() <= ENT_TOL + 14 * 2735 * 2.0 ** -24


@pytest.mark.parametrize("n", [3, 600])
def test_rows_with_one_likely_token(n):
    """The largest logit, near 29, adds exactly 1 to the sum, all others together at most 2^-22 (what is lost of them beside
    it); the difference from the log-sum-exp and its rest is exact: log-probabilities of almost 0 to 2^-22, not to 30 times the
    rounding of a factor (4e-7)."""
    z = logits_of("random", n, 2000, torch.float32, 9).clamp(max=10.5)
    z[:, 777] = 29 + torch.rand(n, generator=gen(3), device="cuda")
    others = torch.exp(z.double() - z[:, 777:778].double()).sum(1) - 1
    assert others.max() < 2.0 ** -22
    at = torch.full((n, 1), 777, device="cuda")
    want = reference(z, at)[0]
    r = top_logprobs_from_logits(z, 1, at[:, 0])
    for got in (r.top_logprobs, r.logprobs[:, None], token_logprobs_from_logits(z, at)[0]):
        assert (got.double() - want).abs().max() <= 2.0 ** -22


def test_logits_written_to_before_the_backward_are_noticed():
    z = logits_of("random", 4, 300, torch.float32, 2)
    for op in (lambda x: top_logprobs_from_logits(x, 3).top_logprobs, lambda x: token_logprobs_from_logits(x, torch.zeros(4, 1, dtype=torch.int64, device="cuda"))[0]):
        x = z.clone().requires_grad_(True) * 1
        out = op(x)
        with torch.no_grad():
            x += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_offsets_beyond_32_bits():
    z = logits_of("random", 3, 1000, torch.bfloat16, 1)
    buf = torch.empty(2 ** 31 + 5000, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((3, 1000), (2 ** 30 + 8, 1))
    far.copy_(z)
    ids = torch.randint(0, 1000, (3, 6), generator=gen(1), device="cuda")
    g = torch.randn(3, 6, generator=gen(2), device="cuda")
    results = []
    for x in (z.clone(), far):
        x = x.detach().requires_grad_(True)
        r = top_logprobs_from_logits(x, 9, ids[:, 0])
        lp, ent = token_logprobs_from_logits(x, ids, inplace_backward=True)
        grad, = torch.autograd.grad([lp, ent], x, [g, g[:, 0].clone()])
        assert grad.data_ptr() == x.data_ptr()
        results.append([r.top_ids, r.top_logprobs.detach(), r.logprobs.detach(), lp.detach(), ent.detach(), grad.clone()])
    assert all(torch.equal(a, b) for a, b in zip(*results))


GRAD_CASES = [
    (1, 9, 3, torch.float32, "random", "plain"),
    (3, 129, 20, torch.bfloat16, "random", "shifted"),
    (61, 4099, 64, torch.bfloat16, "random", "plain"),
    (5, 3000, 20, torch.float32, "banned", "strided"),
    (2, 40000, 128, torch.bfloat16, "constant", "plain"),
    (187, 50257, 8, torch.float32, "peaked", "plain"),
    (1540, 515, 5, torch.bfloat16, "random", "plain"),
]


@pytest.mark.parametrize("n,v,k,dtype,pattern,layout", GRAD_CASES)
def test_top_alternatives_gradient(n, v, k, dtype, pattern, layout):
    z = logits_of(pattern, n, v, dtype, n + v)
    g = gen(n)
    g_top, g_lp, g_en = (torch.randn(*s, generator=g, device="cuda") for s in ((n, k), (n,), (n,)))
    labels = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
    labels[0] = order(z, 1)[0, 0]  # a label that is an alternative too
    labels[-1] = -100
    x = laid_out(z, layout).requires_grad_(True)
    r = top_logprobs_from_logits(x, k, labels)
    got, = torch.autograd.grad([r.top_logprobs, r.logprobs, r.entropy], x, [g_top, g_lp, g_en])
    assert got.dtype == dtype and got.shape == x.shape
    ids = torch.cat([labels[:, None].long(), order(z, k)], 1)
    _, _, ref, size = reference(z, ids, torch.cat([g_lp[:, None], g_top], 1), g_en)
    check_grad(got, ref, size, dtype)


@pytest.mark.parametrize("n,v,k,dtype,layout,ids_dtype", [
    (1, 1, 1, torch.float32, "plain", torch.int64),
    (4, 33, 40, torch.bfloat16, "shifted", torch.int32),  # more ids than tokens: repeats
    (3, 1000, 512, torch.float32, "plain", torch.int64),
    (50, 32768, 16, torch.bfloat16, "strided", torch.int64),
    (187, 151936, 8, torch.bfloat16, "plain", torch.int32),
    (1600, 777, 20, torch.float32, "plain", torch.int64),
])
def test_given_tokens(n, v, k, dtype, layout, ids_dtype):
    z = logits_of("random", n, v, dtype, n + 7 * v)
    g = gen(v)
    ids = torch.randint(-2, v + 2, (n, k), generator=g, device="cuda").clamp(max=v + 1).to(ids_dtype)
    if v > 2:
        ids[0, 0], ids[0, -1] = v - 1, v - 1
    g_ids, g_en = torch.randn(n, k, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    lp, ent, ref, size = reference(z, ids, g_ids, g_en)
    for inplace in (False, True):
        x = laid_out(z.clone(), layout).requires_grad_(True)
        got_lp, got_ent = token_logprobs_from_logits(x, ids, inplace_backward=inplace)
        assert (got_lp.double() - lp).abs().max() <= LP_TOL and (got_ent.double() - ent).abs().max() <= ENT_TOL
        got, = torch.autograd.grad([got_lp, got_ent], x, [g_ids, g_en])
        assert (got.data_ptr() == x.data_ptr()) == inplace
        check_grad(got, ref, size, dtype)
        if inplace and layout == "strided":  # what lies between the rows is left as it was
            assert (x.detach().as_strided((n, v + 5), (v + 5, 1))[:-1, v:] == 99.0).all()


def test_gradients_agree_with_differences():
    n, v, k = 3, 40, 6
    g = gen(1)
    z = torch.randn(n, v, generator=g, device="cuda")
    ids = torch.randint(0, v, (n, k), generator=g, device="cuda")
    w, we = torch.randn(n, k, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    x = z.clone().requires_grad_(True)
    lp, ent = token_logprobs_from_logits(x, ids)
    grad, = torch.autograd.grad((lp * w).sum() + (ent * we).sum(), x)

    def value(zz):
        a, b = reference(zz, ids)
        return ((a * w).sum() + (b * we).sum()).item()

    for t, j in ((0, 0), (0, int(ids[0, 0])), (1, 7), (2, 39), (2, int(ids[2, 3]))):
        h = 1e-5
        up, down = z.double().clone(), z.double().clone()
        up[t, j] += h
        down[t, j] -= h
        # the difference's own error is h^2 times a third derivative, and 1e-16 * |value| / h
        assert abs((value(up) - value(down)) / (2 * h) - grad[t, j].item()) <= 1e-4


def test_one_gradient_at_a_time_and_leading_dimensions():
    z = logits_of("random", 6, 500, torch.float32, 8)
    x = z.view(2, 3, 500).clone().requires_grad_(True)
    r = top_logprobs_from_logits(x, 4, torch.zeros(2, 3, dtype=torch.int64, device="cuda"))
    assert r.top_ids.shape == (2, 3, 4) and r.logprobs.shape == r.entropy.shape == (2, 3)
    assert not r.top_ids.requires_grad and r.top_logprobs.requires_grad
    ids, none = order(z, 4), torch.zeros(6, 4, device="cuda")
    zero = torch.zeros(6, device="cuda")
    one, = torch.autograd.grad(r.top_logprobs.sum(), x, retain_graph=True)
    _, _, ref, size = reference(z, ids, none + 1, zero)
    check_grad(one.view(6, 500), ref, size, torch.float32)
    one, = torch.autograd.grad(r.entropy.sum(), x, retain_graph=True)
    _, _, ref, size = reference(z, ids, none, zero + 1)
    check_grad(one.view(6, 500), ref, size, torch.float32)
    one, = torch.autograd.grad(r.logprobs.sum(), x)
    _, _, ref, size = reference(z, torch.zeros(6, 1, dtype=torch.int64, device="cuda"), zero[:, None] + 1, zero)
    check_grad(one.view(6, 500), ref, size, torch.float32)


def test_agrees_with_the_operator_for_one_label():
    """One given token per position is what logprobs_and_entropy_from_logits computes; the two read a row in the same
    order, and differ by the roundings of LP_TOL at most."""
    z = logits_of("random", 33, 5000, torch.bfloat16, 2)
    lab = torch.randint(0, 5000, (33,), generator=gen(3), device="cuda")
    a, b = logprobs_and_entropy_from_logits(z, lab), token_logprobs_from_logits(z, lab[:, None])
    assert (a[0] - b[0][:, 0]).abs().max() <= LP_TOL and (a[1] - b[1]).abs().max() <= ENT_TOL


def test_expanded_rows_and_empty_batches():
    row = logits_of("random", 1, 700, torch.float32, 4)
    x = row.clone().requires_grad_(True)
    r = top_logprobs_from_logits(x.expand(5, 700), 3, inplace_backward=True)
    assert torch.equal(r.top_ids, order(row, 3).expand(5, 3))
    got, = torch.autograd.grad(r.top_logprobs.sum(), x)
    _, _, ref, size = reference(row, order(row, 3), torch.full((1, 3), 5.0, device="cuda"), torch.zeros(1, device="cuda"))
    check_grad(got, ref, size, torch.float32)
    e = torch.empty(0, 700, device="cuda", requires_grad=True)
    r = top_logprobs_from_logits(e, 3, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert r.top_ids.shape == (0, 3) and r.logprobs.shape == (0,)
    lp, ent = token_logprobs_from_logits(e, torch.empty(0, 2, dtype=torch.int64, device="cuda"))
    assert lp.shape == (0, 2)
    assert torch.autograd.grad(lp.sum() + ent.sum(), e)[0].shape == (0, 700)


def test_an_inplace_backward_runs_once():
    x = logits_of("random", 3, 300, torch.float32, 1).requires_grad_(True)
    lp, _ = token_logprobs_from_logits(x, torch.zeros(3, 1, dtype=torch.int64, device="cuda"), inplace_backward=True)
    torch.autograd.grad(lp.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="inplace_backward"):
        torch.autograd.grad(lp.sum(), x)


def test_results_repeat_bit_for_bit():
    z = logits_of("random", 40, 50257, torch.bfloat16, 6)
    ids = torch.randint(0, 3, (40, 64), generator=gen(2), device="cuda")  # many repeats
    g_ids, g_en = torch.randn(40, 64, generator=gen(3), device="cuda"), torch.randn(40, generator=gen(4), device="cuda")

    def once():
        x = z.clone().requires_grad_(True)
        lp, ent = token_logprobs_from_logits(x, ids)
        r = top_logprobs_from_logits(z, 64)
        return [lp.detach(), ent.detach(), r.top_logprobs, r.top_ids,
                torch.autograd.grad([lp, ent], x, [g_ids, g_en])[0]]

    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    """Forward and backward as a graph, replayed on other inputs with eager work between the replays."""
    n, v, k = 30, 32768, 12
    z = torch.empty(n, v, device="cuda", dtype=torch.bfloat16)
    g_top, g_en = torch.randn(n, k, generator=gen(1), device="cuda"), torch.randn(n, generator=gen(2), device="cuda")

    def step():
        r = top_logprobs_from_logits(z, k)
        grad, = torch.autograd.grad([r.top_logprobs, r.entropy], z, [g_top, g_en])
        return r.top_logprobs.detach(), r.entropy.detach(), r.top_ids, grad

    z.copy_(logits_of("random", n, v, torch.bfloat16, 1))
    z.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (2, 3, 4):
        with torch.no_grad():
            z.copy_(logits_of("few_values" if seed == 3 else "random", n, v, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_on_another_stream():
    z = logits_of("random", 64, 50257, torch.bfloat16, 9)
    want = top_logprobs_from_logits(z, 10)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = top_logprobs_from_logits(z, 10)
    side.synchronize()
    assert torch.equal(got.top_ids, want.top_ids) and torch.equal(got.top_logprobs, want.top_logprobs)


def test_saved_tensors_from_a_hook_are_looked_at_again():
    """A hook that hands back tensors in host memory, or others than were saved, refuses the backward: nothing is launched."""
    z = logits_of("random", 3, 300, torch.float32, 2)

    def backward_with(unpack):
        x = z.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            r = top_logprobs_from_logits(x, 3, torch.zeros(3, dtype=torch.int64, device="cuda"))
        return torch.autograd.grad(r.top_logprobs.sum() + r.logprobs.sum(), x)[0]

    want = backward_with(lambda t: t)
    assert torch.equal(backward_with(lambda t: t.clone()), want)
    for unpack in (lambda t: t.cpu(), lambda t: t.cpu() if t.dim() == 1 else t, lambda t: t.cpu() if t.dtype == torch.int64 else t,
                   lambda t: t[:2] if t.dim() == 2 else t, lambda t: t[:1] if t.dim() == 1 else t):
        with pytest.raises(RuntimeError):
            backward_with(unpack)


def test_a_gradient_is_not_differentiated_again():
    x = logits_of("random", 3, 300, torch.float32, 2).requires_grad_(True)
    lp, _ = token_logprobs_from_logits(x, torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
    g, = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):  # a penalty on the gradient is no constant
        (lp.sum() + g.square().sum()).backward()
    with pytest.raises(RuntimeError, match="second time|freed"):
        lp2, _ = token_logprobs_from_logits(x, torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
        torch.autograd.grad(lp2.sum(), x)
        torch.autograd.grad(lp2.sum(), x)


def test_a_logit_changed_before_the_backward_is_noticed():
    x = logits_of("random", 3, 300, torch.float32, 2).requires_grad_(True)
    y = x * 1
    lp, _ = token_logprobs_from_logits(y, torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(lp.sum(), x)


def test_two_streams_at_once():
    """Batches of few rows, whose rows several workgroups share: calls that overlap on two streams, and calls of other shapes in
    between, leave each other's counters alone."""
    zs = [logits_of("random", n, v, torch.bfloat16, n) for n, v in ((3, 151936), (70, 50257), (300, 32768), (1, 151936))]
    ids = [torch.randint(0, z.shape[1], (z.shape[0], 4), generator=gen(i), device="cuda") for i, z in enumerate(zs)]
    want = [(top_logprobs_from_logits(z, 9), token_logprobs_from_logits(z, i)) for z, i in zip(zs, ids)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for s, out in zip(streams, got):
            with torch.cuda.stream(s):
                out.append([(top_logprobs_from_logits(z, 9), token_logprobs_from_logits(z, i)) for z, i in zip(zs, ids)])
    torch.cuda.synchronize()
    for out in got[0] + got[1]:
        for (a, b), (c, d) in zip(out, want):
            assert torch.equal(a.top_ids, c.top_ids) and torch.equal(a.top_logprobs, c.top_logprobs) and torch.equal(a.entropy, c.entropy)
            assert torch.equal(b[0], d[0]) and torch.equal(b[1], d[1])


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    z = logits_of("random", 2, 50, torch.float32, 1)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            top_logprobs_from_logits(fwd.make_dual(z, torch.ones_like(z)), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_vocabulary_of_one_token_in_any_layout(dtype):
    """Its stride says nothing: a column of a matrix, a transposed row."""
    wide = torch.randn(5, 7, device="cuda", generator=gen(1)).to(dtype)
    for z in (wide[:, :1], wide[:1, :5].t(), wide[:, 3:4], wide.t()[:5, 2:3]):
        x = z.detach().requires_grad_(True)
        r = top_logprobs_from_logits(x, 1, torch.zeros(5, dtype=torch.int64, device="cuda"))
        lp, ent = token_logprobs_from_logits(x, torch.tensor([[0, 1]], device="cuda").expand(5, 2))
        assert not any(t.any() for t in (r.top_ids, r.top_logprobs, r.logprobs, r.entropy, lp, ent))
        grad, = torch.autograd.grad([r.top_logprobs.sum() + r.logprobs.sum() + lp.sum() + ent.sum()], x)
        assert grad.shape == (5, 1) and grad.dtype == dtype and not grad.any()
