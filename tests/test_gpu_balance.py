"""The router's balance loss, the experts' loads and the gradient, against the same in 64 bits."""

import math

import pytest
import torch

from axon_amd.models.fsdp_models import CausalLM
from axon_amd.protocol import DataProto
from axon_amd.trainer.algos.loss import router_balance_loss

pytestmark = pytest.mark.gpu

# A score is off by the rounding of its exponential's argument (twice 40 * 2^-24, |logit| <= 20), by the exponential
# (2^-22), a sum and a division: 6e-6.  Sums over tokens add chains of at most 256 roundings of 2^-24 (1.5e-5 at the worst).
REL = 2.5e-5


def case(layers, n, e, k, dtype, seed, mask=None, pattern="random"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xs = []
    for _ in range(layers):
        x = 2 * torch.randn(n, e, generator=g, device="cuda") + torch.randn(e, generator=g, device="cuda")
        if pattern == "ties":
            x = torch.randint(-1, 2, (n, e), generator=g, device="cuda").float()
        elif pattern == "constant":
            x = torch.zeros_like(x)
        elif pattern == "closed":  # experts that the router may not choose
            x[:, ::3] = -math.inf
        xs.append(x.clamp(-math.inf, 20).to(dtype))
    m = None
    if mask is not None:
        m = (torch.rand(n, generator=g, device="cuda") < 0.6)
        m = m.to(mask)
    return xs, m, g


def reference(xs, k, mask, cu, ids, score):
    n, e = xs[0].shape
    keep = torch.ones(n, dtype=torch.bool, device="cuda") if mask is None else mask != 0
    bounds = [0, n] if cu is None else cu.tolist()
    spans = [(a, b) for a, b in zip(bounds[:-1], bounds[1:]) if b > a and keep[a:b].any()]
    inside = torch.zeros(n, dtype=torch.bool, device="cuda")
    if bounds[-1] > bounds[0]:
        inside[bounds[0]:bounds[-1]] = True
    loss, counts, grads, sizes = 0.0, [], [], []
    for i, x in enumerate(xs):
        x = x.double()
        s = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
        p = s if score == "softmax" else s / s.sum(1, keepdim=True)
        chosen = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :k] if ids is None else ids[i].long()
        ok = (chosen >= 0) & (chosen < e)
        hit = torch.zeros_like(x).scatter_add_(1, torch.where(ok, chosen, 0), ok.double()) * (keep & inside)[:, None]
        counts.append(hit.sum(0).long())
        grad, size = torch.zeros_like(x), torch.zeros_like(x)
        for a, b in spans:
            t = float(keep[a:b].sum())
            w = hit[a:b].sum(0) * e / (k * t * t) / (len(spans) * len(xs))
            loss += (w * (p[a:b] * keep[a:b, None]).sum(0)).sum().item()
            dot = (p[a:b] * w).sum(1, keepdim=True)
            # 1 - sigmoid(x) = sigmoid(-x): the difference cancels in 64 bits too (0 from x = 37 on)
            slope = p[a:b] * (1 if score == "softmax" else torch.sigmoid(-x[a:b])) * keep[a:b, None]
            grad[a:b], size[a:b] = slope * (w - dot), slope * (w + dot)
        grads.append(grad)
        sizes.append(size)
    return loss, torch.stack(counts), grads, sizes


def check(xs, k, *, mask=None, cu=None, ids=None, score="softmax", stacked=False, up=0.3):
    loss_ref, counts_ref, grads_ref, sizes = reference(xs, k, mask, cu, ids, score)
    leaves = [torch.stack(xs).requires_grad_(True)] if stacked else [x.requires_grad_(True) for x in xs]
    loss, counts = router_balance_loss(leaves[0] if stacked else leaves, k, token_mask=mask, cu_seqlens=cu, expert_ids=ids,
                                       score_fn=score)
    assert counts.dtype == torch.int64 and torch.equal(counts, counts_ref)
    assert loss.dtype == torch.float32 and abs(loss.item() - loss_ref) <= 2 * REL * abs(loss_ref)
    got = torch.autograd.grad(loss, leaves, torch.tensor(up, device="cuda"))
    got = list(got[0].unbind(0)) if stacked else got
    for d, ref, size, x in zip(got, grads_ref, sizes, xs):
        assert d.dtype == x.dtype and d.shape == x.shape
        bound = 3 * REL * up * size + 1e-30
        if d.dtype == torch.bfloat16:
            bound = bound + 2.0 ** -8 * up * ref.abs() + 1e-38
        assert ((d.double() - up * ref).abs() <= bound).all()


CASES = [
    # layers, tokens, experts, k, dtype, mask, score, pattern
    (1, 1, 1, 1, torch.float32, None, "softmax", "random"),
    (2, 3, 5, 2, torch.bfloat16, None, "sigmoid", "random"),
    (1, 257, 8, 2, torch.float32, torch.int64, "softmax", "random"),
    (3, 100, 16, 16, torch.bfloat16, torch.float32, "softmax", "ties"),
    (2, 513, 32, 4, torch.float32, torch.bool, "sigmoid", "ties"),
    (1, 1021, 60, 4, torch.bfloat16, torch.int64, "softmax", "random"),
    (4, 300, 64, 6, torch.float32, None, "sigmoid", "closed"),
    (2, 777, 128, 8, torch.bfloat16, torch.float32, "softmax", "ties"),
    (1, 300, 129, 3, torch.float32, None, "softmax", "random"),
    (2, 64, 160, 6, torch.bfloat16, None, "sigmoid", "random"),
    (1, 333, 256, 8, torch.float32, torch.int32, "softmax", "closed"),
    (1, 100, 511, 10, torch.bfloat16, None, "softmax", "random"),
    (2, 50, 1000, 32, torch.float32, torch.int64, "sigmoid", "ties"),
    (1, 40, 1024, 1, torch.bfloat16, None, "softmax", "constant"),
    (70, 40, 12, 3, torch.bfloat16, torch.int64, "softmax", "random"),  # more layers than a launch takes
    (3, 6000, 128, 8, torch.bfloat16, None, "softmax", "random"),
]


@pytest.mark.parametrize("layers,n,e,k,dtype,mask,score,pattern", CASES)
def test_batch(layers, n, e, k, dtype, mask, score, pattern):
    xs, m, _ = case(layers, n, e, k, dtype, n + e, mask, pattern)
    check(xs, k, mask=m, score=score, stacked=layers > 1 and n % 2 == 0)


@pytest.mark.parametrize("lens", [[7], [1, 1, 1, 300, 1, 40], [0, 5, 0, 0, 260, 31, 0], [256, 256], [255, 2, 255], [3] * 120])
@pytest.mark.parametrize("layers,e,k,dtype,score", [(2, 60, 4, torch.bfloat16, "softmax"), (1, 256, 8, torch.float32, "sigmoid")])
def test_sequences(lens, layers, e, k, dtype, score):
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    n = sum(lens) + 5  # the last five tokens belong to no sequence
    xs, m, _ = case(layers, n, e, k, dtype, n, torch.int64)
    m[: lens[0]] = 0  # a sequence without tokens that count
    check(xs, k, mask=m, cu=cu, score=score)
    check([x.detach() for x in xs], k, cu=cu, score=score)


def test_tokens_before_the_first_sequence():
    """They belong to none, like those behind the last."""
    xs, m, _ = case(2, 700, 24, 3, torch.float32, 8, torch.int64)
    cu = torch.tensor([290, 300, 300, 690], dtype=torch.int32, device="cuda")
    check(xs, 3, mask=m, cu=cu)


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_given_choices(ids_dtype):
    xs, m, g = case(3, 300, 64, 6, torch.bfloat16, 5, torch.float32)
    ids = [torch.randint(-1, 65, (300, 6), generator=g, device="cuda").to(ids_dtype) for _ in xs]
    cu = torch.tensor([0, 100, 290], dtype=torch.int32, device="cuda")
    check(xs, 6, mask=m, ids=ids)
    check([x.detach() for x in xs], 6, mask=m, ids=ids, cu=cu, score="sigmoid")
    a = router_balance_loss(torch.stack([x.detach() for x in xs]), 6, expert_ids=torch.stack(ids))
    b = router_balance_loss([x.detach() for x in xs], 6, expert_ids=ids)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_uniform_scores_have_loss_one():
    """Equal scores and equally many choices: sum_e E / (k T) (k T / E) (1 / E) = 1."""
    x = torch.zeros(64, 16, device="cuda")
    ids = (torch.arange(64, device="cuda")[:, None] * 4 + torch.arange(4, device="cuda")) % 16
    loss, counts = router_balance_loss(x, 4, expert_ids=ids)
    assert abs(loss.item() - 1) <= REL and counts.shape == (16,) and (counts == 16).all()


def test_agrees_with_differences():
    xs, m, g = case(2, 20, 12, 3, torch.float32, 1, torch.int64)
    ids = [torch.randint(0, 12, (20, 3), generator=g, device="cuda") for _ in xs]
    for score in ("softmax", "sigmoid"):
        leaves = [x.clone().requires_grad_(True) for x in xs]
        loss, _ = router_balance_loss(leaves, 3, token_mask=m, expert_ids=ids, score_fn=score)
        grads = torch.autograd.grad(loss, leaves)
        for t, e in ((0, 0), (5, 11), (int(m.nonzero()[0]), 4)):
            h = 1e-5
            pair = []
            for sign in (h, -h):
                moved = [x.double().clone() for x in xs]
                moved[1][t, e] += sign
                pair.append(reference(moved, 3, m, None, ids, score)[0])
            # h^2 times a third derivative, and 1e-16 / h of the loss
            assert abs((pair[0] - pair[1]) / (2 * h) - grads[1][t, e].item()) <= 1e-7


def test_masked_rows_do_not_matter():
    """NaN and infinities where the mask is zero change nothing, and their gradient is zero."""
    xs, m, _ = case(1, 90, 24, 4, torch.float32, 3, torch.int64)
    want = router_balance_loss(xs, 4, token_mask=m)
    bad = xs[0].clone()
    off = (m == 0).nonzero().flatten()
    bad[off[0]], bad[off[1]], bad[off[2]] = math.nan, math.inf, -math.inf
    bad.requires_grad_(True)
    got = router_balance_loss(bad, 4, token_mask=m)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1][0])
    d, = torch.autograd.grad(got[0], bad)
    assert torch.isfinite(d).all() and not d[off].any()
    nothing = router_balance_loss(bad, 4, token_mask=torch.zeros_like(m))
    assert nothing[0].item() == 0 and not nothing[1].any()
    d, = torch.autograd.grad(nothing[0], bad)
    assert not d.any()
    empty = torch.empty(0, 24, device="cuda", requires_grad=True)
    loss, counts = router_balance_loss([empty], 4)
    assert loss.item() == 0 and not counts.any() and torch.autograd.grad(loss, empty)[0].shape == (0, 24)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = xs[0].clone().requires_grad_(True)
    loss, counts = router_balance_loss(x, 4, cu_seqlens=none)
    assert loss.item() == 0 and not counts.any() and not torch.autograd.grad(loss, x)[0].any()


def test_layouts_and_partial_gradients():
    n, e, k = 130, 40, 4
    xs, _, _ = case(3, n, e, k, torch.bfloat16, 9)
    want_loss, want_counts = router_balance_loss(xs, k)
    wide = torch.zeros(n, e + 3, device="cuda", dtype=torch.bfloat16)  # odd strides, odd starts
    views = []
    for x in xs:
        buf = wide.clone()
        buf[:, 1:1 + e] = x
        views.append(buf[:, 1:1 + e])
    for form in (views, [x.view(10, 13, e) for x in xs], [x.t().contiguous().t() for x in xs], torch.stack(xs)):
        loss, counts = router_balance_loss(form, k)
        assert torch.equal(loss, want_loss) and torch.equal(counts, want_counts)
    a, b, c = (x.clone().requires_grad_(r) for x, r in zip(xs, (True, False, True)))
    loss, _ = router_balance_loss([a, b, c], k)
    loss.backward()
    assert b.grad is None and a.grad is not None and c.grad is not None
    full = [x.clone().requires_grad_(True) for x in xs]
    router_balance_loss(full, k)[0].backward()
    assert torch.equal(full[0].grad, a.grad) and torch.equal(full[2].grad, c.grad)
    same = xs[0].clone().requires_grad_(True)  # one tensor for two layers: its gradients add up
    loss, _ = router_balance_loss([same, same], k)
    d, = torch.autograd.grad(loss, same)
    one = xs[0].clone().requires_grad_(True)
    d1, = torch.autograd.grad(router_balance_loss(one, k)[0], one)
    # halves of bf16 numbers are exact, and so is their sum
    assert torch.equal(d, d1)


def test_results_repeat_and_replay():
    xs, m, _ = case(2, 900, 64, 6, torch.bfloat16, 2, torch.float32)
    cu = torch.tensor([0, 200, 201, 900], dtype=torch.int32, device="cuda")
    xs = [x.requires_grad_(True) for x in xs]
    up = torch.ones((), device="cuda")

    def step():
        loss, counts = router_balance_loss(xs, 6, token_mask=m, cu_seqlens=cu)
        return [loss.detach(), counts, *torch.autograd.grad(loss, xs, up)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (4, 5, 6):
        with torch.no_grad():
            for x, y in zip(xs, case(2, 900, 64, 6, torch.bfloat16, seed)[0]):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for _ in range(2):
            for a, b in zip(held, step()):
                assert torch.equal(a, b)


@pytest.mark.parametrize("padded", [False, True])
def test_as_a_term_of_the_trainers_loss(padded):
    n, e, k = 240, 16, 2
    g = torch.Generator(device="cuda").manual_seed(4)
    xs, _, _ = case(2, n, e, k, torch.float32, 6)
    shape = (4, 60) if padded else (n,)
    rand = lambda: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    att = (torch.rand(*shape, generator=g, device="cuda") < 0.8).long()
    lp, ent, old, adv = rand(), rand().abs(), rand(), rand()
    cu = None if padded else torch.tensor([0, 100, 180, 240], dtype=torch.int32, device="cuda")
    seqs = torch.tensor([0, 60, 120, 180, 240], dtype=torch.int32, device="cuda") if padded else cu

    def run(args, router):
        data = DataProto.from_dict(tensors={"old_log_probs": old, "advantages": adv, "response_mask": torch.ones(*shape, device="cuda"),
                                            **({"attention_mask": att} if padded else {})},
                                   meta_info={} if padded else {"cu_seqlens": cu})
        meta = {"loss_fn": "ppo", "loss_fn_args": args, "dp_replicas": 2, "n_micro_batches": 4, "temperature": 1.0}
        module = lambda inputs, m: {"log_probs": lp, "entropys": ent, **({"router_logits": router} if router else {})}  # noqa: E731
        return CausalLM.forward_backward_fn(module, data, meta)

    plain, metrics = run({}, None)
    assert not any("router" in key for key in metrics)
    leaves = [x.clone().requires_grad_(True) for x in xs]
    args = {"router_aux_loss_coef": 0.01, "router_top_k": k, "router_balance_per_sequence": True, "router_score_fn": "sigmoid"}
    loss, metrics = run(args, leaves)
    mask = att if padded else None
    want, counts = router_balance_loss(xs, k, token_mask=mask, cu_seqlens=seqs, score_fn="sigmoid")
    # the mean over four micro-batches of two replicas, whose gradients are added and averaged: a quarter of the coefficient
    # three roundings of fp32 numbers of the losses' size
    assert abs(loss.item() - plain.item() - 0.01 / 4 * want.item()) <= 4 * 2.0 ** -24 * (abs(plain.item()) + abs(loss.item()) + 1)
    assert metrics["router_balance_loss"] == want.item() and metrics["router_aux_loss_coef"] == 0.01
    load = (counts.amax(1) / counts.double().mean(1)).max().item()
    assert abs(metrics["router_max_load"] - load) <= 4 * 2.0 ** -24 * load
    got = torch.autograd.grad(loss, leaves)
    ref = reference(xs, k, mask.reshape(-1) if padded else None, seqs, None, "sigmoid")
    for d, r, size in zip(got, ref[2], ref[3]):
        assert ((d.double() - 0.0025 * r).abs() <= 3 * REL * 0.0025 * size + 1e-30).all()
    with pytest.raises(ValueError, match="router_logits"):
        run(args, None)
    with pytest.raises(ValueError, match="router_top_k"):
        run({"router_aux_loss_coef": 0.01}, leaves)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("e", [6, 64, 300, 700])
def test_rows_far_from_zero(e, dtype):
    """Rows that a mask of a large number or of the type's lowest has left nothing of, and rows of vanishing sigmoids: the
    differences from a row's largest logit are those of other rows."""
    lowest, k = torch.finfo(dtype).min, 4
    x, _, g = case(1, 41, e, k, torch.float32, e)
    x = x[0]
    x[0], x[1], x[2], x[3] = -1e9, lowest, x[2] * 1000 - 1e12, x[3] + 50000
    x[4, : e - 2] = lowest
    x[5], x[6, ::2] = torch.finfo(dtype).max, -1e9
    check([x.to(dtype)], k)
    y = 2 * torch.randn(41, e, generator=g, device="cuda")
    y[0] -= 100  # beyond what 32 bits hold of a sigmoid
    y[1] -= 600
    y[2, 1:] = lowest
    y[2, 0] = -95
    y[3] += 50
    y[4, ::2] -= 90
    y[5] = -62.5
    check([y.to(dtype)], k, score="sigmoid")


def test_offsets_beyond_32_bits():
    xs, _, _ = case(1, 3, 16, 2, torch.bfloat16, 5)
    buf = torch.empty(2 ** 31 + 5000, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((3, 16), (2 ** 30 + 8, 1))
    far.copy_(xs[0])
    check([far.detach()], 2)


def test_a_saved_tensor_of_another_type_is_refused():
    xs, m, _ = case(2, 30, 16, 2, torch.float32, 3, torch.int64)
    leaves = [x.clone().requires_grad_(True) for x in xs]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.int() if t.dtype == torch.int64 else t):
        loss, _ = router_balance_loss(leaves, 2, token_mask=m)
    with pytest.raises(RuntimeError, match="another type"):
        torch.autograd.grad(loss, leaves)


def test_padded_rows_of_another_length_than_the_outputs():
    """Router logits of whole rows beside outputs of their responses: sequences are rows of the router logits."""
    x, _, _ = case(1, 240, 16, 2, torch.float32, 6)
    lp = torch.randn(4, 20, device="cuda")
    ones = torch.ones(4, 20, device="cuda")
    meta = {"loss_fn": "ppo", "dp_replicas": 1, "temperature": 1.0,
            "loss_fn_args": {"router_aux_loss_coef": 0.1, "router_top_k": 2, "router_balance_per_sequence": True}}

    def run(router):
        data = DataProto.from_dict(tensors={"old_log_probs": lp, "advantages": lp, "response_mask": ones})
        module = lambda inputs, m: {"log_probs": lp, "entropys": ones, "router_logits": router}  # noqa: E731
        return CausalLM.forward_backward_fn(module, data, meta)[1]["router_balance_loss"]

    cu = torch.arange(5, dtype=torch.int32, device="cuda") * 60
    want = router_balance_loss(x, 2, cu_seqlens=cu)[0].item()
    for router in (x, x[0], torch.stack(x), (x[0].view(4, 60, 16),)):
        assert run(router) == want
    with pytest.raises(ValueError, match="rows of one length"):
        run([x[0][:239]])


def test_saved_tensors_from_a_hook_are_looked_at_again():
    xs, m, _ = case(2, 30, 16, 2, torch.float32, 3, torch.int64)
    cu = torch.tensor([0, 10, 30], dtype=torch.int32, device="cuda")

    def backward_with(unpack):
        leaves = [x.clone().requires_grad_(True) for x in xs]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            loss, _ = router_balance_loss(leaves, 2, token_mask=m, cu_seqlens=cu)
        return torch.autograd.grad(loss, leaves)

    want = backward_with(lambda t: t)
    odd = lambda t: torch.cat([t, t], 1)[:, : t.shape[1]] if t.dim() == 2 else t  # noqa: E731  (another row stride)
    for same in (backward_with(lambda t: t.clone()), backward_with(odd)):
        assert all(torch.equal(a, b) for a, b in zip(same, want))
    for unpack in (lambda t: t.cpu(), lambda t: t.cpu() if t.dim() == 1 else t, lambda t: t.cpu() if t.dim() == 3 else t,
                   lambda t: t[:20] if t.dim() == 2 else t, lambda t: t[:2] if t.dtype == torch.int32 else t):
        with pytest.raises(RuntimeError):
            backward_with(unpack)


@pytest.mark.parametrize("bits", [0x7FFF, 0x7FC0, 0x7F81, 0x7F80, 0xFFFF, 0xFFC0, 0xFF81, 0xFF80])
@pytest.mark.parametrize("e,k", [(6, 2), (60, 4), (128, 8), (700, 3)])
def test_masked_rows_of_any_bf16_pattern_do_not_matter(e, k, bits):
    """NaN of every kind and infinities at expert 0 and elsewhere in rows that the mask leaves out, the first of a run among them:
    the results are those of zeros there, bit for bit."""
    xs, _, _ = case(2, 75, e, k, torch.bfloat16, e)
    cu = torch.tensor([0, 33, 75], dtype=torch.int32, device="cuda")
    mask = torch.ones(75, dtype=torch.int64, device="cuda")
    off = torch.tensor([0, 33, 34, 74], device="cuda")
    mask[off] = 0
    odd = torch.tensor([bits], dtype=torch.int32, device="cuda").to(torch.int16).view(torch.bfloat16)
    clean, bad = [], []
    for x in xs:
        y = x.clone()
        y[off] = 0
        z = y.clone()
        z[off, 0] = odd
        z[33] = odd
        z[34, e - 1] = odd
        clean.append(y.requires_grad_(True))
        bad.append(z.requires_grad_(True))
    for score in ("softmax", "sigmoid"):
        for seqs in (None, cu):
            want, got = (router_balance_loss(x, k, token_mask=mask, cu_seqlens=seqs, score_fn=score) for x in (clean, bad))
            assert torch.equal(got[1], want[1]) and got[1].sum().item() == 2 * 71 * k
            assert torch.equal(got[0], want[0])
            for a, b in zip(torch.autograd.grad(got[0], bad), torch.autograd.grad(want[0], clean)):
                assert torch.equal(a, b) and not a[off].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("e,k", [(3, 2), (60, 4), (128, 128), (700, 9)])
def test_a_nan_counts_as_the_lowest_for_the_choices(e, k, dtype):
    """In rows that count, whatever its sign and its bits: as -inf, equal ones by ascending expert; the loss is then NaN."""
    g = torch.Generator(device="cuda").manual_seed(e)
    x = torch.randint(-2, 3, (40, e), generator=g, device="cuda").to(dtype)
    word, bits = (torch.int16, (0x7FFF, 0x7FC0, 0x7F81, -1, -0x40, -0x7F)) if dtype == torch.bfloat16 else (
        torch.int32, (0x7FFFFFFF, 0x7FC00000, 0x7F800001, -1, -0x400000, -0x7FFFFF))
    for i, b in enumerate(bits):
        odd = torch.tensor([b], dtype=word, device="cuda").view(dtype)
        assert torch.isnan(odd).all()
        x[i, : e - i % 2] = odd  # all of a row, and all but its last
        x[10 + i, i % e] = odd
        x[20 + i, ::2] = odd
    x[30, ::2], x[31] = -math.inf, math.inf
    loss, counts = router_balance_loss(x, k)
    low = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    chosen = torch.sort(low.double(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(counts, torch.bincount(chosen.flatten(), minlength=e)) and torch.isnan(loss)


@pytest.mark.parametrize("n,e", [(130, 40), (7, 3), (1, 1)])
def test_every_layers_gradient_has_its_own_storage(n, e):
    """What is kept, saved or resized of one layer's gradient is that layer's alone."""
    xs, _, _ = case(4, n, e, 1, torch.bfloat16, 9)
    xs = [x.requires_grad_(i != 2) for i, x in enumerate(xs)]
    router_balance_loss(xs, 1)[0].backward()
    grads = [x.grad for x in xs if x.grad is not None]
    assert len(grads) == 3
    for d in grads:
        assert d.untyped_storage().nbytes() == n * e * 2 and d.storage_offset() == 0 and d.is_contiguous()
    assert len({d.untyped_storage().data_ptr() for d in grads}) == 3
    kept = [d.clone() for d in grads]
    grads[0].add_(1)
    grads[1].untyped_storage().resize_(0)
    assert torch.equal(grads[2], kept[2]) and torch.equal(grads[0], kept[0] + 1)


@pytest.mark.parametrize("per_sequence", [False, True])
@pytest.mark.parametrize("keep", [0.7, 0.05])
def test_packed_routers_beside_a_padded_batch(per_sequence, keep):
    """Remove-padding: the routers saw the tokens that attention_mask keeps, the batch and its outputs are padded."""
    rows, length, e, k = 5, 60, 16, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    att = (torch.rand(rows, length, generator=g, device="cuda") < keep).long()
    att[2] = 0  # a row of which nothing is left
    att[0, 0] = 1
    n = int(att.sum())
    xs, _, _ = case(2, n, e, k, torch.float32, 6)
    lp = torch.randn(rows, length, generator=g, device="cuda")
    args = {"router_aux_loss_coef": 0.1, "router_top_k": k, "router_balance_per_sequence": per_sequence}

    def run(router):
        data = DataProto.from_dict(tensors={"old_log_probs": lp, "advantages": lp, "response_mask": torch.ones_like(lp),
                                            "attention_mask": att})
        meta = {"loss_fn": "ppo", "loss_fn_args": args, "dp_replicas": 1, "temperature": 1.0}
        module = lambda inputs, m: {"log_probs": lp, "entropys": lp.abs(), "router_logits": router}  # noqa: E731
        return CausalLM.forward_backward_fn(module, data, meta)

    leaves = [x.clone().requires_grad_(True) for x in xs]
    loss, metrics = run(leaves)
    cu = torch.nn.functional.pad(att.sum(1).cumsum(0), (1, 0)).int() if per_sequence else None
    want, counts = router_balance_loss(xs, k, cu_seqlens=cu)
    load = (counts.amax(1) / counts.double().mean(1)).max().item()
    assert metrics["router_balance_loss"] == want.item() and abs(metrics["router_max_load"] - load) <= 4 * 2.0 ** -24 * load
    ref = reference(xs, k, None, cu, None, "softmax")
    for d, r, size in zip(torch.autograd.grad(loss, leaves), ref[2], ref[3]):
        assert ((d.double() - 0.1 * r).abs() <= 3 * REL * 0.1 * size + 1e-30).all()
    assert run(torch.stack(xs))[1]["router_balance_loss"] == want.item()
    for wrong in ([x[:-1] for x in xs], [torch.cat([x, x[:1]]) for x in xs]):
        with pytest.raises(ValueError, match="attention_mask"):
            run(wrong)
    with pytest.raises(ValueError):  # more tokens than the batch has entries
        run([torch.zeros(rows * length + 1, e, device="cuda")])
    whole = [torch.randn(rows, length, e, generator=g, device="cuda")]
    att_loss = router_balance_loss(whole, k, token_mask=att,
                                   cu_seqlens=torch.arange(rows + 1, dtype=torch.int32, device="cuda") * length if per_sequence else None)[0]
    assert run(whole)[1]["router_balance_loss"] == att_loss.item()
