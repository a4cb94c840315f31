"""Controls of logits where an index, a sum or an arrangement is at its limit, against their definition in 64 bits."""

import math

import pytest
import torch

from axon_amd.utils.torch.controls import LogitControls, controlled_logits, controlled_logprobs_from_logits

import controls_reference as R

pytestmark = pytest.mark.gpu

# As derived beside the tests of ordinary rows: a log-probability of logits of at most 80, and an entropy of about 12 such terms.
LP_TOL = 1.1e-4
ENT_TOL = 12 * LP_TOL


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("v", [40, 8192, 16383, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("most", [1, 3, 4, 5])
def test_rows_of_few_ids_under_penalties(v, dtype, most):
    """Masks that leave a lane between none and ``most`` of its ids, in every wavefront of a workgroup, beside histories of the same ids."""
    n = 24
    g = gen(v + most)
    z = (torch.randn(n, v, generator=g, device="cuda") * 3).to(dtype)
    keep = torch.rand(n, v, generator=g, device="cuda") < 0.3 * most / (16 if dtype == torch.float32 else 32)
    keep[:, -1] = True
    keep[3] = False
    tokens = torch.randint(0, v, (n,), generator=g, device="cuda")
    tokens[::3] = v - 1
    lens = [13, 11]
    kw = dict(repetition_penalty=1.4, frequency_penalty=0.3, presence_penalty=0.2)
    bias_ids, bias = torch.arange(0, v, 7, device="cuda"), torch.randn(len(range(0, v, 7)), generator=g, device="cuda")
    ctl = LogitControls(tokens, torch.tensor([0, 13, 24], dtype=torch.int32, device="cuda"), allowed=R.pack(keep), temperature=0.9,
                        bias_ids=bias_ids, bias=bias, **kw)
    out, slope, _ = R.controlled(z, R.spans_of(lens, "all"), tokens, repetition=1.4, frequency=0.3, presence=0.2, temperature=0.9,
                                 bias_ids=bias_ids.cpu(), bias=bias.cpu(), keep=list(keep))
    labels = torch.where(torch.arange(n, device="cuda") % 2 == 0, v - 1, tokens)
    lp_want, ent_want = R.scored(out, slope, labels)
    lp, ent = controlled_logprobs_from_logits(z, labels, ctl)
    gone = lp_want == -math.inf
    assert gone[3] and torch.equal(lp.cpu() == -math.inf, gone)
    assert ((lp.double().cpu() - lp_want).abs()[~gone] <= LP_TOL).all()
    assert ((ent.double().cpu() - ent_want).abs() <= ENT_TOL).all()


def test_a_history_that_ends_where_32_bits_do():
    """The longest history that is taken, 2^31 - 2 tokens (8.6 GB), most of them padding."""
    n, v = 2 ** 31 - 2, 8
    tokens = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    at = torch.tensor([0, 1, 4096, 2 ** 30, n - 8192, n - 4097, n - 4096, n - 513, n - 512, n - 2, n - 1], device="cuda")
    ids = torch.tensor([0, 1, 0, 2, 3, 3, 4, 3, 5, 5, 6], device="cuda")
    tokens[at] = ids.int()
    z = torch.linspace(-2.0, 2.0, v, device="cuda")[None]
    ctl = LogitControls(tokens[None], positions="last", frequency_penalty=0.5, presence_penalty=0.25, repetition_penalty=2.0)
    count = torch.bincount(ids, minlength=v).float()[None]
    want = torch.where(count > 0, torch.where(z > 0, z / 2, z * 2), z) - 0.5 * count - 0.25 * (count > 0)
    assert (controlled_logits(z, ctl) - want).abs().max() <= 8 * 2.0 ** -24 * 5


@pytest.mark.parametrize("remove_padding", [True, False])
@pytest.mark.parametrize("left", [False, True])
@pytest.mark.parametrize("loss_fn,extra", [("ppo", {}), ("ppo", dict(kl_coef=0.1, kl_type="k1")), ("ppo", dict(kl_coef=0.1, kl_type="k2")),
                                           ("ppo", dict(kl_coef=0.1, kl_type="abs+", entropy_coef=0.01)), ("reinforce", {})])
def test_a_step_whose_prompts_hold_what_the_controls_rule_out(remove_padding, left, loss_fn, extra):
    """A prompt, the padding and the first token of a sequence are no draws of the sampler: the step's loss, its metrics and its gradient are
    numbers, and those of the same step with its log-probabilities kept at the response's positions only."""
    from types import SimpleNamespace

    from axon_amd.models.fsdp_models import CausalLM
    from axon_amd.protocol import DataProto
    from axon_amd.utils.fsdp.forward_utils import fsdp_model_forward

    g = gen(7)
    b, t, h, v, prompt = 3, 12, 32, 500, 4
    lens = [12, 8, 5]
    emb, w = torch.randn(v, h, generator=g, device="cuda"), torch.randn(v, h, generator=g, device="cuda")
    place = lambda x, i: [0] * (t - lens[i]) + x if left else x + [0] * (t - lens[i])
    row = lambda i: [9] + [3, 9, 40] + (torch.randint(10, 400, (lens[i] - prompt,), generator=g, device="cuda")).tolist()  # 9: ruled out
    batch = {"input_ids": torch.tensor([place(row(i), i) for i in range(b)], device="cuda"),
             "attention_mask": torch.tensor([place([1] * lens[i], i) for i in range(b)], device="cuda"),
             "response_mask": torch.tensor([place([0] * prompt + [1] * (lens[i] - prompt), i) for i in range(b)], device="cuda"),
             "position_ids": torch.zeros(b, t, dtype=torch.int64, device="cuda")}
    keep = torch.ones(1, v, dtype=torch.bool, device="cuda")
    keep[:, 3] = False
    controls = dict(repetition_penalty=1.2, bias_ids=torch.tensor([9], device="cuda"), bias=torch.tensor([-math.inf], device="cuda"),
                    allowed=R.pack(keep))
    own = batch["response_mask"] != 0
    bent = torch.ones(v, device="cuda", requires_grad=True)

    class Model(torch.nn.Module):
        def forward(self, input_ids=None, attention_mask=None, position_ids=None, use_cache=False):
            return SimpleNamespace(logits=emb[input_ids] @ w.t() / h ** 0.5 * bent)

    def forward(kept):
        ent, lp = fsdp_model_forward(Model(), batch, 0.9, True, use_remove_padding=remove_padding, use_fused_kernels=False,
                                     logit_controls=controls)
        return (ent, lp) if not kept else (ent, torch.where(own, lp, 0.0))

    noise = 0.1 * torch.randn(b, t, generator=g, device="cuda")
    advantages = torch.randn(b, t, generator=g, device="cuda")

    def step(kept):
        with torch.no_grad():
            _, old = forward(kept)
        mask = batch["response_mask"].float()
        data = DataProto.from_dict(tensors={"old_log_probs": old + noise * mask, "ref_log_prob": old - noise * mask, "advantages": advantages,
                                            "response_mask": mask})
        meta = {"loss_fn": loss_fn, "loss_fn_args": dict(extra), "dp_replicas": 1, "n_micro_batches": 1, "temperature": 0.9}
        module = lambda inputs, m: dict(zip(("entropys", "log_probs"), forward(kept)))  # noqa: E731
        loss, metrics = CausalLM.forward_backward_fn(module, data, meta)
        return old, loss, metrics, *torch.autograd.grad(loss, bent)

    old, loss, metrics, grad = step(False)
    assert torch.isfinite(old).all() and (old[~own] == 0).all() and (old[own] < 0).all()
    assert torch.isfinite(loss) and torch.isfinite(grad).all() and (grad != 0).any()
    assert all(math.isfinite(float(x)) for x in metrics.values())
    _, want, want_metrics, want_grad = step(True)
    assert torch.equal(loss, want) and metrics == want_metrics and torch.equal(grad, want_grad)


@pytest.mark.parametrize("remove_padding", [True, False])
def test_a_step_without_a_response_mask_scores_what_is_there(remove_padding):
    from types import SimpleNamespace

    from axon_amd.utils.fsdp.forward_utils import fsdp_model_forward

    ids = torch.tensor([[0, 5, 6, 7], [8, 9, 0, 0]], device="cuda")
    there = torch.tensor([[0, 1, 1, 1], [1, 1, 0, 0]], device="cuda")
    logits = torch.randn(2, 4, 50, generator=gen(3), device="cuda")
    model = lambda **kw: SimpleNamespace(logits=logits if not remove_padding else logits[there != 0][None])  # noqa: E731
    _, lp = fsdp_model_forward(model, {"input_ids": ids, "attention_mask": there, "position_ids": ids}, 1.0, use_fused_kernels=False,
                               use_remove_padding=remove_padding, logit_controls=dict(presence_penalty=0.0))
    want = torch.zeros(2, 4, dtype=torch.float64, device="cuda")
    log_p = torch.log_softmax(logits.double(), 2)
    for i, p in ((0, 2), (0, 3), (1, 1)):
        want[i, p] = log_p[i, p - 1, ids[i, p]]
    assert (lp - want).abs().max() <= LP_TOL


@pytest.mark.parametrize("temperature", [1e20, 1e27, 1e29, 1e31, 3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("per_seq", [False, True])
def test_what_is_out_is_out_at_any_temperature(temperature, dtype, per_seq):
    """Whole rows, rows of few ids, and a vocabulary that ends inside a wavefront's ids."""
    n, v = 70, 3001
    g = gen(5)
    z = (torch.randn(n, v, generator=g, device="cuda") * 3).to(dtype)
    keep = torch.rand(n, v, generator=g, device="cuda") < 0.5
    keep[::3] = torch.rand(n, v, generator=g, device="cuda")[::3] < 0.002
    keep[1::7] = True
    keep[:, 11] = True
    labels = torch.full((n,), 11, dtype=torch.int64, device="cuda")
    value = torch.full((1,), temperature, device="cuda") if per_seq else temperature
    ctl = LogitControls(cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device="cuda"), allowed=R.pack(keep), temperature=value)
    out, slope, _ = R.controlled(z, R.spans_of([n], "all"), None, keep=list(keep), temperature=temperature)
    ones = torch.ones(n, device="cuda")
    lp_want, ent_want, grad, size = R.scored(out, slope, labels, ones, ones)
    z.requires_grad_(True)
    lp, ent = controlled_logprobs_from_logits(z, labels, ctl)
    assert ((lp.double().cpu() - lp_want).abs() <= LP_TOL).all() and ((ent.double().cpu() - ent_want).abs() <= ENT_TOL).all()
    d, = torch.autograd.grad([lp, ent], z, [ones, ones])
    # 1 / T and a gradient with it may be numbers that 32 bits hold in steps of 2^-149 (bf16: 2^-133)
    step = 2.0 ** (-133 if dtype == torch.bfloat16 else -149)
    bound = 2 * ENT_TOL * size + (2.0 ** -8 * grad.abs() if dtype == torch.bfloat16 else 0.0) + step * (2 + 3 * temperature * size)
    assert ((d.double().cpu() - grad).abs() <= bound).all() and (d[~keep] == 0).all()


@pytest.mark.parametrize("cu", [[3, 3, 9], [2, 2, 2, 7, 9], [3, 9], [1, 1, 6]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("many", [9, 40000])  # rows: where there are many, a wavefront walks several of them
def test_rows_in_front_of_the_first_sequence(cu, dtype, many):
    """They have no history; the sequences behind them have their own, and their own biases."""
    n, v, seqs = many, 2500 if many < 100 else 90, len(cu) - 1
    g = gen(len(cu))
    z = (torch.randn(n, v, generator=g, device="cuda") * 2).to(dtype)
    tokens = torch.randint(0, 40, (n,), generator=g, device="cuda")
    bias_ids = torch.randint(0, 60, (seqs, 20), generator=g, device="cuda")
    bias = torch.randn(seqs, 20, generator=g, device="cuda")
    freq = torch.rand(seqs, generator=g, device="cuda")
    kw = dict(repetition_penalty=1.5, frequency_penalty=freq, bias_ids=bias_ids, bias=bias)
    ctl = LogitControls(tokens, torch.tensor(cu, dtype=torch.int32, device="cuda"), **kw)
    spans = [(i, a, p + 1) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])) for p in range(a, b)]
    rows = slice(cu[0], cu[-1])
    out, slope, size = R.controlled(z[rows], spans, tokens, repetition=1.5, frequency=freq.cpu(), bias_ids=bias_ids.cpu(), bias=bias.cpu())
    got = controlled_logits(z, ctl)[rows].double().cpu()
    assert ((got - out).abs() <= 7 * 2.0 ** -24 * size + (2.0 ** -8 * out.abs() if dtype == torch.bfloat16 else 0.0) + 1e-30).all()
    labels = tokens.roll(-1)
    lp_want, ent_want = R.scored(out, slope, labels[rows])
    lp, ent = controlled_logprobs_from_logits(z, labels, ctl)
    assert ((lp[rows].double().cpu() - lp_want).abs() <= LP_TOL).all() and ((ent[rows].double().cpu() - ent_want).abs() <= ENT_TOL).all()


@pytest.mark.parametrize("temperature", [1.2e-38, 1e-30, 1e-3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_temperatures_next_to_nothing(temperature, dtype):
    """Logits of the temperature's size: penalties beside them are all there is."""
    n, v = 70, 3001
    g = gen(6)
    z = (torch.randn(n, v, generator=g, device="cuda") * 3 * temperature * 16).to(dtype)
    keep = torch.rand(n, v, generator=g, device="cuda") < 0.5
    keep[::3] = torch.rand(n, v, generator=g, device="cuda")[::3] < 0.002
    keep[:, 11] = True
    labels = torch.full((n,), 11, dtype=torch.int64, device="cuda")
    ctl = LogitControls(allowed=R.pack(keep), temperature=temperature)
    out, slope, _ = R.controlled(z, R.spans_of([n], "all"), None, keep=list(keep), temperature=temperature)
    ones = torch.ones(n, device="cuda")
    lp_want, ent_want, grad, size = R.scored(out, slope, labels, ones, ones)
    z.requires_grad_(True)
    lp, ent = controlled_logprobs_from_logits(z, labels, ctl)
    # logits over the temperature of up to 220 instead of 80
    assert ((lp.double().cpu() - lp_want).abs() <= 3 * LP_TOL).all() and ((ent.double().cpu() - ent_want).abs() <= 3 * ENT_TOL).all()
    d, = torch.autograd.grad([lp, ent], z, [ones, ones])
    # a probability below 2^-126 is 0, and up to 150 / T times that is missing (1.8e-36 / T); a row's constants are the upstream gradients
    # times 1 + entropy over T, which at the smallest temperature is beyond 32 bits (8e37 * 5): there the gradient is not compared
    bound = 6 * ENT_TOL * size + (2.0 ** -8 * grad.abs() if dtype == torch.bfloat16 else 0.0) + 1e-35 / temperature
    assert temperature < 1e-37 or ((d.double().cpu() - grad).abs() <= bound).all() and (d[~keep] == 0).all()
