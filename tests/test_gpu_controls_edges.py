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
