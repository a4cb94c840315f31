"""Backward passes that write their gradient over the logits, beside other operators on the same logits."""

import pytest
import torch

from axon_amd.utils.torch.ops import (entropy_from_logits, logprobs_and_entropy_from_logits, logprobs_from_logits,
                                      token_logprobs_from_logits, top_logprobs_from_logits)

pytestmark = pytest.mark.gpu


def _one(x):
    return token_logprobs_from_logits(x, torch.zeros(x.shape[0], 1, dtype=torch.int64, device="cuda"), inplace_backward=True)[0]


def _label(x, **kw):
    return logprobs_from_logits(x, torch.zeros(x.shape[0], dtype=torch.int64, device="cuda"), **kw)


WRITERS = {  # operators that write their gradient over the logits
    "tokens": _one,
    "top": lambda x: top_logprobs_from_logits(x, 3, inplace_backward=True).top_logprobs,
    "label": _label,  # as it does by default
    "label_and_entropy": lambda x: logprobs_and_entropy_from_logits(x, torch.zeros(x.shape[0], dtype=torch.int64, device="cuda"), True)[0],
}
READERS = {
    "tokens": lambda x: token_logprobs_from_logits(x, torch.zeros(x.shape[0], 1, dtype=torch.int64, device="cuda"))[0],
    "top": lambda x: top_logprobs_from_logits(x, 3).top_logprobs,
    "label": lambda x: _label(x, inplace_backward=False),
    "entropy": entropy_from_logits,
    "product": lambda x: x * x,
    **{"inplace_" + name: op for name, op in WRITERS.items()},
}


@pytest.mark.parametrize("leaf", [True, False])
@pytest.mark.parametrize("writer", WRITERS)
@pytest.mark.parametrize("reader", READERS)
def test_logits_that_a_backward_has_written_over_are_not_read_as_logits(reader, writer, leaf):
    """The later operator's backward comes first.  Where it writes over the logits, the earlier one's refuses; where it only reads
    them, both have the gradients that they have by themselves."""
    z = torch.randn(4, 300, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))

    def logits():
        x = z.clone().requires_grad_(True)
        return (x, x) if leaf else (x, x * 1)

    root, x = logits()
    first, second = READERS[reader](x), WRITERS[writer](x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([first.sum() + second.sum()], root)
    if reader.startswith("inplace"):
        return
    root, x = logits()
    first, second = WRITERS[writer](x), READERS[reader](x)
    both, = torch.autograd.grad([first.sum() + second.sum()], root)
    alone = []
    for op in (READERS[reader], WRITERS[writer]):
        root, x = logits()
        alone.append(torch.autograd.grad(op(x).sum(), root)[0].clone())
    assert torch.equal(both, alone[0] + alone[1])


@pytest.mark.parametrize("writer", WRITERS)
def test_a_second_backward_over_written_logits_is_refused(writer):
    x = torch.randn(4, 300, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).requires_grad_(True)
    out = WRITERS[writer](x).sum()
    torch.autograd.grad(out, x, retain_graph=True)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, x)
    # the next forward reads what is there now
    assert torch.autograd.grad(WRITERS[writer](x).sum(), x)[0].shape == x.shape
