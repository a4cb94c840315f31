"""Temperatures and penalties without a reciprocal in 32 bits are refused, on the host: nothing is launched."""

import ctypes

import pytest
import torch

from axon_amd import _lib
from axon_amd.utils.torch.controls import LogitControls
from axon_amd.utils.torch.distillation import distillation_from_logits, distillation_loss_from_logits

SMALL = [1e-39, 2.0 ** -126 * 0.999, 1e-50]


@pytest.mark.parametrize("x", SMALL + [1e39])
def test_entry_points(x):
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="temperature must be positive"):
        LogitControls(temperature=x)
    with pytest.raises(ValueError, match="repetition_penalty must be positive"):
        LogitControls(ids[None], repetition_penalty=x)
    z, at, lq = torch.zeros(4, 50), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    for call in (lambda: distillation_from_logits(z, at, lq, temperature=x),
                 lambda: distillation_loss_from_logits(z, at, lq, torch.ones(4), temperature=x)):
        with pytest.raises(ValueError, match="temperature must be positive"):
            call()
    LogitControls(ids[None], temperature=2.0 ** -126, repetition_penalty=2.0 ** -126)


@pytest.mark.parametrize("x", SMALL[:2])
def test_the_c_entry_points(x):
    lib = _lib.load()
    p = ctypes.addressof(ctypes.create_string_buffer(64)) & ~15  # any address: nothing is read
    for c in (dict(repetition_all=1.0, temperature_all=x), dict(repetition_all=x, temperature_all=1.0)):
        s = _lib.ControlsStruct(**c)
        assert lib.axon_controls_apply(p, 0, 100, 2, 100, ctypes.byref(s), p, 100, None) == -1
    ws = lib.axon_distill_workspace_bytes(0, 2, 100)
    assert lib.axon_distill_fwd(p, 0, 100, 2, 100, p, 1, p, 3, None, 0, 1, 0.5, x, p, p, p, p, p, ws, 0, None) == -1
    assert lib.axon_distill_bwd(p, 0, 100, 2, 100, p, 1, 3, None, x, p, p, p, 0, p, 100, None) == -1


def test_flags_of_the_tail():
    lib = _lib.load()
    p = ctypes.addressof(ctypes.create_string_buffer(64)) & ~15
    ws = lib.axon_distill_workspace_bytes(0, 2, 100)
    for tail in (3, 3 + 4, 16, -1, 3 + 8):
        assert lib.axon_distill_fwd(p, 0, 100, 2, 100, p, 1, p, 3, None, 0, tail, 0.5, 1.0, p, p, p, p, p, ws, 0, None) == -1
    for tail in (0 + 4, 1 + 8, 2 + 4):  # taken: the workspace is looked at next
        assert lib.axon_distill_fwd(p, 0, 100, 2, 100, p, 1, p, 3, None, 0, tail, 0.5, 1.0, p, p, p, p, p, ws - 1, 0, None) == -3
