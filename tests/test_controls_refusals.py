"""What the controls' entry points refuse, on the host: nothing is launched."""

import ctypes

import pytest
import torch

from axon_amd import _lib
from axon_amd.utils.torch.controls import LogitControls, controlled_logits, controlled_logprobs_from_logits

Z = torch.zeros(4, 50)
IDS = torch.zeros(4, dtype=torch.int64)
CU = torch.tensor([0, 3, 4], dtype=torch.int32)


@pytest.mark.parametrize("kw", [
    dict(positions="first"), dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(temperature=0.0),
    dict(temperature=float("inf")), dict(frequency_penalty=float("nan")), dict(presence_penalty=float("inf")),
    dict(repetition_penalty=1.1), dict(frequency_penalty=0.1), dict(presence_penalty=torch.zeros(2)),
    dict(token_ids=IDS.float()), dict(token_ids=IDS.view(1, 2, 2)), dict(token_ids=IDS, cu_seqlens=CU[None]),
    dict(token_ids=IDS, response_mask=torch.ones(3)), dict(response_mask=torch.ones(4)),
    dict(token_ids=IDS, attention_mask=torch.ones(1, 4)), dict(attention_mask=torch.ones(4)),
    dict(token_ids=IDS, cu_seqlens=CU, repetition_penalty=torch.ones(3)),
    dict(token_ids=IDS, cu_seqlens=CU, temperature=torch.ones(2, dtype=torch.int64)),
    dict(token_ids=IDS, cu_seqlens=CU, temperature=torch.ones(2, 1)),
    dict(token_ids=IDS, cu_seqlens=CU, temperature=torch.ones(2, requires_grad=True)),
    dict(bias=torch.zeros(3)), dict(bias_ids=IDS), dict(bias=torch.zeros(3), bias_ids=IDS),
    dict(bias=torch.zeros(4), bias_ids=IDS.float()), dict(bias=torch.zeros(4, requires_grad=True), bias_ids=IDS),
    dict(bias=torch.zeros(3, 4), bias_ids=IDS.expand(3, 4), token_ids=IDS, cu_seqlens=CU),
    dict(bias=torch.zeros(()), bias_ids=IDS[0]),
    dict(allowed=torch.ones(2, dtype=torch.int64)), dict(allowed=torch.ones(4, 50, dtype=torch.bool)),
    dict(allowed=torch.ones(0, 2, dtype=torch.int32)), dict(allowed=torch.ones(1, 2, 2, dtype=torch.int32)),
    dict(allowed_index=IDS), dict(allowed=torch.ones(2, dtype=torch.int32), allowed_index=IDS.float()),
])
def test_controls_that_make_no_sense_are_refused(kw):
    with pytest.raises(ValueError):
        LogitControls(**kw)


@pytest.mark.parametrize("kw", [dict(repetition_penalty="1.1"), dict(temperature=None), dict(frequency_penalty=True)])
def test_values_that_are_no_numbers_are_refused(kw):
    with pytest.raises(TypeError):
        LogitControls(IDS, CU, **kw)


@pytest.mark.parametrize("kw", [
    dict(token_ids=IDS[:3], presence_penalty=1.0),  # rows that are no positions
    dict(token_ids=IDS, cu_seqlens=CU, positions="last", presence_penalty=1.0),
    dict(temperature=torch.ones(3), positions="last"), dict(temperature=torch.ones(4)),
    dict(allowed=torch.ones(1, dtype=torch.int32)), dict(allowed=torch.ones(3, 2, dtype=torch.int32)),
    dict(allowed=torch.ones(3, 2, dtype=torch.int32), allowed_index=IDS[:3]),
])
def test_controls_of_other_logits_are_refused(kw):
    ctl = LogitControls(**kw)
    with pytest.raises(ValueError):
        controlled_logits(Z, ctl)
    with pytest.raises(ValueError):
        controlled_logprobs_from_logits(Z, IDS, ctl)


def test_logits_and_labels_that_do_not_fit_are_refused():
    ctl = LogitControls()
    for z in (Z.half(), Z.double(), Z.long()):
        with pytest.raises(ValueError, match="fp32 or bf16"):
            controlled_logits(z, ctl)
        with pytest.raises(ValueError, match="fp32 or bf16"):
            controlled_logprobs_from_logits(z, IDS, ctl)
    for labels in (IDS[:3], IDS.float(), IDS[:, None], IDS.to(torch.int16)):
        with pytest.raises(ValueError, match="labels"):
            controlled_logprobs_from_logits(Z, labels, ctl)
    with pytest.raises(TypeError):
        controlled_logits(Z, dict(temperature=2.0))
    with pytest.raises(ValueError, match="written over"):
        controlled_logits(Z.clone().requires_grad_(True), ctl, inplace=True)


def test_tensors_that_are_not_on_a_gpu_are_refused():
    with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
        controlled_logits(Z, LogitControls())
    with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
        controlled_logprobs_from_logits(Z, IDS, LogitControls(IDS, CU, repetition_penalty=1.1))


def test_the_c_entry_points_check_their_arguments():
    lib = _lib.load()
    p = ctypes.addressof(ctypes.create_string_buffer(64)) & ~15  # any address: nothing is read
    ok = dict(repetition_all=1.0, temperature_all=1.0)

    def apply(logits=p, dtype=0, ld=100, n=2, v=100, out=p, ld_out=100, **c):
        s = _lib.ControlsStruct(**{**ok, **c})
        return lib.axon_controls_apply(logits, dtype, ld, n, v, ctypes.byref(s), out, ld_out, None)

    assert apply(n=0) == 0
    tokens = dict(token_ids=p, n_tokens=2, n_seqs=1, uniform_len=2, every_position=1, presence_all=1.0)
    for bad in (dict(logits=None), dict(out=None), dict(dtype=2), dict(ld=99), dict(ld_out=99), dict(n=-1), dict(v=0),
                dict(logits=p + 2), dict(repetition_all=0.0), dict(temperature_all=-1.0), dict(frequency_all=float("nan")),
                dict(n_bias=2), dict(mask_kind=3), dict(n_seqs=-1), dict(temperature=p), dict(tokens, n_seqs=0),
                dict(tokens, uniform_len=0)):
        assert apply(**bad) == -1, bad
    for bad in (dict(n=1 << 24), dict(v=1 << 30, ld=1 << 30, ld_out=1 << 30), dict(allowed=p, allowed_rows=1, allowed_stride=3),
                dict(allowed=p, allowed_rows=3, allowed_stride=4), dict(tokens, n_tokens=3), dict(tokens, n=3),
                dict(tokens, every_position=0), dict(temperature=p, n_seqs=3)):
        assert apply(**bad) == -2, bad
    assert lib.axon_controls_apply(p, 0, 100, 2, 100, None, p, 100, None) == -1
    s = _lib.ControlsStruct(**ok)
    ws = lib.axon_controls_logprob_workspace_bytes(2, 100)
    assert ws > 0 and lib.axon_controls_logprob_workspace_bytes(-1, 100) < 0

    def fwd(labels=p, lp=p, stats=p, w=p, wb=ws):
        return lib.axon_controls_logprob_fwd(p, 0, 100, 2, 100, ctypes.byref(s), labels, 1, lp, p, stats, w, wb, 0, None)

    assert fwd(labels=None) == fwd(lp=None) == fwd(stats=None) == -1
    assert fwd(w=None) == fwd(wb=ws - 1) == fwd(w=p + 8) == -3
    assert lib.axon_controls_logprob_bwd(p, 0, 100, 2, 100, ctypes.byref(s), p, 1, None, p, p, p, 100, None) == -1
    assert lib.axon_controls_apply_bwd(p, 0, 100, 2, 100, ctypes.byref(s), None, 100, p, 100, None) == -1


def test_a_trainers_forward_refuses_what_it_cannot_score():
    from axon_amd.utils.fsdp.forward_utils import fsdp_model_forward

    ids = torch.zeros(2, 4, dtype=torch.int64)
    batch = {"input_ids": ids, "attention_mask": torch.ones_like(ids), "position_ids": ids}
    model = lambda **kw: type("Out", (), {"logits": torch.zeros(*kw["input_ids"].shape, 9)})()
    with pytest.raises(ValueError, match="use_fused_kernels=False"):
        fsdp_model_forward(model, batch, 1.0, logit_controls={"repetition_penalty": 1.1})
    for padding in (True, False):
        how = dict(use_fused_kernels=False, use_remove_padding=padding)
        with pytest.raises(ValueError, match="got temperature, token_ids"):
            fsdp_model_forward(model, batch, 1.0, logit_controls={"temperature": 2.0, "token_ids": ids}, **how)
        with pytest.raises(ValueError, match="allowed_index"):
            fsdp_model_forward(model, batch, 1.0, logit_controls={"allowed_index": ids[:, 1:]}, **how)
        with pytest.raises(_lib.AxonAmdError):  # there is no kernel for logits on the host
            fsdp_model_forward(model, batch, 1.0, logit_controls={"repetition_penalty": 1.1}, **how)
