"""What the alternatives' entry points refuse, on the host: nothing is launched."""

import ctypes

import pytest
import torch

from axon_amd import _lib
from axon_amd.utils.torch.ops import token_logprobs_from_logits, top_logprobs_from_logits

Z = torch.zeros(4, 50)


@pytest.mark.parametrize("k", [0, -1, 51, 129, 1 << 40])
def test_a_count_out_of_range_is_refused(k):
    with pytest.raises(ValueError, match="k must be between"):
        top_logprobs_from_logits(Z, k)


@pytest.mark.parametrize("k", [1.0, True, None, "3"])
def test_a_count_that_is_no_int_is_refused(k):
    with pytest.raises(TypeError, match="k must be an int"):
        top_logprobs_from_logits(Z, k)


def test_other_types_are_refused():
    for z in (Z.half(), Z.double(), Z.long()):
        with pytest.raises(ValueError, match="fp32 or bf16"):
            top_logprobs_from_logits(z, 3)
        with pytest.raises(ValueError, match="fp32 or bf16"):
            token_logprobs_from_logits(z, torch.zeros(4, 2, dtype=torch.int64))


@pytest.mark.parametrize("labels", [torch.zeros(3, dtype=torch.int64), torch.zeros(4), torch.zeros(4, dtype=torch.int16)])
def test_labels_that_do_not_fit_are_refused(labels):
    with pytest.raises(ValueError):
        top_logprobs_from_logits(Z, 3, labels)


@pytest.mark.parametrize("ids", [torch.zeros(4, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(4, 2),
                                 torch.zeros(4, 0, dtype=torch.int64), torch.zeros(4, 513, dtype=torch.int64),
                                 torch.zeros(2, 2, 2, dtype=torch.int64)])
def test_token_ids_that_do_not_fit_are_refused(ids):
    with pytest.raises(ValueError):
        token_logprobs_from_logits(Z, ids)


def test_tensors_that_are_not_on_a_gpu_are_refused():
    with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
        top_logprobs_from_logits(Z, 3)
    with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
        token_logprobs_from_logits(Z, torch.zeros(4, 2, dtype=torch.int64))


def test_the_c_entry_points_check_their_arguments():
    """Status codes of calls that a kernel must not see: null pointers, sizes, small workspaces, unaligned rows."""
    lib = _lib.load()
    p = ctypes.addressof(ctypes.create_string_buffer(64)) & ~15  # any address: nothing is read
    ws = lib.axon_logits_top_workspace_bytes(0, 2, 100000)
    assert ws > 0 and lib.axon_logits_top_workspace_bytes(7, 2, 100) < 0 and lib.axon_logits_top_workspace_bytes(0, 2, 0) < 0

    def top(logits=p, dtype=0, ld=100000, n=2, v=100000, k=3, logprob=None, labels=None, lse=p, lp=p, ids=p, w=p, wb=ws):
        return lib.axon_logits_top_fwd(logits, dtype, ld, n, v, k, labels, 1, logprob, p, lse, lp, ids, w, wb, 0, None)

    assert top(n=0) == 0
    for bad in (dict(logits=None), dict(dtype=2), dict(ld=99999), dict(n=-1), dict(v=0), dict(lse=None), dict(lp=None),
                dict(ids=None), dict(w=None), dict(logprob=p), dict(logits=p + 2)):
        assert top(**bad) == -1, bad
    for bad in (dict(k=0), dict(k=129), dict(k=101, v=100), dict(n=1 << 25), dict(v=1 << 30, ld=1 << 30)):
        assert top(**bad) == -2, bad
    assert top(wb=ws - 1) == -3

    def tokens(logits=p, ids=p, k=3, out=p, lse=p, n=2, v=100000, w=p, wb=1 << 20):
        return lib.axon_logits_tokens_fwd(logits, 0, v, n, v, ids, 1, k, out, p, lse, w, wb, 0, None)

    assert tokens(n=0) == 0
    for bad in (dict(logits=None), dict(ids=None), dict(out=None), dict(lse=None)):
        assert tokens(**bad) == -1, bad
    assert tokens(k=0) == tokens(k=513) == -2
    assert tokens(wb=0) == tokens(w=None) == -3

    def bwd(ids=p, k=3, labels=p, lse=p, ent=p, g_ids=p, g_label=p, g_en=p, out=p, ld_d=100):
        return lib.axon_logits_tokens_bwd(p, 0, 100, 2, 100, ids, 1, k, labels, 1, lse, ent, g_ids, g_label, g_en, out, ld_d, None)

    for bad in (dict(ids=None), dict(labels=None), dict(lse=None), dict(ent=None), dict(out=None), dict(ld_d=99), dict(out=p + 1)):
        assert bwd(**bad) == -1, bad
    assert bwd(k=513) == bwd(k=-1) == -2


def test_the_heads_operands_are_checked_on_the_host():
    from axon_amd.utils.kernel.linear_top_logprobs import linear_token_logprobs, linear_top_logprobs

    h, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(50, 64, dtype=torch.bfloat16)
    ids = torch.zeros(4, 2, dtype=torch.int64)
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(logit_softcapping=-1.0), dict(logit_softcapping=float("nan")), dict(labels=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            linear_top_logprobs(h, w, 3, **bad)
    for hh, ww in ((h.double(), w), (h, w.long()), (h, w[:, :32]), (h, w[0]), (h.view(-1)[0], w)):
        with pytest.raises(ValueError):
            linear_top_logprobs(hh, ww, 3)
    for bad in (ids[0], ids[:3], ids[None]):
        with pytest.raises(ValueError):
            linear_token_logprobs(h, w, bad)
    for call in (lambda: linear_top_logprobs(h, w, 3), lambda: linear_token_logprobs(h, w, ids)):
        with pytest.raises(_lib.AxonAmdError, match="no CPU fallback"):
            call()


def test_the_heads_c_entry_points_check_their_arguments():
    lib = _lib.load()
    p = (ctypes.addressof(ctypes.create_string_buffer(64)) + 15) & ~15
    big = 1 << 40
    assert lib.axon_lmhead_top_workspace_bytes(4, 64, 50) > 0
    assert lib.axon_lmhead_top_workspace_bytes(4, 33, 50) == -2 and lib.axon_lmhead_top_workspace_bytes(4, 0, 50) == -1

    def top(h=p, w=p, lab=None, n=4, hs=64, v=50, inv_t=1.0, cap=0.0, k=3, lp=None, ent=p, lse=p, eb=p, tl=p, ti=p, ws=p, wb=big, z=p,
            zb=big):
        return lib.axon_lmhead_top_fwd(h, w, lab, 1, n, hs, v, inv_t, cap, k, lp, ent, lse, eb, tl, ti, ws, wb, z, zb, None)

    assert top(n=0) == 0
    for bad in (dict(h=None), dict(w=None), dict(lab=p), dict(lp=p), dict(ent=None), dict(lse=None), dict(eb=None), dict(tl=None),
                dict(ti=None), dict(ws=None), dict(inv_t=0.0), dict(cap=-1.0), dict(h=p + 2), dict(n=-1), dict(z=None), dict(z=p + 8)):
        assert top(**bad) == -1, bad
    assert top(k=0) == top(k=129) == top(k=51) == top(hs=33) == -2
    assert top(wb=lib.axon_lmhead_top_workspace_bytes(4, 64, 50) - 512) == -3
    assert top(zb=lib.axon_lmhead_top_logits_bytes(4, 64, 50) - 1) == -3 and lib.axon_lmhead_top_logits_bytes(4, 33, 50) == -2

    def fwd(ids=p, k=3, lp=p, n=4, wb=big, hs=64, z=None, zb=0):
        return lib.axon_lmhead_tokens_fwd(p, p, ids, 1, n, hs, 50, 1.0, 0.0, k, lp, p, p, p, p, wb, z, zb, None)

    assert fwd(n=0) == 0 and fwd(ids=None) == fwd(lp=None) == -1 and fwd(k=0) == fwd(k=514) == -2 and fwd(wb=0) == -3
    assert fwd(z=p, zb=16) == -3 and fwd(z=p + 8, zb=big) == -1 and fwd(z=p, zb=big, hs=96) == -2

    def bwd(g=p, ids=p, k=3, lp=p, dw=p, ws=p, wb=0, n=4):
        return lib.axon_lmhead_tokens_bwd(g, p, p, p, ids, 1, k, lp, p, p, n, 64, 50, 1.0, 0.0, p, dw, ws, wb, None, 0, None)

    assert bwd(g=None) == bwd(ids=None) == bwd(lp=None) == bwd(dw=None) == bwd(ws=None) == -1
    assert bwd(k=0) == bwd(k=514) == -2 and bwd() == -3


@pytest.mark.parametrize("labels", [(3, 2), (6,), (1, 2, 3), (2, 3, 1), (2, 1, 3)])
def test_labels_of_another_arrangement_are_refused(labels):
    """As many as there are positions, but not where they lie: which belongs to which is not guessed."""
    with pytest.raises(ValueError, match="do not lie beside"):
        top_logprobs_from_logits(torch.zeros(2, 3, 50), 3, torch.zeros(labels, dtype=torch.int64))
