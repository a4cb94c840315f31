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
    ws = lib.axon_logits_top_workspace_bytes(0, 2, 100)
    assert ws > 0 and lib.axon_logits_top_workspace_bytes(7, 2, 100) < 0 and lib.axon_logits_top_workspace_bytes(0, 2, 0) < 0

    def top(logits=p, dtype=0, ld=100, n=2, v=100, k=3, logprob=None, labels=None, lse=p, lp=p, ids=p, w=p, wb=ws):
        return lib.axon_logits_top_fwd(logits, dtype, ld, n, v, k, labels, 1, logprob, p, lse, lp, ids, w, wb, 0, None)

    assert top(n=0) == 0
    for bad in (dict(logits=None), dict(dtype=2), dict(ld=99), dict(n=-1), dict(v=0), dict(lse=None), dict(lp=None),
                dict(ids=None), dict(w=None), dict(logprob=p), dict(logits=p + 2)):
        assert top(**bad) == -1, bad
    for bad in (dict(k=0), dict(k=129), dict(k=101), dict(n=1 << 25), dict(v=1 << 30, ld=1 << 30)):
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
