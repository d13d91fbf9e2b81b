"""The decay-attention layer's refusals and autograd rules, without a GPU."""
import ctypes

import pytest
import torch


# ------------------------------------------------------------------------------------------ states in order
@pytest.mark.parametrize("src,dst,n_rows,n_src", [
    ((4096, 8192), (8192, 4096), 4, 4),          # two states that would change places
    ((4096, 8192), (16384, 4096 + 64), 4, 4),    # a part of another state
    ((4096, 8192), (16384, 16384 + 128), 4, 4),  # two outputs over one another
    ((4096, 8192), (16384, 8192), 2, 4),
    ((4096, 8192), (16384, (1 << 20) - 64), 4, 4),   # the order itself
])
def test_reorder_refuses_outputs_over_any_state_and_one_another(src, dst, n_rows, n_src):
    from icml_b200 import _lib
    arr = ctypes.c_void_p * 2
    rc = _lib.lib().pgf_beam_reorder(arr(*src), arr(*dst), (ctypes.c_int64 * 2)(64, 64), 2, 1 << 20, n_rows, n_src, None)
    assert rc != 0 and "overwrite" in _lib.last_error()


# ----------------------------------------------------------------------------------------- prompts and models
def _model(variant="decay"):
    from icml_b200.lm import PGFLanguageModel
    return PGFLanguageModel(31, 64, 16, 128, 2, 64, "cpu", variant=variant)


@pytest.mark.parametrize("lengths", [[6, 3], [5, 2 ** 40], [0, 5], [5, -1]])
def test_prefill_refuses_lengths_outside_the_prompt(lengths):
    from icml_b200.generate import beam_search, prefill
    ids = torch.zeros(2, 5, dtype=torch.int64)
    for call in (lambda n: prefill(_model(), ids, n), lambda n: beam_search(_model(), ids, 2, 2, n)):
        with pytest.raises(ValueError, match="1 to 5 tokens"):
            call(torch.tensor(lengths))


def test_sequence_sharding_refuses_a_decay_model():
    """The variant has no segment form: named on the host, before any operator runs."""
    from icml_b200 import seqpar
    m, ids = _model(), torch.zeros(1, 8, dtype=torch.int64)
    x = torch.zeros(1, 8, 64)
    for call in (lambda: seqpar.lm_forward_backward(m, ids, ids, seqpar.SeqGroup()),
                 lambda: seqpar.block_forward(m.backbone.layers[0], x, seqpar.SeqGroup()),
                 lambda: seqpar.block_backward(m.backbone.layers[0], x, x, None, seqpar.SeqGroup())):
        with pytest.raises(ValueError, match="PGFDecayBlock"):
            call()
