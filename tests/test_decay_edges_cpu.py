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


# ------------------------------------------------------------------------------------------ autograd rules
@pytest.fixture
def plain_ops(monkeypatch):
    """The layer's operators as host functions that differentiate what they are given (float64)."""
    from icml_b200 import pgf_decay
    from tests import decay_oracle as O
    kw64 = dict(R=8, base=100.0, pairs="halves", eps=1e-6)

    def rotate(q, k, wq, wk, turns, positions):
        return tuple(O.norm_rotate(x, w, positions, *kw64.values()) for x, w in ((q, wq), (k, wk)))

    def rotate_bwd(q, k, gq, gk, wq, wk, turns, positions):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
            g = torch.autograd.grad(rotate(*leaves, turns, positions), leaves, (gq, gk))
        return dict(zip(("grad_q", "grad_k", "grad_wq", "grad_wk"), g))

    def attend(q, k, v, ld, scale=None, state=None, lengths=None):
        return O.decay_attn(q, k, v, ld, scale, state, lengths)

    def attend_bwd(q, k, v, ld, g, scale=None, state=None, g_state=None, lengths=None, need_g_log_decay=False):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in (q, k, v, state, ld)]
            out = attend(*leaves[:3], leaves[4], scale, leaves[3])
            r = torch.autograd.grad(out, leaves, (g, torch.zeros_like(state) if g_state is None else g_state))
        return dict(zip(("grad_q", "grad_k", "grad_v", "grad_state", "grad_log_decay"), r))

    def gemm(a, b, a_trans=False, b_trans=False, out_dtype=None, addend=None):
        return (a.t() if a_trans else a) @ (b if b_trans else b.t())

    for name, f in (("qk_norm_rotate_fwd", rotate), ("qk_norm_rotate_bwd", rotate_bwd), ("decay_attn_fwd", attend),
                    ("decay_attn_bwd", attend_bwd), ("gemm", gemm)):
        monkeypatch.setattr(pgf_decay.ops, name, f)
    return pgf_decay


def _leaves(*shapes):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in shapes]


def test_positions_changed_before_the_backward_are_noticed(plain_ops):
    q, k, wq, wk = _leaves((1, 3, 2, 8), (1, 3, 1, 8), (8,), (8,))
    positions = torch.arange(3)[None]
    a, b = plain_ops.qk_norm_rotate(q, k, wq, wk, None, positions=positions)
    want = torch.autograd.grad(a.sum() + b.sum(), [q, k, wq, wk])
    assert torch.autograd.gradcheck(lambda *t: plain_ops.qk_norm_rotate(*t, None, positions=positions), [q, k, wq, wk])
    a, b = plain_ops.qk_norm_rotate(q, k, wq, wk, None, positions=positions)
    positions += 1                         # as a decoding loop moves on
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (a.sum() + b.sum()).backward()
    positions -= 1
    a, b = plain_ops.qk_norm_rotate(q, k, wq, wk, None, positions=positions)
    assert all(torch.equal(x, y) for x, y in zip(want, torch.autograd.grad(a.sum() + b.sum(), [q, k, wq, wk])))


def test_second_derivatives_are_refused(plain_ops):
    q, k, wq, wk, v, s, ld, x, W = _leaves((1, 3, 2, 8), (1, 3, 1, 8), (8,), (8,), (1, 3, 2, 4), (1, 2, 8, 4), (2,), (3, 8), (4, 8))
    positions = torch.arange(3)[None]

    def rotated():
        return plain_ops.qk_norm_rotate(q, k, wq, wk, None, positions=positions)[0], q

    def attended():
        return plain_ops.decay_attention(q, k, v, ld, scale=0.5, state=s)[0], v

    for f in (rotated, attended, lambda: (plain_ops._LinearFn.apply(x, W), x)):
        y, leaf = f()
        (first,) = torch.autograd.grad((y * y).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (first * leaf).sum().backward()
        (plain,) = torch.autograd.grad((lambda y: (y * y).sum())(f()[0]), leaf)
        assert torch.equal(first, plain)


@pytest.mark.parametrize("base", [-10000.0, float("nan"), 0.0, 0.01])
def test_rotary_turns_refuse_bases_without_frequencies(base):
    from icml_b200 import ops
    with pytest.raises(ValueError):
        ops.rotary_turns(8, base, "cpu")
