"""CPU checks of the decay-attention layer's C entry points: arguments are refused on the host, with the
reason in pgf_last_error, before any CUDA call."""
import pytest


def _lib():
    from icml_b200 import _lib as m
    return m, m.lib()


P = 256  # never dereferenced


def _rotate(L, D=64, R=64, pairs=0, dtype=0, q=P, turns=P, B=1, Hq=1, Hk=1):
    return L.pgf_qk_norm_rotate_fwd(q, None, P, None, None, None, turns, None, 0, P, P, B, 4, Hq, Hk, D, R, pairs, 1e-6,
                                    dtype, None)


def _attn(L, H=4, Hq=4, Hk=2, Hv=1, Dk=64, Dv=64, dtype=0, q=P, ld=P, B=1, T=4):
    return L.pgf_decay_attn_fwd(q, None, P, None, P, None, ld, None, None, P, None, B, T, H, Hq, Hk, Hv, Dk, Dv, 1.0, dtype,
                                None, 0, None)


def _step(L, state=4096, out=1 << 20, rows=None, n_src=2):
    return L.pgf_decay_attn_step(P, None, P, None, P, None, P, state, rows, n_src, P, out, 2, 1, 1, 1, 1, 64, 64, 1.0, 0, None)


def _beam(L, K=4, V=100, end=-1, fin=None, dtype=0, logits=P, B=1):
    return L.pgf_beam_select(logits, P, fin, P, P, P, P, B, K, V, end, dtype, None)


@pytest.mark.parametrize("call,word", [
    (lambda L: _rotate(L, D=257), "head width"), (lambda L: _rotate(L, R=63), "rotated width"),
    (lambda L: _rotate(L, D=32), "rotated width"), (lambda L: _rotate(L, pairs=2), "pairs"),
    (lambda L: _rotate(L, dtype=5), "dtype"), (lambda L: _rotate(L, q=None), "null"), (lambda L: _rotate(L, turns=None), "null"),
    (lambda L: _rotate(L, B=-1), "bad shape"),
    (lambda L: _attn(L, Hq=3), "must divide"), (lambda L: _attn(L, Hv=0), "must divide"), (lambda L: _attn(L, Dk=0), "head widths"),
    (lambda L: _attn(L, Dv=257), "head widths"), (lambda L: _attn(L, dtype=2), "dtype"), (lambda L: _attn(L, q=None), "null"),
    (lambda L: _attn(L, ld=None), "null"), (lambda L: _attn(L, T=-1), "bad shape"),
    (lambda L: _step(L, out=4096 + 64), "overwrite"), (lambda L: _step(L, out=4096, rows=P), "overwrite"),
    (lambda L: _step(L, n_src=3), "3 states for 2 rows"), (lambda L: _step(L, state=None), "null"),
    (lambda L: _beam(L, K=33), "bad shape"), (lambda L: _beam(L, K=0), "bad shape"), (lambda L: _beam(L, V=1 << 30), "bad shape"),
    (lambda L: _beam(L, end=100), "end token"), (lambda L: _beam(L, fin=P), "end token"), (lambda L: _beam(L, dtype=3), "dtype"),
    (lambda L: _beam(L, logits=None), "null"),
])
def test_refused_on_the_host(call, word):
    m, L = _lib()
    assert call(L) != 0
    assert word in m.last_error()


def test_empty_calls_touch_nothing():
    _, L = _lib()
    assert _rotate(L, B=0) == 0 and _attn(L, B=0) == 0 and _beam(L, B=0) == 0
    assert L.pgf_beam_reorder(None, None, None, 0, None, 4, 4, None) == 0


def test_backward_reports_a_small_workspace():
    m, L = _lib()
    rc = L.pgf_qk_norm_rotate_bwd(P, None, P, None, P, P, None, None, P, None, 0, P, P, P, P, 0, 1, 4, 1, 1, 64, 64, 0, 1e-6, 0,
                                  P, 16, None)
    assert rc != 0 and "workspace" in m.last_error()
    assert L.pgf_decay_attn_workspace(2, 100, 4, 4, 4, 4, 64, 64, 1, 1) > 0
    assert L.pgf_decay_attn_workspace(2, 100, 4, 3, 4, 4, 64, 64, 1, 1) == 0


def test_python_operators_refuse_host_tensors():
    import torch

    from icml_b200 import ops
    x = torch.zeros(1, 2, 1, 16)
    with pytest.raises(RuntimeError):
        ops.qk_norm_rotate_fwd(x, x)
    with pytest.raises(RuntimeError):
        ops.decay_attn_fwd(x, x, x, torch.zeros(1))
    with pytest.raises(RuntimeError):
        ops.beam_select(torch.zeros(1, 1, 4), torch.zeros(1, 1))
    with pytest.raises(RuntimeError):
        ops.beam_reorder([x], torch.zeros(1, dtype=torch.int64))


def test_rotary_turns_are_fractions_of_a_turn():
    import math

    from icml_b200 import ops
    t = ops.rotary_turns(8, 100.0, "cpu")
    for i, f in enumerate(t.tolist()):
        assert abs(f / 2.0 ** 64 - 100.0 ** (-2 * i / 8) / (2 * math.pi)) < 1e-16
