"""Edges of the decay-attention layer's operators on the GPU: states that leave in shared memory's last places,
rows that need no reading, values that are no numbers, lengths of any whole type.

Tolerances are those of test_gpu_decay.py: 1e-5 of the 2-norm for what comes back as float32, 6e-3 for bfloat16;
whatever is called twice gives the same bits.
"""
import math

import pytest
import torch

from tests import decay_oracle as O
from tests.test_gpu_decay import BOTH, DEV, _beam_check, _close, _gen, _n

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------------------- states that leave
@pytest.mark.parametrize("Dk,Dv", [(64, 128), (48, 80), (64, 64), (128, 128), (128, 64)])
def test_final_states_of_whole_walks_repeat(Dk, Dv):
    """bfloat16 calls that are not cut hand their states over inside the kernel: the same bits in every one of a
    thousand calls, within the bound of float64."""
    from icml_b200 import ops
    from icml_b200._lib import lib
    B, L, H = 8, 130, 16
    assert lib().pgf_decay_attn_workspace(B, L, H, H, H, H, Dk, Dv, 1, 0) == 0, "cut"
    g = _gen(Dk * 1000 + Dv)
    q, k, v, go = (_n(g, B, L, H, d).bfloat16() for d in (Dk, Dk, Dv, Dv))
    ld = -torch.exp2(-1.0 - 0.5 * torch.arange(H, device=DEV)).float()
    s, gs = _n(g, B, H, Dk, Dv), _n(g, B, H, Dk, Dv)

    def call():
        _, end = ops.decay_attn_fwd(q, k, v, ld, state=s)
        return end, ops.decay_attn_bwd(q, k, v, ld, go, state=s, g_state=gs)["grad_state"]

    end, grad = call()
    s64 = s.double().requires_grad_()
    o, want = O.decay_attn(q.double(), k.double(), v.double(), ld.double(), Dk ** -0.5, s64, None)
    (g64,) = torch.autograd.grad((o * go.double()).sum() + (want * gs.double()).sum(), s64)
    _close(end, want, 1e-5, "state", 2)
    _close(grad, g64, 1e-5, "grad_state", 2)
    off = torch.zeros(2, dtype=torch.int64, device=DEV)
    for _ in range(1000):
        e, r = call()
        off += torch.stack([(e != end).sum(), (r != grad).sum()])
    assert not off.any(), off.tolist()


# ------------------------------------------------------------------------------------- rows without a choice
@pytest.mark.parametrize("live", [0, 1])
@pytest.mark.parametrize("B,K,V,dtype", [(16, 8, 50257, torch.bfloat16), (2, 4, 100003, torch.float32), (2, 16, 33000, torch.float32)])
def test_beam_rows_that_need_no_reading_leave_nothing_behind(B, K, V, dtype, live):
    """Sequences whose beams have all finished, and whose beams but one stand at -inf, at sizes whose rows are copied
    into shared memory: the selection is right, and the calls that follow at once give the bits of calls alone."""
    from icml_b200 import ops
    g = _gen(B + K)
    logits, scores = (3 * _n(g, B, K, V)).to(dtype), -10 + _n(g, B, K)
    q, k, v = (_n(g, 4, 256, 4, 64).bfloat16() for _ in range(3))
    ld = torch.full((4,), -0.05, device=DEV)
    done = torch.ones(B, K, dtype=torch.bool, device=DEV)
    if live:
        scores[:, 1:] = -math.inf
        done[:] = False
    torch.cuda.synchronize()
    alone, s_alone = ops.decay_attn_fwd(q, k, v, ld)
    torch.cuda.synchronize()
    _beam_check(logits, scores, done, V - 1)
    first = ops.beam_select(logits, scores, done, end_id=V - 1)
    if not live:
        order = torch.sort(scores, dim=1, descending=True, stable=True)
        assert torch.equal(first[0], order.values) and bool((first[2] == V - 1).all()) and bool(first[3].all())
        assert torch.equal(first[1], order.indices + K * torch.arange(B, device=DEV)[:, None])
    for _ in range(50):
        again = ops.beam_select(logits, scores, done, end_id=V - 1)
        out, end = ops.decay_attn_fwd(q, k, v, ld)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert torch.equal(out, alone) and torch.equal(end, s_alone)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("V", [50257, 1029, 100003])
def test_beam_nan_counts_in_every_column(V, dtype):
    """A NaN logit makes its row's log sum NaN and the row's candidates -inf wherever it stands: first and last
    column (single elements in front of and behind the 16-byte pieces, as rows of an odd width start anywhere), in a
    piece of its own kind, and among banned tokens."""
    g = _gen(V)
    B, K = 4, 4
    base = (3 * _n(g, B, K, V)).to(dtype)
    scores = -_n(g, B, K).abs()
    banned = slice(V // 2 - 100, V // 2 + 100)
    spots = [slice(0, 1), slice(V - 1, V), slice(1, 2), slice(V // 2, V // 2 + 1), slice(V // 2, V // 2 + 32), slice(7, 8)]
    for n, at in enumerate(spots):
        for k in range(K):
            logits = base.clone()
            logits[:, :, banned] = -math.inf
            logits[:, k, at] = math.nan
            so, flat, _ = _beam_check(logits, scores, None, None)
            assert not (flat // V == k).any(), (n, k)
    logits = base.clone()
    logits[:] = -math.inf
    logits[:, 1:, V - 1] = math.nan
    logits[:, 0, 3] = 1.0
    so, flat, _ = _beam_check(logits, scores, None, None)
    assert torch.equal(flat[:, 0], torch.full((B,), 3, device=DEV)) and bool((so[:, 1:] == -math.inf).all())


# ---------------------------------------------------------------------------------------------- decays, lengths
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("B,L", [(3, 70), (1, 4000)])
def test_a_decay_that_is_no_number_shows(B, L, dtype):
    """A NaN decay makes its head's outputs, states and gradients NaN, at one token and over cut walks, and leaves the
    other heads' bits alone; a row without tokens keeps its state."""
    from icml_b200 import ops
    g = _gen(L)
    q, k, v, go = (_n(g, B, L, 2, 64).to(dtype) for _ in range(4))
    s, gs = _n(g, B, 2, 64, 64), _n(g, B, 2, 64, 64)
    good, bad = torch.tensor([-0.1, -0.1], device=DEV), torch.tensor([math.nan, -0.1], device=DEV)

    def call(ld, lengths=None):
        out, end = ops.decay_attn_fwd(q, k, v, ld, state=s, lengths=lengths)
        r = ops.decay_attn_bwd(q, k, v, ld, go, state=s, g_state=gs, lengths=lengths, need_g_log_decay=True)
        one, new = ops.decay_attn_step(q[:, 0], k[:, 0], v[:, 0], ld, s)
        heads = [out.transpose(1, 2), end, r["grad_q"].transpose(1, 2), r["grad_k"].transpose(1, 2),
                 r["grad_v"].transpose(1, 2), r["grad_state"], one, new]
        return [t.transpose(0, 1) for t in heads] + [r["grad_log_decay"]]

    for i, (a, b) in enumerate(zip(call(good), call(bad))):
        assert torch.equal(a[1], b[1]), i
        assert bool(b[0].isnan().all() if i not in (3, 4) else b[0].isnan().any()), i
    none = torch.zeros(B, dtype=torch.int32, device=DEV)
    out, end, *_, g0, _, _, gl = call(bad, none)
    assert not out.any() and torch.equal(end.transpose(0, 1), s) and torch.equal(g0.transpose(0, 1), gs)


@pytest.mark.parametrize("dtype", BOTH)
def test_lengths_of_any_whole_type(dtype):
    """Lengths below zero and beyond the sequence, in 64 bits too, count as none and all."""
    from icml_b200 import ops
    g = _gen(11)
    B, L = 6, 200
    q, k, v, go = (_n(g, B, L, 2, 64).to(dtype) for _ in range(4))
    ld = torch.tensor([-0.1, -0.01], device=DEV)

    def call(n):
        out, end = ops.decay_attn_fwd(q, k, v, ld, lengths=n)
        return [out, end, *ops.decay_attn_bwd(q, k, v, ld, go, lengths=n, need_g_log_decay=True).values()]

    far = torch.tensor([2 ** 63 - 1, 2 ** 32 + 5, 2 ** 31, -1, -2 ** 63, 77], device=DEV)
    want = call(torch.tensor([L, L, L, 0, 0, 77], dtype=torch.int32, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(call(far), want))
    assert all(torch.equal(a, b) for a, b in zip(call(far.clamp(-2 ** 15, 2 ** 15 - 1).short()), want))
    high = torch.tensor([2 ** 31 + 9, 2 ** 32 - 1, L, 0, 0, 77], device=DEV).to(torch.uint32)
    assert all(torch.equal(a, b) for a, b in zip(call(high), want))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("L", [700, 4000])
def test_a_value_that_is_no_number_stays_in_its_column(L, dtype):
    """A NaN value makes its column NaN from its token on, in its row and head; within its 128 tokens, whose products
    are formed together, earlier outputs may be NaN too, and nothing else changes."""
    from icml_b200 import ops
    g = _gen(L)
    q, k, v = (_n(g, 2, L, 2, 64).to(dtype) for _ in range(3))
    ld = torch.tensor([-0.1, -0.01], device=DEV)
    base = ops.decay_attn_fwd(q, k, v, ld)
    v = v.clone()
    v[0, 300, 1, 5] = math.nan
    out, end = ops.decay_attn_fwd(q, k, v, ld)
    assert bool(out[0, 300:, 1, 5].isnan().all()) and bool(end[0, 1, :, 5].isnan().all())
    out[0, 256:, 1, 5] = base[0][0, 256:, 1, 5]
    end[0, 1, :, 5] = base[1][0, 1, :, 5]
    assert torch.equal(out, base[0]) and torch.equal(end, base[1])
