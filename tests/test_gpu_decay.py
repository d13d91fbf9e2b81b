"""The decay-attention layer's operators on the GPU against float64.

Tolerances, relative in the 2-norm over each (batch row, head), set from the arithmetic:
* float32 results are float32 sums of at most about 1,000 terms; with roundings of 2^-24 that add up
  like a random walk a result is off by about sqrt(1000) 2^-24 = 2e-6 of its terms' norm, and 1e-5 leaves
  room for sums that cancel by a factor of five.
* bfloat16 results take one rounding at the end (2^-9 at most) and, inside, at most one of the scores and
  one of the state: three roundings, 3 x 2^-9 = 5.9e-3 if they all add up.
Sums over tokens or heads that come back as float32 (grad_w, grad_log_decay, states) keep the float32 bound
for either type, as their inputs are exact and nothing in them is rounded to 16 bits.
"""
import math
import zlib

import pytest
import torch

from tests import decay_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: 1e-5, torch.bfloat16: 6e-3}
BOTH = [torch.float32, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _n(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _close(got, ref, tol, name, slices=0, size=None):
    """|got - ref| <= tol |ref| in the 2-norm of every slice over the first `slices` dimensions; size: the
    norm of the terms instead of the result's, where the terms of a single element may cancel."""
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    got, ref = got.double(), ref.double()
    assert torch.isfinite(got).all(), name
    n = math.prod(ref.shape[:slices])
    err = (got - ref).reshape(n, -1).norm(dim=1)
    lim = tol * (ref if size is None else size).reshape(n, -1).norm(dim=1)
    assert bool((err <= lim + 1e-30).all()), f"{name}: {(err / lim.clamp_min(1e-30)).max().item():.2f} times the bound"


# ------------------------------------------------------------------------------------- norm and rotation
QK = [  # B, L, Hq, Hk, D, R, pairs
    (1, 1, 1, 1, 64, 64, "halves"), (2, 7, 3, 1, 128, 128, "halves"), (1, 300, 16, 4, 64, 32, "halves"),
    (3, 33, 2, 2, 80, 16, "neighbours"), (2, 65, 4, 2, 256, 256, "neighbours"), (1, 5, 2, 1, 33, 32, "halves"),
    (2, 9, 1, 3, 17, 0, "halves"), (64, 1, 8, 8, 96, 96, "neighbours"), (1, 19, 2, 0, 48, 24, "halves"),
    (1, 1201, 12, 12, 16, 16, "halves"), (1, 3, 1, 1, 1, 0, "halves"), (1, 40, 3, 2, 255, 254, "neighbours"),
]


def _qk(case, dtype, packed=True):
    B, L, Hq, Hk, D, R, pairs = case
    g = _gen(zlib.crc32(repr(case).encode()))
    row = _n(g, B, L, Hq + 2 * Hk, D).to(dtype)
    q, k = row[:, :, :Hq], row[:, :, Hq:Hq + Hk]
    pos = torch.randint(0, 1_000_000, (B, L), generator=g, device=DEV)
    return g, q, k, 1 + 0.2 * _n(g, D), 1 + 0.2 * _n(g, D), pos


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("case", QK, ids=str)
def test_norm_rotate_forward_and_backward(case, dtype):
    from icml_b200 import ops
    B, L, Hq, Hk, D, R, pairs = case
    g, q, k, wq, wk, pos = _qk(case, dtype)
    turns = ops.rotary_turns(R, 10000.0, DEV)
    kw = dict(positions=pos, eps=1e-5, pairs=pairs)
    qo, ko = ops.qk_norm_rotate_fwd(q, k, wq, wk, turns, **kw)
    gq, gk = _n(g, *q.shape).to(dtype), _n(g, *k.shape).to(dtype)
    r = ops.qk_norm_rotate_bwd(q, k, gq, gk, wq, wk, turns, **kw)
    for x, w, out, go, gx, gw in ((q, wq, qo, gq, r["grad_q"], r["grad_wq"]), (k, wk, ko, gk, r["grad_k"], r["grad_wk"])):
        if x.numel() == 0:
            assert out.shape == x.shape and not gw.any()
            continue
        xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
        ref = O.norm_rotate(xd, wd, pos, R, 10000.0, pairs, 1e-5)
        ref.backward(go.double())
        _close(out, ref, TOL[dtype], "out")
        # D = 1: the norm's gradient is a difference that all but vanishes; its terms set the scale
        if D > 1:
            _close(gx, xd.grad, TOL[dtype], "grad_x")
        _close(gw, wd.grad, 1e-5, "grad_w")


def test_norm_rotate_defaults_and_accumulation():
    """No weights, no rotation, positions from a start, one position row for the batch; gradients of
    weights added into buffers; layouts that need a copy give the same bits."""
    from icml_b200 import ops
    case = (2, 31, 4, 2, 64, 64, "halves")
    g, q, k, wq, wk, _ = _qk(case, torch.bfloat16)
    turns = ops.rotary_turns(64, 10000.0, DEV)
    at = torch.arange(900000, 900031, device=DEV)
    a = ops.qk_norm_rotate_fwd(q, k, wq, wk, turns, start=900000)
    for b in (ops.qk_norm_rotate_fwd(q, k, wq, wk, turns, positions=at),
              ops.qk_norm_rotate_fwd(q.contiguous(), k.transpose(2, 3).contiguous().transpose(2, 3), wq, wk, turns,
                                     positions=at.expand(2, 31).int()),
              ops.qk_norm_rotate_fwd(q.transpose(1, 2).contiguous().transpose(1, 2), k, wq, wk, turns, start=900000)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    plain = ops.qk_norm_rotate_fwd(q, k)
    zero = torch.zeros(2, 31, device=DEV)
    _close(plain[0], O.norm_rotate(q.double(), None, zero, 0, 1.0, "halves", 1e-6), TOL[torch.bfloat16], "plain")
    gq, gk = _n(g, *q.shape).bfloat16(), _n(g, *k.shape).bfloat16()
    r = ops.qk_norm_rotate_bwd(q, k, gq, gk, wq, wk, turns, start=900000)
    acc = {"grad_wq": _n(g, 64), "grad_wk": _n(g, 64)}
    want = {n: t.clone() + r[n] for n, t in acc.items()}
    r2 = ops.qk_norm_rotate_bwd(q, k, gq, gk, wq, wk, turns, start=900000, acc=acc)
    assert r2["grad_wq"] is acc["grad_wq"] and all(torch.equal(acc[n], want[n]) for n in acc)
    assert set(ops.qk_norm_rotate_bwd(q, k, gq, gk)) == {"grad_q", "grad_k"}


def test_norm_rotate_gradient_against_differences():
    """Directional derivative of sum(out * G) by central differences of the float32 forward.  With a step of
    2^-6 the difference's own error is about step^2 / 6 = 4e-5 of the third derivative, and the forward's
    rounding 1e-6 / 2^-6 = 6e-5: 1e-3 holds both."""
    from icml_b200 import ops
    case = (2, 13, 4, 2, 48, 32, "neighbours")
    g, q, k, wq, wk, pos = _qk(case, torch.float32)
    turns = ops.rotary_turns(32, 10000.0, DEV)
    kw = dict(positions=pos, pairs="neighbours")
    gq, gk = _n(g, *q.shape), _n(g, *k.shape)
    r = ops.qk_norm_rotate_bwd(q, k, gq, gk, wq, wk, turns, **kw)
    d = [_n(g, *t.shape) for t in (q, k, wq, wk)]

    def f(e):
        a, b = ops.qk_norm_rotate_fwd(q + e * d[0], k + e * d[1], wq + e * d[2], wk + e * d[3], turns, **kw)
        return (a.double() * gq).sum() + (b.double() * gk).sum()

    e = 2.0 ** -6
    num = (f(e) - f(-e)) / (2 * e)
    parts = [(r[n].double() * t).sum() for n, t in zip(("grad_q", "grad_k", "grad_wq", "grad_wk"), d)]
    scale = sum((r[n].double() * t).square().sum() for n, t in zip(("grad_q", "grad_k", "grad_wq", "grad_wk"), d)).sqrt()
    assert abs(num - sum(parts)) <= 1e-3 * (scale + num.abs())


# ------------------------------------------------------------------------------------ attention, prompts
ATTN = [  # B, L, H, Hq, Hk, Hv, Dk, Dv
    (1, 1, 1, 1, 1, 1, 64, 64), (2, 2, 2, 2, 2, 2, 16, 16), (1, 127, 2, 2, 2, 2, 64, 64), (1, 128, 2, 1, 2, 2, 64, 64),
    (3, 129, 2, 2, 1, 2, 64, 64), (2, 300, 4, 2, 1, 4, 128, 128), (1, 513, 3, 3, 3, 1, 64, 128),
    (1, 385, 2, 2, 2, 2, 128, 64), (2, 200, 2, 2, 2, 2, 33, 17), (1, 70, 1, 1, 1, 1, 256, 40), (1, 65, 2, 2, 2, 2, 40, 200),
    (1, 700, 1, 1, 1, 1, 48, 80), (5, 31, 6, 3, 2, 6, 96, 8), (1, 260, 2, 2, 2, 2, 8, 120), (2, 64, 2, 2, 2, 2, 1, 1),
    (40, 150, 8, 8, 8, 8, 64, 64),
]


def _attn(case, dtype, state=True, seed=0):
    B, L, H, Hq, Hk, Hv, Dk, Dv = case
    g = _gen(seed + zlib.crc32(repr(case).encode()))
    q, k, v = _n(g, B, L, Hq, Dk).to(dtype), _n(g, B, L, Hk, Dk).to(dtype), _n(g, B, L, Hv, Dv).to(dtype)
    ld = -torch.exp2(-1.0 - torch.arange(H, device=DEV) * 1.5).float()
    s = _n(g, B, H, Dk, Dv) if state else None
    return g, q, k, v, ld, s


def _ref(q, k, v, ld, scale, state, lengths, go=None, gs=None):
    leaves = [t.double().requires_grad_() for t in (q, k, v, ld)]
    s = torch.zeros(q.shape[0], ld.numel(), q.shape[-1], v.shape[-1], dtype=torch.float64, device=DEV) \
        if state is None else state.double()
    s.requires_grad_()
    o, end = O.decay_attn(*leaves, scale, s, lengths)
    if go is None:
        return o.detach(), end.detach()
    loss = (o * go.double()).sum()
    if gs is not None:
        loss = loss + (end * gs.double()).sum()
    return o.detach(), end.detach(), torch.autograd.grad(loss, leaves + [s])


def _check_all(q, k, v, ld, state, lengths, go, gs, dtype, scale=None):
    from icml_b200 import ops
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    o, end, grads = _ref(q, k, v, ld, sc, state, lengths, go, gs)
    out, e = ops.decay_attn_fwd(q, k, v, ld, scale=scale, state=state, lengths=lengths)
    r = ops.decay_attn_bwd(q, k, v, ld, go, scale=scale, state=state, g_state=gs, lengths=lengths, need_g_log_decay=True)
    t = TOL[dtype]
    _close(out.transpose(1, 2), o.transpose(1, 2), t, "out", 2)
    _close(e, end, 1e-5, "state", 2)
    for name, ref in zip(("grad_q", "grad_k", "grad_v"), grads):
        _close(r[name].transpose(1, 2), ref.transpose(1, 2), t, name, 2)
    _close(r["grad_state"], grads[4], 1e-5, "grad_state", 2)
    # every head's decay sums terms of either sign over all tokens; its own terms set the scale
    lim = 1e-5 * (grads[3].abs() + grads[3].norm()) + 1e-6 * (go.double().square().sum() * o.square().sum()).sqrt()
    assert bool(((r["grad_log_decay"] - grads[3]).abs() <= lim).all()), (r["grad_log_decay"], grads[3])
    return out, e, r


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("case", ATTN, ids=str)
def test_attention_forward_and_backward(case, dtype):
    B, L, H, Hq, Hk, Hv, Dk, Dv = case
    g, q, k, v, ld, s = _attn(case, dtype)
    go, gs = _n(g, B, L, H, Dv).to(dtype), _n(g, B, H, Dk, Dv)
    _check_all(q, k, v, ld, s, None, go, gs, dtype)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("case", [(6, 301, 2, 2, 2, 2, 64, 64), (6, 260, 4, 2, 1, 4, 128, 128), (6, 100, 2, 2, 2, 2, 24, 40),
                                  (6, 90, 1, 1, 1, 1, 19, 5)], ids=str)
def test_attention_lengths_hide_what_lies_behind_them(case, dtype):
    """Rows of length 0, 1, a chunk's edge and all; NaN and infinities behind them change nothing, and
    the outputs and gradients there are zeros."""
    B, L, H, Hq, Hk, Hv, Dk, Dv = case
    g, q, k, v, ld, s = _attn(case, dtype)
    n = torch.tensor([0, 1, min(64, L), L, L // 2 + 1, L - 1], device=DEV)
    go, gs = _n(g, B, L, H, Dv).to(dtype), _n(g, B, H, Dk, Dv)
    behind = (torch.arange(L, device=DEV) >= n[:, None])
    dirty = []
    for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (go, -math.inf)):
        t = t.clone()
        t[behind] = bad
        dirty.append(t)
    clean = [torch.where(behind[..., None, None], 0.0, t.float()).to(dtype) for t in (q, k, v, go)]
    from icml_b200 import ops
    out, e, r = _check_all(*clean[:3], ld, s, n, clean[3], gs, dtype)
    out2, e2 = ops.decay_attn_fwd(*dirty[:3], ld, state=s, lengths=n)
    r2 = ops.decay_attn_bwd(*dirty[:3], ld, dirty[3], state=s, g_state=gs, lengths=n, need_g_log_decay=True)
    assert torch.equal(out, out2) and torch.equal(e, e2) and all(torch.equal(r[x], r2[x]) for x in r)
    assert torch.equal(e[0], s[0])
    for t in (out2, r2["grad_q"], r2["grad_k"], r2["grad_v"]):
        assert not t[behind].any()


@pytest.mark.parametrize("dtype", BOTH)
def test_attention_extreme_decays(dtype):
    """No decay at all, a decay of zero (each token sees itself alone), and one that forgets within a token."""
    case = (1, 200, 3, 3, 3, 3, 64, 64)
    g, q, k, v, _, s = _attn(case, dtype)
    ld = torch.tensor([0.0, -math.inf, -30.0], device=DEV)
    from icml_b200 import ops
    out, e = ops.decay_attn_fwd(q, k, v, ld, state=s)
    ref, end = _ref(q, k, v, ld.clamp(min=-1e4), 64 ** -0.5, s, None)
    _close(out.transpose(1, 2), ref.transpose(1, 2), TOL[dtype], "out", 2)
    _close(e, end, 1e-5, "state", 2)
    go, gs = _n(g, 1, 200, 3, 64).to(dtype), _n(g, 1, 3, 64, 64)
    r = ops.decay_attn_bwd(q, k, v, ld, go, state=s, g_state=gs)
    _, _, grads = _ref(q, k, v, ld.clamp(min=-1e4), 64 ** -0.5, s, None, go, gs)
    for name, want in zip(("grad_q", "grad_k", "grad_v"), grads):
        _close(r[name].transpose(1, 2), want.transpose(1, 2), TOL[dtype], name, 2)


@pytest.mark.parametrize("dtype", BOTH)
def test_attention_views_streams_and_repeats(dtype):
    """Parts of one projection, head-major and odd-pitched layouts, another stream: the same bits each time."""
    from icml_b200 import ops
    B, L, H, D = 2, 333, 4, 64
    g = _gen(5)
    row = _n(g, B, L, 3 * H, D).to(dtype)
    q, k, v = (row[:, :, i * H:(i + 1) * H] for i in range(3))
    ld = -torch.exp2(-2.0 - torch.arange(H, device=DEV)).float()
    go = _n(g, B, L, H, D).to(dtype)

    def run(q, k, v, go):
        o, e = ops.decay_attn_fwd(q, k, v, ld)
        return [o, e] + list(ops.decay_attn_bwd(q, k, v, ld, go, need_g_log_decay=True).values())

    base = run(*(t.contiguous() for t in (q, k, v, go)))
    for other in ((q, k, v, go), tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, go)),
                  tuple(t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v, go))):
        assert all(torch.equal(a, b) for a, b in zip(base, run(*other)))
    wide = torch.zeros(B, L, H, D + 1, dtype=dtype, device=DEV)  # a pitch that 16-byte loads cannot take
    odd = []
    for t in (q, k, v, go):
        w = wide.clone()
        w[..., :D] = t
        odd.append(w[..., :D])
    for a, b in zip(base, run(*odd)):
        _close(b, a, TOL[dtype] if a.dtype == dtype else 1e-5, "odd pitch")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        there = run(q, k, v, go)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(base, there))


def test_attention_in_pieces_is_the_whole():
    """A prompt walked in two calls through the state, then token by token."""
    from icml_b200 import ops
    case = (2, 400, 2, 2, 2, 2, 64, 64)
    _, q, k, v, ld, _ = _attn(case, torch.float32)
    o, e = ops.decay_attn_fwd(q, k, v, ld)
    a, s = ops.decay_attn_fwd(q[:, :377], k[:, :377], v[:, :377], ld)
    b, s = ops.decay_attn_fwd(q[:, 377:390], k[:, 377:390], v[:, 377:390], ld, state=s)
    c = []
    for t in range(390, 400):
        x, s = ops.decay_attn_step(q[:, t], k[:, t], v[:, t], ld, s, out_state=s if t % 2 else None)
        c.append(x[:, None])
    _close(torch.cat([a, b] + c, 1), o, 1e-5, "out")
    _close(s, e, 1e-5, "state")


def test_attention_gradient_against_differences():
    """The loss is linear in q, in k, in v and in each state, so central differences along one of them are
    exact but for rounding (1e-6 / step); along ln(decay) the step^2 term adds 2^-16."""
    from icml_b200 import ops
    case = (1, 150, 2, 2, 1, 2, 24, 40)
    g, q, k, v, ld, s = _attn(case, torch.float32)
    go, gs = _n(g, 1, 150, 2, 40), _n(g, 1, 2, 24, 40)
    r = ops.decay_attn_bwd(q, k, v, ld, go, state=s, g_state=gs, need_g_log_decay=True)

    def f(q, k, v, ld, s):
        o, e = ops.decay_attn_fwd(q, k, v, ld, state=s)
        return (o.double() * go).sum() + (e.double() * gs).sum()

    args = [q, k, v, ld, s]
    for i, name in enumerate(("grad_q", "grad_k", "grad_v", "grad_log_decay", "grad_state")):
        d, e = _n(g, *args[i].shape), (2.0 ** -8 if name == "grad_log_decay" else 1.0)
        if name == "grad_log_decay":
            d = d * ld.abs()  # relative to each head's own
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + e * d, args[i] - e * d
        num = (f(*hi) - f(*lo)) / (2 * e)
        got = (r[name].double() * d).sum()
        size = (r[name].double() * d).norm() + got.abs()
        assert abs(num - got) <= 2e-3 * size, (name, num, got)


# -------------------------------------------------------------------------------------- attention, steps
STEP = [(1, 1, 1, 1, 1, 64, 64), (3, 4, 2, 1, 4, 128, 128), (130, 8, 8, 8, 8, 64, 64), (2, 3, 3, 3, 1, 33, 17),
        (1, 2, 2, 2, 2, 256, 256), (2, 2, 1, 2, 2, 16, 80), (300, 2, 2, 2, 2, 1, 1)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("case", STEP, ids=str)
def test_step(case, dtype):
    from icml_b200 import ops
    B, H, Hq, Hk, Hv, Dk, Dv = case
    g = _gen(3)
    row = _n(g, B, Hq + Hk, Dk).to(dtype)
    q, k, v = row[:, :Hq], row[:, Hq:], _n(g, B, Hv, Dv).to(dtype)
    ld = -torch.exp2(-2.0 - torch.arange(H, device=DEV)).float()
    n = B + 3
    s = _n(g, n, H, Dk, Dv)
    rows = torch.randint(0, n, (B,), generator=g, device=DEV)
    keep = s.clone()
    o, new = ops.decay_attn_step(q, k, v, ld, s, rows=rows)
    ro, rs = O.decay_step(q.double(), k.double(), v.double(), ld.double(), s[rows].double(), Dk ** -0.5)
    assert torch.equal(s, keep)
    _close(o, ro, TOL[dtype], "out")
    terms = lambda s: O.decay_step(q.double(), k.double().abs(), v.double().abs(), ld.double(), s.double().abs(), 1.0)[1]  # noqa: E731
    _close(new, rs, 1e-6, "state", 2, terms(s[rows]))  # a rounding of each term and one of their sum
    own = s[:B].clone()
    o2, new2 = ops.decay_attn_step(q, k, v, ld, own, out_state=own, scale=0.5)
    ro, rs = O.decay_step(q.double(), k.double(), v.double(), ld.double(), s[:B].double(), 0.5)
    assert new2 is own
    _close(o2, ro, TOL[dtype], "out in place")
    _close(own, rs, 1e-6, "state in place", 2, terms(s[:B]))


def test_step_out_of_range_rows_start_from_zeros():
    from icml_b200 import ops
    g = _gen(4)
    q, k, v, ld = _n(g, 2, 1, 16), _n(g, 2, 1, 16), _n(g, 2, 1, 16), torch.tensor([-0.1], device=DEV)
    s = _n(g, 2, 1, 16, 16)
    _, new = ops.decay_attn_step(q, k, v, ld, s, rows=torch.tensor([-1, 2], device=DEV))
    _close(new, k.double()[..., None] * v.double()[..., None, :], 1e-6, "state")


# -------------------------------------------------------------------------------------------------- beams
def _beam_check(logits, scores, finished, end):
    from icml_b200 import ops
    B, K, V = logits.shape
    so, rows, tokens, fin = ops.beam_select(logits, scores, finished, end_id=end)
    c = O.beam_candidates(logits, scores, finished, end if end is not None else 0)
    want, at = torch.sort(c, dim=1, descending=True, stable=True)
    first = K * torch.arange(B, device=DEV)[:, None]
    flat = (rows - first) * V + tokens
    assert bool(((rows >= first) & (rows < first + K) & (tokens >= 0) & (tokens < V)).all())
    # each chosen candidate is worth what is said of it, to a rounding of its log sum
    assert torch.allclose(so.double(), c.gather(1, flat).double(), rtol=3e-7, atol=2e-6)
    assert torch.allclose(so, want[:, :K], rtol=3e-7, atol=2e-6)
    assert bool((so[:, 1:] <= so[:, :-1]).all())
    same = (so[:, 1:] == so[:, :-1])
    assert bool((flat[:, 1:] > flat[:, :-1])[same].all()), "ties go to the lowest index"
    assert all(len(set(r)) == K for r in flat.tolist()), "a candidate twice"
    if finished is not None or end is not None:
        was = finished.view(-1)[rows] if finished is not None else torch.zeros_like(fin)
        assert torch.equal(fin, was | (tokens == (-1 if end is None else end)))
    return so, flat, at[:, :K]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 1, 50257), (3, 2, 7), (2, 3, 1000), (4, 4, 4099), (2, 5, 333), (3, 8, 50257),
                                   (2, 9, 515), (1, 16, 2050), (2, 17, 31), (1, 32, 5000), (2, 32, 32), (40, 7, 130)])
def test_beam_select(B, K, V, dtype):
    g = _gen(B * 1000 + K)
    logits, scores = (3 * _n(g, B, K, V)).to(dtype), -10 + _n(g, B, K)
    _, flat, at = _beam_check(logits, scores, None, None)
    if dtype == torch.float32:  # no two candidates are this close here
        assert (flat == at).float().mean() > 0.99
    finished = torch.rand(B, K, generator=g, device=DEV) < 0.4
    _beam_check(logits, scores, finished, V // 2)
    scores[:, 1:] = -math.inf
    _beam_check(logits, scores, None, V - 1)


def test_beam_select_ties_and_masks():
    """Equal logits everywhere (more ties than any list holds), rows of -inf, NaN and +inf, whole numbers
    only: the order is the index."""
    from icml_b200 import ops
    B, K, V = 2, 4, 30000
    logits = torch.zeros(B, K, V, device=DEV)
    scores = torch.zeros(B, K, device=DEV)
    so, rows, tokens, _ = ops.beam_select(logits, scores)
    assert torch.equal(tokens, torch.arange(K, device=DEV).expand(B, K)) and torch.equal(rows, 4 * torch.arange(B, device=DEV)[:, None].expand(B, K))
    logits[:, 0] = -math.inf           # a row with nothing left
    logits[0, 1, 5] = math.nan
    logits[1, 1, 5] = math.inf
    so, rows, tokens, _ = ops.beam_select(logits, scores)
    assert torch.equal(rows - 4 * torch.arange(B, device=DEV)[:, None], torch.full((B, K), 2, device=DEV))
    assert torch.equal(tokens, torch.arange(K, device=DEV).expand(B, K))
    logits[:] = -math.inf
    so, rows, tokens, _ = ops.beam_select(logits, scores)
    assert bool((so == -math.inf).all()) and torch.equal(tokens, torch.arange(K, device=DEV).expand(B, K))
    assert torch.equal(rows, 4 * torch.arange(B, device=DEV)[:, None].expand(B, K))
    logits = torch.randint(0, 3, (B, K, V), generator=_gen(1), device=DEV).float()
    _, flat, at = _beam_check(logits, torch.tensor([[-1.0, -1.0, -9.0, -9.0]] * B, device=DEV), None, None)


def test_beam_finished_rows_and_unaligned_logits():
    from icml_b200 import ops
    B, K, V, end = 2, 3, 101, 0
    g = _gen(8)
    buf = _n(g, B * K * V + 1).bfloat16()
    logits = buf[1:].view(B, K, V)
    scores = torch.tensor([[-1.0, -2.0, -3.0], [-math.inf, -5.0, -1.0]], device=DEV)
    done = torch.ones(B, K, dtype=torch.bool, device=DEV)
    so, rows, tokens, fin = ops.beam_select(logits, scores, done, end_id=end)
    assert torch.equal(so, torch.tensor([[-1.0, -2.0, -3.0], [-1.0, -5.0, -math.inf]], device=DEV))
    assert torch.equal(rows, torch.tensor([[0, 1, 2], [5, 4, 3]], device=DEV))
    assert torch.equal(tokens[:, :2], torch.zeros(2, 2, dtype=torch.int64, device=DEV)) and bool(fin.all())
    done[:] = False
    _beam_check(logits, scores, done, end)


def test_beam_reorder():
    from icml_b200 import ops
    g = _gen(9)
    states = [_n(g, 12, 2, 16, 16), _n(g, 12, 5).bfloat16(), torch.arange(12, device=DEV), _n(g, 12, 70000),
              torch.rand(12, 3, generator=g, device=DEV) < 0.5, torch.empty(12, 0, device=DEV)] + [_n(g, 12, 3) for _ in range(70)]
    rows = torch.randint(0, 12, (4, 5), generator=g, device=DEV)
    for got, s in zip(ops.beam_reorder(states, rows), states):
        assert torch.equal(got, s[rows.view(-1)])
    out = torch.empty(2, 2, 16, 16, device=DEV)
    (got,) = ops.beam_reorder(states[:1], torch.tensor([3, 12], device=DEV), out=[out])
    assert got is out and torch.equal(out[0], states[0][3]) and not out[1].any()
    assert ops.beam_reorder([], rows) == []


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from icml_b200 import ops
    z = lambda *s, d=torch.float32: torch.zeros(*s, dtype=d, device=DEV)  # noqa: E731
    q, k, v, ld, s = z(2, 8, 4, 16), z(2, 8, 2, 16), z(2, 8, 4, 24), z(4), z(2, 4, 16, 24)
    t = ops.rotary_turns(16, 10000.0, DEV)
    bad = [
        lambda: ops.qk_norm_rotate_fwd(q.cpu(), k.cpu()),
        lambda: ops.qk_norm_rotate_fwd(q, k.bfloat16()),
        lambda: ops.qk_norm_rotate_fwd(q.half(), k.half()),
        lambda: ops.qk_norm_rotate_fwd(q, z(2, 8, 2, 24)),
        lambda: ops.qk_norm_rotate_fwd(q, k, z(15)),
        lambda: ops.qk_norm_rotate_fwd(q, k, turns=ops.rotary_turns(18, 10000.0, DEV)),
        lambda: ops.qk_norm_rotate_fwd(q, k, turns=t, positions=z(2, 8)),
        lambda: ops.qk_norm_rotate_fwd(q, k, turns=t, positions=z(3, 8, d=torch.int64)),
        lambda: ops.qk_norm_rotate_fwd(q, k, turns=t, pairs="odd"),
        lambda: ops.qk_norm_rotate_fwd(z(1, 1, 1, 257), z(1, 1, 1, 257)),
        lambda: ops.qk_norm_rotate_bwd(q, k, q, q),
        lambda: ops.rotary_turns(7),
        lambda: ops.decay_attn_fwd(q.cpu(), k.cpu(), v.cpu(), ld.cpu()),
        lambda: ops.decay_attn_fwd(q, k, v.bfloat16(), ld),
        lambda: ops.decay_attn_fwd(q, k, v, z(6)),
        lambda: ops.decay_attn_fwd(q, k, v, ld.double()),
        lambda: ops.decay_attn_fwd(q, k, z(2, 9, 4, 24), ld),
        lambda: ops.decay_attn_fwd(q, z(2, 8, 2, 24), v, ld),
        lambda: ops.decay_attn_fwd(z(1, 1, 1, 257), z(1, 1, 1, 257), z(1, 1, 1, 8), z(1)),
        lambda: ops.decay_attn_fwd(q, k, v, ld, state=z(2, 4, 24, 16)),
        lambda: ops.decay_attn_fwd(q, k, v, ld, state=s.bfloat16()),
        lambda: ops.decay_attn_fwd(q, k, v, ld, lengths=z(2)),
        lambda: ops.decay_attn_fwd(q, k, v, ld, lengths=z(3, d=torch.int32)),
        lambda: ops.decay_attn_bwd(q, k, v, ld, q),
        lambda: ops.decay_attn_bwd(q, k, v, ld, z(2, 8, 4, 24), g_log_decay_acc=z(3)),
        lambda: ops.decay_attn_step(q[:, 0], k[:, 0], v[:, 0], ld, z(3, 4, 16, 24)),
        lambda: ops.decay_attn_step(q[:, 0], k[:, 0], v[:, 0], ld, s, rows=z(2)),
        lambda: ops.decay_attn_step(q[:, 0], k[:, 0], v[:, 0], ld, s, rows=z(2, d=torch.int64), out_state=s),
        lambda: ops.decay_attn_step(q[:, 0], k[:, 0], v[:, 0], ld, s.transpose(2, 3).contiguous().transpose(2, 3)),
        lambda: ops.beam_select(z(1, 2, 5), z(1, 3)),
        lambda: ops.beam_select(z(1, 33, 5), z(1, 33)),
        lambda: ops.beam_select(z(1, 2, 5, d=torch.float16), z(1, 2)),
        lambda: ops.beam_select(z(1, 2, 5), z(1, 2, d=torch.float64)),
        lambda: ops.beam_select(z(1, 2, 5), z(1, 2), z(1, 2, d=torch.bool)),
        lambda: ops.beam_select(z(1, 2, 5), z(1, 2), end_id=5),
        lambda: ops.beam_reorder([z(4, 2)], z(2)),
        lambda: ops.beam_reorder([z(4, 2), z(5, 2)], z(2, d=torch.int64)),
        lambda: ops.beam_reorder([z(4, 2)], z(2, d=torch.int64), out=[z(3, 2)]),
        lambda: ops.beam_reorder([s], z(2, d=torch.int64), out=[s]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            f()
            pytest.fail(f"call {i} was not refused", pytrace=False)


def test_empty_calls():
    from icml_b200 import ops
    z = lambda *s, d=torch.float32: torch.zeros(*s, dtype=d, device=DEV)  # noqa: E731
    a, b = ops.qk_norm_rotate_fwd(z(0, 5, 2, 16), z(0, 5, 1, 16))
    assert a.shape == (0, 5, 2, 16) and b.shape == (0, 5, 1, 16)
    r = ops.qk_norm_rotate_bwd(z(2, 0, 2, 16), z(2, 0, 1, 16), z(2, 0, 2, 16), z(2, 0, 1, 16), z(16), z(16))
    assert not r["grad_wq"].any() and not r["grad_wk"].any()
    s = _n(_gen(1), 2, 3, 16, 8)
    o, e = ops.decay_attn_fwd(z(2, 0, 3, 16), z(2, 0, 3, 16), z(2, 0, 3, 8), z(3), state=s)
    assert o.shape == (2, 0, 3, 8) and torch.equal(e, s)
    r = ops.decay_attn_bwd(z(2, 0, 3, 16), z(2, 0, 3, 16), z(2, 0, 3, 8), z(3), z(2, 0, 3, 8), state=s, g_state=s,
                           need_g_log_decay=True)
    assert torch.equal(r["grad_state"], s) and not r["grad_log_decay"].any()
    o, e = ops.decay_attn_fwd(z(0, 4, 3, 16), z(0, 4, 3, 16), z(0, 4, 3, 8), z(3))
    assert o.shape == (0, 4, 3, 8) and e.shape == (0, 3, 16, 8)
    o, e = ops.decay_attn_step(z(0, 3, 16), z(0, 3, 16), z(0, 3, 8), z(3), z(0, 3, 16, 8))
    assert o.shape == (0, 3, 8)
    so, *_ = ops.beam_select(z(0, 2, 9), z(0, 2))
    assert so.shape == (0, 2)
