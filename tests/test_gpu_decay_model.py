"""The decay-attention layer, its language model and its beam search on the GPU.

A layer is compared with autograd of its float64 statement at the bounds that every layer here is held to
(parity.py: 1e-4 of the largest element in float32, 3e-2 in the 2-norm with bfloat16 activations).
"""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import pgf_oracle as PO
from tests import decay_oracle as O
from tests.parity import BF16_RTOL, assert_close, rel_err

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(2, 300, 128, 64, 2, 1), (1, 129, 96, 24, 3, 3), (3, 1, 64, 8, 1, 1), (2, 70, 80, 33, 5, 1)]  # B L d Dk H Hk


def _block(shape, seed=0):
    from icml_b200.pgf_decay import PGFDecayBlock
    B, L, d, Dk, H, Hk = shape
    torch.manual_seed(seed + L)
    blk = PGFDecayBlock(d, Dk, 2 * d, 128, H, Hk)
    with torch.no_grad():
        for p in (blk.norm1.weight, blk.norm2.weight, blk.mixer.q_norm, blk.mixer.k_norm, blk.mixer.out_norm.weight, blk.b1, blk.b2):
            p.add_(0.1 * torch.randn_like(p))
    return blk, torch.randn(B, L, d), torch.randn(B, L, d)


def _layer64(blk, p, x):
    m, eps = blk.mixer, blk.norm1.eps

    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w

    B, L, _ = x.shape
    q, k, v = m.heads(norm(x, p["norm1.weight"]) @ p["mixer.qkv_proj.weight"].t())
    pos = torch.arange(L, dtype=torch.float64).expand(B, L)
    R = m.d_state // 2 * 2
    q = O.norm_rotate(q, p["mixer.q_norm"], pos, R, 10000.0, "halves", eps)
    k = O.norm_rotate(k, p["mixer.k_norm"], pos, R, 10000.0, "halves", eps)
    o, _ = O.decay_attn(q, k, v, F.logsigmoid(p["mixer.decay"]), m.d_state ** -0.5, None, None)
    x1 = x + norm(o.flatten(-2), p["mixer.out_norm.weight"]) @ p["mixer.out_proj.weight"].t()
    f = PO.ffn_forward(norm(x1, p["norm2.weight"]).flatten(0, 1), p["W1"], p["b1"], p["W2"], p["b2"], "gelu")
    return f.view(x.shape) + x1


def _truth(blk, x, g):
    p = {k: v.detach().double().requires_grad_() for k, v in blk.named_parameters()}
    x = x.double().requires_grad_()
    y = _layer64(blk, p, x)
    gr = torch.autograd.grad(y, [x, *p.values()], g.double())
    return y.detach(), gr[0], dict(zip(p, gr[1:]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_layer_forward_and_backward(shape, dtype):
    blk, x, g = _block(shape)
    x, g = x.to(dtype), g.to(dtype)
    y_ref, gx_ref, g_ref = _truth(blk, x, g)
    blk.to(DEV)
    x, g = x.to(DEV), g.to(DEV)
    y, kept = blk.pgf_forward(x, return_ssm_states=True, keep_scan=True)
    again, none = blk.pgf_forward(x, return_ssm_states=True)
    assert none is None and torch.equal(y, again) and torch.equal(y, blk.pgf_forward(x))
    r = blk.pgf_backward(x, g)
    rk = blk.pgf_backward(x, g, ssm_states=kept)
    assert set(r["grads"]) == set(g_ref) == set(rk["grads"])
    if dtype == torch.float32:
        assert_close(y, y_ref, name="output")
        assert_close(r["grad_input"], gx_ref, name="grad_input")
        for k, v in g_ref.items():
            assert_close(r["grads"][k], v, name=k)
    else:
        assert rel_err(y, y_ref) < BF16_RTOL and rel_err(r["grad_input"], gx_ref) < BF16_RTOL
    for k in g_ref:
        assert torch.equal(r["grads"][k], rk["grads"][k]), k
    if dtype == torch.float32:
        xa = x.clone().requires_grad_()
        blk(xa).backward(g)
        assert_close(xa.grad, gx_ref, name="autograd grad_input")
        for k, p in blk.named_parameters():
            assert_close(p.grad, g_ref[k], name=f"autograd {k}")


def test_functions_with_state_and_one_output():
    from icml_b200.pgf_decay import decay_attention
    torch.manual_seed(3)
    q, k, v = (torch.randn(2, 40, h, 16, device=DEV, requires_grad=True) for h in (4, 2, 1))
    ld = torch.tensor([-0.01, -0.2, -1.0, 0.0], device=DEV, requires_grad=True)
    s = torch.randn(2, 4, 16, 16, device=DEV, requires_grad=True)
    lens = torch.tensor([40, 13], device=DEV)
    leaves = [q, k, v, ld, s]
    out64 = O.decay_attn(*[t.detach().double().requires_grad_() for t in leaves[:4]], 0.25, s.detach().double(), lens)
    for which in (0, 1):  # the gradient of either output alone
        l64 = [t.detach().double().requires_grad_() for t in leaves]
        w64 = O.decay_attn(l64[0], l64[1], l64[2], l64[3], 0.25, l64[4], lens)[which]
        assert torch.equal(w64.detach(), out64[which].detach())
        co = torch.randn(w64.shape, device=DEV)
        ref = torch.autograd.grad(w64, l64, co.double(), allow_unused=True)
        got = torch.autograd.grad(decay_attention(q, k, v, ld, state=s, lengths=lens)[which], leaves, co, allow_unused=True)
        for n, a, b in zip("qkvds", got, ref):
            assert_close(a, torch.zeros_like(a, dtype=torch.float64) if b is None else b, name=f"output {which}, {n}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefill_and_steps_are_the_whole_sequence(dtype):
    blk, x, _ = _block((2, 300, 128, 64, 2, 1))
    blk.to(DEV)
    x = x.to(DEV, dtype)
    whole = blk.pgf_forward(x)
    # in two parts, and with a shorter second row followed by single tokens
    y0, s = blk.prefill(x[:, :170])
    y1, s_end = blk.prefill(x[:, 170:], state=s, start=170)
    parts = torch.cat([y0, y1], 1)
    lengths = torch.tensor([290, 11], device=DEV)
    y, s = blk.prefill(x[:, :290], lengths=lengths)
    pos = lengths.clone()
    singles = []
    for _ in range(10):
        xt = x[torch.arange(2, device=DEV), pos]
        yt, s = blk.step(xt, s, pos, out_state=s)
        singles.append(yt - whole[torch.arange(2, device=DEV), pos])
        pos += 1
    off = torch.stack(singles)
    scale = whole.abs().max().item()
    if dtype == torch.float32:
        assert_close(parts, whole, name="two parts")
        assert off.abs().max().item() <= 1e-5 + 1e-4 * scale
        assert_close(s[0], s_end[0], name="state behind the sequence")
    else:
        assert rel_err(parts, whole) < BF16_RTOL
        assert off.norm().item() < BF16_RTOL * torch.stack([whole[0, 290:].norm(), whole[1, 11:21].norm()]).norm().item()


def _model(dtype=torch.float32, vocab=61, layers=2, n_heads=2, n_kv_heads=1):
    from icml_b200.lm import PGFLanguageModel
    torch.manual_seed(11)
    return PGFLanguageModel(vocab, 64, 32, 128, layers, 64, DEV, act_dtype=dtype, init_std=0.3, variant="decay",
                            final_norm=True, n_heads=n_heads, n_kv_heads=n_kv_heads)


@pytest.mark.parametrize("stash", ["device", "scan"])
def test_model_step_gradients(stash):
    from icml_b200 import lm
    m = _model()
    m.stash = lm.LayerStash(stash)
    ids = torch.randint(61, (2, 65), generator=torch.Generator().manual_seed(5))
    loss, grads = m.forward_backward(ids[:, :-1].to(DEV), ids[:, 1:].to(DEV))
    emb, head = (w.detach().cpu().double().requires_grad_() for w in (m.emb_weight, m.lm_head_weight))
    fw = m.final_norm.weight.detach().cpu().double().requires_grad_()
    x = emb[ids[:, :-1]]
    ps = []
    for layer in m.backbone.layers:
        p = {k: v.detach().cpu().double().requires_grad_() for k, v in layer.named_parameters()}
        x = _layer64(layer, p, x)
        ps.append(p)
    x = x / (x.square().mean(-1, keepdim=True) + m.final_norm.eps).sqrt() * fw
    ref = F.cross_entropy((x @ head.t()).flatten(0, 1), ids[:, 1:].flatten())
    ref.backward()
    assert abs(loss.item() - ref.item()) <= 1e-5 + 1e-4 * abs(ref.item())
    assert_close(grads["emb"], emb.grad, name="emb")
    assert_close(grads["lm_head"], head.grad, name="lm_head")
    assert_close(grads["final_norm"], fw.grad, name="final_norm")
    for i, p in enumerate(ps):
        for k, v in p.items():
            assert_close(grads[f"layers.{i}.{k}"], v.grad, name=f"layers.{i}.{k}")


def _plain_search(m, ids, n, steps, K, end):
    """Beams of one prompt, each step from whole forward passes over every beam's tokens."""
    from icml_b200.generate import prefill
    beams = [(0.0, [], False)]
    for _ in range(steps):
        cand = []
        for r, (s, t, done) in enumerate(beams):
            if done:
                cand.append((s, t + [end], True))
                continue
            seq = torch.tensor([ids[:n] + t], device=DEV)
            lp = torch.log_softmax(prefill(m, seq)[0].double(), -1)[0]
            top = lp.topk(min(K + 1, lp.numel()))
            cand += [(s + v, t + [c], c == end) for v, c in zip(top.values.tolist(), top.indices.tolist())]
        cand.sort(key=lambda c: -c[0])
        beams = cand[:K]
    return beams


@pytest.mark.parametrize("beams,end", [(1, None), (4, None), (5, 7), (3, 0)])
def test_beam_search_against_whole_forward_passes(beams, end):
    from icml_b200.generate import beam_search
    m = _model()
    ids = torch.randint(61, (3, 9), generator=torch.Generator().manual_seed(2))
    lengths = torch.tensor([9, 1, 4])
    steps = 6
    tokens, scores, done = beam_search(m, ids.to(DEV), steps, beams, lengths.to(DEV), end)
    assert tokens.shape == (3, beams, steps) and bool((scores[:, 1:] <= scores[:, :-1]).all())
    for b in range(3):
        want = _plain_search(m, ids[b].tolist(), int(lengths[b]), steps, beams, end)
        # a score is a float32 sum of six log probabilities of a float32 model
        assert max(abs(scores[b, k].item() - want[k][0]) for k in range(beams)) < 2e-3
        if min([want[k][0] - want[k + 1][0] for k in range(beams - 1)], default=1.0) > 4e-3:
            assert tokens[b].tolist() == [w[1] for w in want]
            assert done[b].tolist() == [w[2] for w in want]


def test_beam_search_in_bfloat16_and_its_refusals():
    from icml_b200.generate import beam_search
    from icml_b200.lm import PGFLanguageModel
    m = _model(torch.bfloat16)
    ids = torch.zeros(2, 5, dtype=torch.int64, device=DEV)
    tokens, scores, _ = beam_search(m, ids, 4, 32)
    assert bool(torch.isfinite(scores).all()) and int(tokens.max()) < 61
    tokens, scores, _ = beam_search(m, ids, 1, 2)
    assert tokens.shape == (2, 2, 1)
    for kw in (dict(steps=0), dict(steps=1, beams=33), dict(steps=1, beams=0),
               dict(steps=1, lengths=torch.tensor([0, 3], device=DEV))):
        with pytest.raises(ValueError):
            beam_search(m, ids, **kw)
    with pytest.raises(ValueError):
        beam_search(m, ids[:, :0], 1)
    std = PGFLanguageModel(61, 64, 16, 128, 1, 64, DEV, variant="std")
    with pytest.raises(ValueError):
        beam_search(std, ids, 1)


def test_example_runs_and_learns():
    from icml_b200 import generate
    right = generate.main(["--train-steps", "120", "--steps", "6"])
    # chance is 1 in 64 for each of 24 tokens; a third of them is out of its reach
    assert right > 1 / 3


def test_training_step_in_a_graph():
    from icml_b200.lm import GraphedStep
    m = _model(torch.bfloat16)
    ids = torch.randint(61, (2, 65), generator=torch.Generator().manual_seed(5)).to(DEV)
    x, y = ids[:, :-1].contiguous(), ids[:, 1:].contiguous()
    g = GraphedStep(m, x, y)
    first = g.run(x, y).item()
    for _ in range(20):
        last = g.run(x, y)
    assert math.isfinite(first) and last.item() < first
    g.release()


# ------------------------------------------------------------------------- operators' remaining forms
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_without_the_final_state(dtype):
    from icml_b200 import ops
    torch.manual_seed(1)
    q, k, v = (torch.randn(2, 700, 2, 64, device=DEV).to(dtype) for _ in range(3))
    ld = torch.tensor([-0.02, -0.5], device=DEV)
    out, end = ops.decay_attn_fwd(q, k, v, ld)
    bare, none = ops.decay_attn_fwd(q, k, v, ld, want_state=False)
    assert none is None and end.shape == (2, 2, 64, 64)
    # bfloat16 keeps fewer terms of the keys inside when no state leaves: at most one more rounding of 2^-16
    assert (out.double() - bare.double()).norm() <= (1e-5 if dtype == torch.float32 else 6e-3) * out.double().norm()


@pytest.mark.parametrize("V,dtype", [(300_000, torch.bfloat16), (450_001, torch.float32), (1_000_003, torch.bfloat16)])
def test_beam_select_over_large_vocabularies(V, dtype):
    """A block's share of one beam is more than an SM holds."""
    from icml_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = (3 * torch.randn(2, 3, V, generator=g, device=DEV)).to(dtype)
    scores = -torch.rand(2, 3, generator=g, device=DEV)
    so, rows, tokens, _ = ops.beam_select(logits, scores)
    c = O.beam_candidates(logits, scores, None, 0)
    want, at = torch.sort(c, dim=1, descending=True, stable=True)
    assert torch.allclose(so, want[:, :3], rtol=3e-7, atol=2e-6)
    flat = (rows - 3 * torch.arange(2, device=DEV)[:, None]) * V + tokens
    assert torch.allclose(so, c.gather(1, flat), rtol=3e-7, atol=2e-6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,Hk", [(1, 4000, 2, 1), (3, 300, 60, 60)])  # cut into pieces; more heads than SMs
def test_calls_in_a_graph_and_back_to_back(B, L, H, Hk, dtype):
    """The launches of a call overlap one another but neither the calls before nor those behind: replays and
    calls in close order, each with the inputs overwritten in between, give the bits of calls on their own."""
    from icml_b200 import ops
    torch.manual_seed(L)
    sets = [[torch.randn(B, L, h, 64, device=DEV).to(dtype) for h in (H, Hk, Hk, H)] for _ in range(4)]
    ld = -torch.rand(H, device=DEV) * 0.1 - 1e-3

    def call(q, k, v, g):
        out, end = ops.decay_attn_fwd(q, k, v, ld)
        r = ops.decay_attn_bwd(q, k, v, ld, g, need_g_log_decay=True)
        return [out, end, *[r[n] for n in sorted(r)]]

    alone = []
    for s in sets:
        torch.cuda.synchronize()
        alone.append(call(*s))
        torch.cuda.synchronize()
    buf = [t.clone() for t in sets[0]]
    close = []
    for s in sets * 3:
        for d, t in zip(buf, s):
            d.copy_(t)
        close.append([t.clone() for t in call(*buf)])
    for i, got in enumerate(close):
        assert all(torch.equal(a, b) for a, b in zip(got, alone[i % 4])), i
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(*buf)
    for i in (2, 0, 3):
        for d, t in zip(buf, sets[i]):
            d.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, alone[i])), f"replay {i}"
    graph.reset()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_at_any_address(dtype):
    """States that begin 4 bytes behind a 16-byte boundary: the same results within both paths' roundings."""
    from icml_b200 import ops
    torch.manual_seed(8)
    q, k, v, g = (torch.randn(2, 300, 3, 64, device=DEV).to(dtype) for _ in range(4))
    ld = torch.tensor([-0.01, -0.1, -1.0], device=DEV)
    s, gs = torch.randn(2, 3, 64, 64, device=DEV), torch.randn(2, 3, 64, 64, device=DEV)

    def moved(t):
        u = torch.empty(t.numel() + 1, device=DEV)[1:].view(t.shape)
        u.copy_(t)
        assert u.is_contiguous() and u.data_ptr() % 16 == 4
        return u

    def call(s, gs):
        out, end = ops.decay_attn_fwd(q, k, v, ld, state=s)
        r = ops.decay_attn_bwd(q, k, v, ld, g, state=s, g_state=gs, need_g_log_decay=True)
        one, new = ops.decay_attn_step(q[:, 0], k[:, 0], v[:, 0], ld, s)
        return dict(r, out=out, end=end, one=one, new=new)

    a, b = call(s, gs), call(moved(s), moved(gs))
    for n, t in a.items():
        # float32 results: 1e-5 each; bfloat16: three roundings of 2^-9 each
        tol = 2 * (1e-5 if t.dtype == torch.float32 else 6e-3)
        assert (t.double() - b[n].double()).norm() <= tol * t.double().norm(), n
