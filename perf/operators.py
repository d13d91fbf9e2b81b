"""The decay-attention operators as a user calls them, with plain forms to time and compare them against.

Three operators: the per-head norm and rotation of queries and keys (forward, backward), linear attention
with a decay for each head (prompts, training backward, single tokens) and the selection step of a beam
search with the reordering of the recurrent states.  ``own`` picks what ``run`` computes: False, elementary
torch operations in float32; True, this repository's kernels (icml_b200.ops).
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ----------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token for each of 64 sequences: the norm and rotation of that step, latency only
        dict(name="rotate token", op="rotate", dir="fwd", dtype="bf16", B=64, L=1, Hq=8, Hk=8, D=64, R=64,
             pairs="halves", base=10000.0, start=700),
        # the training configuration of 16 x 2048 tokens at width 1024: queries and keys of one layer
        dict(name="rotate train", op="rotate", dir="fwd", dtype="bf16", B=16, L=2048, Hq=16, Hk=16, D=64, R=64,
             pairs="halves", base=10000.0, start=0),
        # its backward on one 65536-token segment of a long sequence, 128-wide heads
        dict(name="rotate grad segment", op="rotate", dir="bwd", dtype="bf16", B=1, L=65536, Hq=8, Hk=8, D=128,
             R=128, pairs="halves", base=500000.0, start=196608),
        # float32, neighbouring pairs, a part of the head rotated, fewer key heads, odd lengths
        dict(name="rotate grad odd", op="rotate", dir="bwd", dtype="f32", B=3, L=1531, Hq=6, Hk=2, D=80, R=32,
             pairs="neighbours", base=10000.0, start=5),
        # a 65536-token prompt (one segment of the long-sequence step) at width 1024: eight heads of 128
        dict(name="attention prompt", op="attn", dir="fwd", dtype="bf16", B=1, L=65536, H=8, Hq=8, Hk=8, Dk=128,
             Dv=128, ragged=False, slope=0.5, learn=False),
        # prompts of several lengths (some empty) in one call, narrow heads, one key head for two states
        dict(name="attention ragged", op="attn", dir="fwd", dtype="bf16", B=7, L=1999, H=8, Hq=4, Hk=4, Dk=64,
             Dv=64, ragged=True, slope=1.0, learn=False),
        # the training backward at 16 x 2048 tokens, width 1024
        dict(name="attention train", op="attn", dir="bwd", dtype="bf16", B=16, L=2048, H=16, Hq=16, Hk=16, Dk=64,
             Dv=64, ragged=False, slope=1.0, learn=True),
        # a float32 training backward of odd sizes (parity runs are float32)
        dict(name="attention grad odd", op="attn", dir="bwd", dtype="f32", B=2, L=777, H=6, Hq=6, Hk=3, Dk=48,
             Dv=80, ragged=True, slope=1.0, learn=True),
        # one decoded token of one sequence
        dict(name="step one", op="step", dtype="bf16", B=1, H=8, Dk=128, Dv=128, beams=False),
        # one decoded token of 16 sequences x 8 beams, each reading its parent's state
        dict(name="step beams", op="step", dtype="bf16", B=128, H=16, Dk=64, Dv=64, beams=True),
        # one step of a beam search for one sequence over the vocabulary of the language model
        dict(name="beam one", op="beam", dtype="f32", B=1, K=4, V=50257, late=False, H=8, Dk=64, Dv=64),
        # 16 sequences of 8 beams, some finished, bf16 logits, with the states of one layer brought in order
        dict(name="beam batch", op="beam", dtype="bf16", B=16, K=8, V=50257, late=True, H=16, Dk=64, Dv=64),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "attn", "attn", "attn", "step", "beam"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "rotate":
        D = rng.choice([16, 32, 48, 64, 80, 96, 128, 256])
        Hk = rng.choice([1, 2, 4, 8])
        Hq = Hk * rng.choice([1, 2, 3])
        tokens = _spread(rng, 1, min(65536, (1 << 26) // (D * (Hq + Hk))))
        B = min(tokens, rng.choice([1, 1, 2, 3, 8, 64]))
        return dict(op=op, dir=rng.choice(["fwd", "bwd"]), dtype=dtype, B=B, L=max(1, tokens // B), Hq=Hq, Hk=Hk, D=D,
                    R=rng.choice([D, D, D // 2]), pairs=rng.choice(["halves", "neighbours"]),
                    base=rng.choice([10000.0, 500000.0]), start=_spread(rng, 1, 900000))
    if op == "attn":
        H = rng.choice([1, 2, 4, 6, 8, 16])
        Hq = H // rng.choice([1, 1, 2]) if H % 2 == 0 else H
        Hk = H // rng.choice([1, 1, 2]) if H % 2 == 0 else H
        Dk = rng.choice([16, 32, 48, 64, 64, 96, 128, 128])
        Dv = rng.choice([Dk, Dk, 32, 64, 80, 128])
        train = rng.random() < 0.5
        tokens = _spread(rng, 1, min(65536, (1 << 24) // (H * (Dk + Dv)) if dtype == "f32" or train
                                     else (1 << 26) // (H * (Dk + Dv))))
        B = min(tokens, rng.choice([1, 1, 2, 5, 16]))
        return dict(op=op, dir="bwd" if train else "fwd", dtype=dtype, B=B, L=max(1, tokens // B), H=H, Hq=Hq, Hk=Hk,
                    Dk=Dk, Dv=Dv, ragged=rng.random() < 0.5, slope=round(rng.uniform(0.05, 2.0), 3),
                    learn=train and rng.random() < 0.5)
    if op == "step":
        H = rng.choice([1, 2, 4, 8, 16])
        Dk = rng.choice([16, 32, 48, 64, 96, 128])
        Dv = rng.choice([Dk, Dk, 32, 80, 128])
        return dict(op=op, dtype=dtype, B=_spread(rng, 1, max(1, min(256, (1 << 24) // (H * Dk * Dv)))), H=H, Dk=Dk,
                    Dv=Dv, beams=rng.random() < 0.5)
    K = rng.choice([1, 2, 3, 4, 5, 8])
    return dict(op=op, dtype=dtype, B=_spread(rng, 1, 16), K=K, V=_spread(rng, 500, 50257), late=rng.random() < 0.5,
                H=rng.choice([2, 4, 8]), Dk=rng.choice([32, 64]), Dv=rng.choice([32, 64]))


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _log_decay(c):
    """ln of each head's decay, ln(1 - 2^(-4 - slope h)): horizons from 16 tokens up, as layers of this kind are set."""
    h = torch.arange(c["H"], device=DEV, dtype=torch.float64)
    return torch.log1p(-torch.exp2(-4.0 - c.get("slope", 0.5) * h.clamp(max=12))).float()


def _turns(c, device=DEV):
    """The rotation's frequencies as 64-bit fixed-point fractions of a turn per position."""
    R = c["R"]
    f = c["base"] ** (-torch.arange(0, R, 2, dtype=torch.float64) / R) / (2 * math.pi)
    return (f * 2.0 ** 64).to(torch.int64).to(device)


def _unit(x, dtype):
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)).to(dtype)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = TYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "rotate":
        B, L, Hq, Hk, D = (c[k] for k in ("B", "L", "Hq", "Hk", "D"))
        # queries, keys and values of one projection, side by side in its rows; values pass by
        qkv = _normal(g, B, L, Hq + 2 * Hk, D).to(dt)
        s["q"], s["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
        s["wq"], s["wk"] = 1 + 0.1 * _normal(g, D), 1 + 0.1 * _normal(g, D)
        s["positions"] = (c["start"] + torch.arange(L, device=DEV)).expand(B, L).contiguous()
        if L == 1:  # sequences that decode together are not equally far
            s["positions"] = s["positions"] + torch.randint(0, 500, (B, 1), generator=g, device=DEV)
        s["turns"] = _turns(c)
        if c["dir"] == "bwd":
            s["gq"], s["gk"] = _normal(g, B, L, Hq, D).to(dt), _normal(g, B, L, Hk, D).to(dt)
    elif c["op"] == "attn":
        B, L, H, Hq, Hk, Dk, Dv = (c[k] for k in ("B", "L", "H", "Hq", "Hk", "Dk", "Dv"))
        s["q"], s["k"] = _unit(_normal(g, B, L, Hq, Dk), dt), _unit(_normal(g, B, L, Hk, Dk), dt)
        s["v"] = _normal(g, B, L, H, Dv).to(dt)
        s["log_decay"] = _log_decay(c)
        s["state"] = _normal(g, B, H, Dk, Dv)  # of what came before
        s["lengths"] = None
        if c["ragged"]:
            n = torch.randint(0, L + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
            n[0] = L
            if B > 1:
                n[-1] = 0
            s["lengths"] = n
        if c["dir"] == "bwd":
            s["g"], s["g_state"] = _normal(g, B, L, H, Dv).to(dt), _normal(g, B, H, Dk, Dv)
    elif c["op"] == "step":
        B, H, Dk, Dv = (c[k] for k in ("B", "H", "Dk", "Dv"))
        s["q"], s["k"] = _unit(_normal(g, B, H, Dk), dt), _unit(_normal(g, B, H, Dk), dt)
        s["v"] = _normal(g, B, H, Dv).to(dt)
        s["log_decay"] = _log_decay(c)
        s["state"] = 4 * _normal(g, B, H, Dk, Dv)
        s["next_state"] = torch.empty_like(s["state"])  # the program keeps two and takes them in turn
        s["rows"] = None
        if c["beams"]:
            n = 8
            r = torch.arange(B, device=DEV)
            s["rows"] = torch.minimum(r // n * n + torch.randint(0, n, (B,), generator=g, device=DEV),
                                      torch.full_like(r, B - 1))
    else:
        B, K, V = c["B"], c["K"], c["V"]
        s["logits"] = (2.5 * _normal(g, B, K, V)).to(dt)
        s["scores"] = -12 + 1.5 * _normal(g, B, K)
        s["finished"] = torch.zeros(B, K, dtype=torch.bool, device=DEV)
        if c["late"]:
            s["finished"] = torch.rand(B, K, generator=g, device=DEV) < 0.2
            s["logits"][:, :, V // 2: V // 2 + 40] = float("-inf")  # tokens that the program bans
        else:  # the first step: all beams are alike, and only the first may go on
            s["scores"][:, 1:] = float("-inf")
        s["end"] = V - 1
        s["states"] = [_normal(g, B * K, c["H"], c["Dk"], c["Dv"])]
    return s


# ----------------------------------------------------------------------------------------- plain forms
def _rotate(x, angle, pairs, back=False):
    """x turned by `angle` (..., R/2) in its first R columns; back: by the opposite angle."""
    n = angle.shape[-1]
    cos, sin = torch.cos(angle), torch.sin(angle) * (-1.0 if back else 1.0)
    if pairs == "halves":
        a, b = x[..., :n], x[..., n:2 * n]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * n:]], -1)
    a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., 2 * n:]], -1)


def _plain_rotate(s):
    c = s["case"]
    # whole turns fall off the 64-bit product: what is left is the angle's place in one turn
    angle = ((s["positions"][..., None] * s["turns"]).float() * (2 * math.pi / 2.0 ** 64))[:, :, None]

    def forward(x, w):
        xf = x.float()
        y = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS) * w
        return _rotate(y, angle, c["pairs"]).to(x.dtype)

    def backward(x, w, g):
        xf = x.float()
        r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
        gu = _rotate(g.float(), angle, c["pairs"], back=True)
        xh, gw = xf * r, gu * w
        return (r * (gw - xh * (gw * xh).mean(-1, keepdim=True))).to(x.dtype), (gu * xh).sum((0, 1, 2))

    if c["dir"] == "fwd":
        return {"q": forward(s["q"], s["wq"]), "k": forward(s["k"], s["wk"])}
    gq, gwq = backward(s["q"], s["wq"], s["gq"])
    gk, gwk = backward(s["k"], s["wk"], s["gk"])
    return {"grad_q": gq, "grad_k": gk, "grad_wq": gwq, "grad_wk": gwk}


CHUNK = 64


def _chunks(x, H, lengths):
    """(B, L, h, D) as float32 (B, H, chunks, CHUNK, D): shared heads repeated, zeros past the length and the end."""
    B, L, h, D = x.shape
    x = x.float()
    if lengths is not None:
        x = x * (torch.arange(L, device=x.device) < lengths[:, None])[:, :, None, None]
    pad = -L % CHUNK
    if pad:
        x = torch.cat([x, x.new_zeros(B, pad, h, D)], 1)
    x = x.permute(0, 2, 1, 3).reshape(B, h, 1, -1, CHUNK, D).expand(B, h, H // h, (L + pad) // CHUNK, CHUNK, D)
    return x.reshape(B, H, -1, CHUNK, D)


def _flat(x, L, h, dtype):
    """Back to (B, L, h, D): heads that share are summed."""
    B, H, n, C, D = x.shape
    return x.reshape(B, h, H // h, n * C, D).sum(2).permute(0, 2, 1, 3)[:, :L].to(dtype)


def _powers(log_decay, e):
    """decay^e for whole e (elsewhere than e < 0, where it is 0): (H, *e.shape)."""
    return torch.where(e >= 0, torch.exp(log_decay.view(-1, *[1] * e.dim()) * e.clamp(min=0)), 0.0)


def _plain_attn(s):
    c = s["case"]
    q, k, v, ld, L, H = s["q"], s["k"], s["v"], s["log_decay"], c["L"], c["H"]
    B, scale = c["B"], c["Dk"] ** -0.5
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), L, device=DEV, dtype=torch.int32)
    Q, K, V = (_chunks(x, H, s["lengths"]) for x in (q, k, v))
    N = Q.shape[2]
    i = torch.arange(CHUNK, device=DEV)
    inside = _powers(ld, (i[:, None] - i[None, :]).float())[:, None]          # (H, 1, C, C)
    first = _powers(ld, (i + 1).float())[:, None, :, None]                    # what a start state weighs at i
    last = _powers(ld, (CHUNK - 1 - i).float())[:, None, :, None]             # what token i weighs in the end state
    at = torch.arange(N + 1, device=DEV)
    over = _powers(ld, CHUNK * (at[:N, None] - 1 - at[None, :N]).float())     # (H, N, N): end of chunk to start of chunk
    lead = _powers(ld, CHUNK * at[:N].float())[:, :, None, None]
    own_kv = (K * last).transpose(-1, -2) @ V                                 # (B, H, N, Dk, Dv)
    S = lead * s["state"][:, :, None] + (over @ own_kv.flatten(-2)).view_as(own_kv)
    # the state after `length` tokens: tokens past it are zeros, so only the decay since then is taken back
    rest = _powers(ld, (n[:, None] - 1 - torch.arange(N * CHUNK, device=DEV)).float())  # (H, B, tokens)
    w = rest.permute(1, 0, 2).reshape(B, H, N, CHUNK, 1)
    total = _powers(ld, n.float()).t()[..., None, None]                       # (B, H, 1, 1)
    end = total * s["state"] + ((K * w).transpose(-1, -2) @ V).sum(2)
    if c["dir"] == "fwd":
        o = ((Q @ K.transpose(-1, -2)) * inside) @ V + first * (Q @ S)
        return {"out": _flat(o * scale, L, H, v.dtype), "state": end}
    G = _chunks(s["g"], H, s["lengths"]) * scale
    own_qg = (Q * first).transpose(-1, -2) @ G                                # the adjoint of a chunk's start state
    # the adjoint of a chunk's end state: the later chunks', and the final state's from the sequence's own end
    X = (over.transpose(-1, -2) @ own_qg.flatten(-2)).view_as(own_qg)
    live = (torch.arange(N * CHUNK, device=DEV) < n[:, None]).view(B, 1, N, CHUNK, 1)
    gS = s["g_state"][:, :, None]
    A = (Q @ K.transpose(-1, -2)) * inside
    W = (G @ V.transpose(-1, -2)) * inside
    dq = W @ K + first * (G @ S.transpose(-1, -2))
    dk = W.transpose(-1, -2) @ Q + last * (V @ X.transpose(-1, -2)) + w * live * (V @ gS.transpose(-1, -2))
    dv = A.transpose(-1, -2) @ G + last * (K @ X) + w * live * (K @ gS)
    g0 = total * s["g_state"] + (lead * own_qg).sum(2)
    r = {"grad_q": _flat(dq, L, c["Hq"], q.dtype), "grad_k": _flat(dk, L, c["Hk"], k.dtype),
         "grad_v": _flat(dv, L, H, v.dtype), "grad_state": g0}
    if c["learn"]:
        # d/d ln(decay): every weight decay^e gives e times itself
        e = (i[:, None] - i[None, :]).clamp(min=0).float()
        gl = (A * (G @ V.transpose(-1, -2)) * e).sum((0, 2, 3, 4))
        far = CHUNK * (at[:N, None] - 1 - at[None, :N]).clamp(min=0).float()
        dS = (over * far @ own_kv.flatten(-2)).view_as(own_kv) + lead * (CHUNK * at[:N].float())[:, None, None] * s["state"][:, :, None]
        gl = gl + (own_qg * dS).sum((0, 2, 3, 4))
        gl = gl + ((Q * first * (i + 1).float()[:, None]).transpose(-1, -2) @ G * S).sum((0, 2, 3, 4))
        left = (CHUNK - 1 - i).float()[:, None]
        gl = gl + ((K * last * left).transpose(-1, -2) @ V * X).sum((0, 2, 3, 4))
        ago = (n[:, None] - 1 - torch.arange(N * CHUNK, device=DEV)).clamp(min=0).float().view(B, 1, N, CHUNK, 1)
        d_end = total * n.float().view(B, 1, 1, 1) * s["state"] + ((K * w * ago).transpose(-1, -2) @ V).sum(2)
        r["grad_log_decay"] = gl + (s["g_state"] * d_end).sum((0, 2, 3))
    return r


def _plain_step(s):
    c = s["case"]
    old = s["state"] if s["rows"] is None else s["state"][s["rows"]]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    new = torch.exp(s["log_decay"])[:, None, None] * old + k[..., None] * v[..., None, :]
    o = (q[..., None] * new).sum(-2) * c["Dk"] ** -0.5
    return {"out": o.to(s["v"].dtype), "state": new}


def _plain_beam(s):
    c = s["case"]
    B, K, V = c["B"], c["K"], c["V"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    cand = s["scores"][..., None] + (x - lse)
    token = torch.arange(V, device=DEV)
    # a finished beam goes on as it is: its one candidate is the end token at its own score
    stay = torch.where(token == s["end"], s["scores"][..., None], float("-inf"))
    cand = torch.where(s["finished"][..., None], stay, cand).nan_to_num(nan=float("-inf"), neginf=float("-inf"), posinf=float("inf"))
    best, at = torch.sort(cand.view(B, K * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    rows = at // V + K * torch.arange(B, device=DEV)[:, None]
    token = at % V
    done = s["finished"].view(-1)[rows] | (token == s["end"])
    return {"scores": best.contiguous(), "rows": rows, "tokens": token, "finished": done,
            "states": [t[rows.view(-1)] for t in s["states"]]}


def run(state):
    s = state
    c = s["case"]
    if not own:
        return {"rotate": _plain_rotate, "attn": _plain_attn, "step": _plain_step, "beam": _plain_beam}[c["op"]](s)
    from icml_b200 import ops
    if c["op"] == "rotate":
        kw = dict(positions=s["positions"], eps=EPS, pairs=c["pairs"])
        if c["dir"] == "fwd":
            q, k = ops.qk_norm_rotate_fwd(s["q"], s["k"], s["wq"], s["wk"], s["turns"], **kw)
            return {"q": q, "k": k}
        return ops.qk_norm_rotate_bwd(s["q"], s["k"], s["gq"], s["gk"], s["wq"], s["wk"], s["turns"], **kw)
    if c["op"] == "attn":
        if c["dir"] == "fwd":
            o, end = ops.decay_attn_fwd(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], lengths=s["lengths"])
            return {"out": o, "state": end}
        return ops.decay_attn_bwd(s["q"], s["k"], s["v"], s["log_decay"], s["g"], state=s["state"],
                                  g_state=s["g_state"], lengths=s["lengths"], need_g_log_decay=c["learn"])
    if c["op"] == "step":
        o, new = ops.decay_attn_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], rows=s["rows"],
                                     out_state=s["next_state"])
        return {"out": o, "state": new}
    scores, rows, tokens, finished = ops.beam_select(s["logits"], s["scores"], s["finished"], end_id=s["end"])
    return {"scores": scores, "rows": rows, "tokens": tokens, "finished": finished,
            "states": ops.beam_reorder(s["states"], rows)}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "rotate":
        n = c["B"] * c["L"] * (c["Hq"] + c["Hk"]) * c["D"]
        passes = 2 if c["dir"] == "fwd" else 3
        return {"bytes": passes * e * n + 8 * c["B"] * c["L"], "flops": (8 if c["dir"] == "fwd" else 18) * n}
    if c["op"] == "attn":
        t = c["B"] * c["L"]
        if c["ragged"]:  # lengths are spread evenly from nothing to all
            t = t * (c["B"] + 1) // (2 * c["B"])
        qk, vo = (c["Hq"] + c["Hk"]) * c["Dk"], 2 * c["H"] * c["Dv"]
        states = c["B"] * c["H"] * c["Dk"] * c["Dv"] * 4
        one = 2 * t * c["H"] * c["Dk"] * c["Dv"]
        if c["dir"] == "fwd":
            return {"bytes": e * t * (qk + vo) + 2 * states, "flops": 2 * one}
        return {"bytes": e * t * (2 * qk + vo + c["H"] * c["Dv"]) + 3 * states, "flops": 5 * one}
    if c["op"] == "step":
        r = c["B"] * c["H"]
        return {"bytes": r * (8 * c["Dk"] * c["Dv"] + e * 2 * (c["Dk"] + c["Dv"])), "flops": 5 * r * c["Dk"] * c["Dv"]}
    n, st = c["B"] * c["K"] * c["V"], c["B"] * c["K"] * c["H"] * c["Dk"] * c["Dv"]
    return {"bytes": e * n + 8 * st + 30 * c["B"] * c["K"], "flops": 4 * n}


# ----------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions, term by term, in float64."""
    s, c = prepare(case, seed), case

    def exact_rotate():
        D, R = c["D"], c["R"]
        n = R // 2
        f = c["base"] ** (-2.0 * torch.arange(n, device=DEV, dtype=torch.float64) / R)
        t = s["positions"].double()[..., None] * f
        turn = torch.polar(torch.ones_like(t), t)[:, :, None]
        first = torch.arange(n, device=DEV) * (1 if c["pairs"] == "halves" else 2)
        second = first + (n if c["pairs"] == "halves" else 1)

        def apply(x, turn):
            y = x.clone()
            z = torch.complex(x[..., first], x[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            return y

        out = {}
        for name, x, w in (("q", s["q"], s["wq"]), ("k", s["k"], s["wk"])):
            x, w = x.double(), w.double()
            norm = (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt()
            if c["dir"] == "fwd":
                out[name] = apply(x / norm * w, turn)
                continue
            gu = apply(s["g" + name].double(), turn.conj())
            out["grad_w" + name] = (gu * x / norm).sum((0, 1, 2))
            inner = (gu * w * x).sum(-1, keepdim=True)
            out["grad_" + name] = gu * w / norm - x * inner / (D * norm.pow(3))
        return out

    def exact_attn():
        """From the sums over all pairs of tokens, a block of rows of one head at a time."""
        B, L, H = c["B"], c["L"], c["H"]
        lens = [L] * B if s["lengths"] is None else s["lengths"].tolist()
        if sum(n * n for n in lens) * H * (c["Dk"] + c["Dv"]) * (1 if c["dir"] == "fwd" else 4) > 4e13:
            return None
        scale = c["Dk"] ** -0.5
        z = lambda *n: torch.zeros(*n, dtype=torch.float64, device=DEV)  # noqa: E731
        fwd = c["dir"] == "fwd"
        out = {"out": z(B, L, H, c["Dv"]), "state": z(B, H, c["Dk"], c["Dv"])} if fwd else {
            "grad_q": z(B, L, c["Hq"], c["Dk"]), "grad_k": z(B, L, c["Hk"], c["Dk"]), "grad_v": z(B, L, H, c["Dv"]),
            "grad_state": z(B, H, c["Dk"], c["Dv"])}
        g_ld = z(H)
        for b in range(B):
            n = lens[b]
            for h in range(H):
                hq, hk = h * c["Hq"] // H, h * c["Hk"] // H
                q, k, v = s["q"][b, :n, hq].double(), s["k"][b, :n, hk].double(), s["v"][b, :n, h].double()
                S0, ld = s["state"][b, h].double(), s["log_decay"][h].double()
                t = torch.arange(n, device=DEV, dtype=torch.float64)
                since, until = torch.exp(ld * (t + 1))[:, None], torch.exp(ld * (n - 1 - t))[:, None]
                if fwd:
                    out["state"][b, h] = torch.exp(ld * n) * S0 + (k * until).T @ v
                else:
                    gS = s["g_state"][b, h].double()
                    g = s["g"][b, :n, h].double() * scale
                    out["grad_state"][b, h] = torch.exp(ld * n) * gS + (q * since).T @ g
                    out["grad_k"][b, :n, hk] += until * (v @ gS.T)
                    out["grad_v"][b, :n, h] += until * (k @ gS)
                    g_ld[h] += n * torch.exp(ld * n) * (gS * S0).sum()
                    g_ld[h] += (((k * until * (n - 1 - t)[:, None]).T @ v) * gS).sum()
                    g_ld[h] += (((q * since * (t + 1)[:, None]).T @ g) * S0).sum()
                step = 2048
                for a in range(0, n, step):
                    m = min(a + step, n)
                    e = t[a:m, None] - t[None, :m]
                    w = torch.where(e >= 0, torch.exp(ld * e.clamp(min=0)), 0.0)
                    qk = q[a:m] @ k[:m].T * w
                    if fwd:
                        out["out"][b, a:m, h] = scale * (qk @ v[:m] + since[a:m] * (q[a:m] @ S0))
                        continue
                    gv = g[a:m] @ v[:m].T * w
                    out["grad_v"][b, :m, h] += qk.T @ g[a:m]
                    out["grad_k"][b, :m, hk] += gv.T @ q[a:m]
                    out["grad_q"][b, a:m, hq] += gv @ k[:m] + since[a:m] * (g[a:m] @ S0.T)
                    g_ld[h] += (q[a:m] @ k[:m].T * gv * e.clamp(min=0)).sum()
        if c["learn"]:
            out["grad_log_decay"] = g_ld
        return out

    if c["op"] == "rotate":
        return exact_rotate()
    if c["op"] == "attn":
        return exact_attn()
    if c["op"] == "step":
        old = s["state"].double()
        if s["rows"] is not None:
            old = old.index_select(0, s["rows"])
        new = old * s["log_decay"].double().exp().view(1, -1, 1, 1) + torch.einsum("bhk,bhv->bhkv", s["k"].double(), s["v"].double())
        return {"out": torch.einsum("bhk,bhkv->bhv", s["q"].double(), new) / math.sqrt(c["Dk"]), "state": new}
    logp = torch.log_softmax(s["logits"].double(), -1)
    cand = s["scores"].double()[..., None] + logp
    for b, k in s["finished"].nonzero().tolist():
        cand[b, k] = float("-inf")
        cand[b, k, s["end"]] = s["scores"][b, k]
    return {"scores": cand.flatten(1).topk(c["K"], -1).values, "rows": None, "tokens": None, "finished": None, "states": None}
