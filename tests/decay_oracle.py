"""Plain float64 statements of the decay-attention layer's operators (checker side only)."""
import math

import torch


def rotate(x, pos, R, base, pairs):
    """x (B, L, h, D) with the first R elements of each head turned by pos (B, L) times base^(-2i/R)."""
    if R == 0:
        return x
    i = torch.arange(R // 2, dtype=torch.float64, device=x.device)
    ang = (pos.double()[..., None] * base ** (-2 * i / R))[:, :, None]
    a = i.long() if pairs == "halves" else 2 * i.long()
    b = a + (R // 2 if pairs == "halves" else 1)
    y = x.clone()
    y[..., a] = x[..., a] * ang.cos() - x[..., b] * ang.sin()
    y[..., b] = x[..., a] * ang.sin() + x[..., b] * ang.cos()
    return y


def norm_rotate(x, w, pos, R, base, pairs, eps):
    u = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return rotate(u if w is None else u * w, pos, R, base, pairs)


def decay_attn(q, k, v, log_decay, scale, state, lengths):
    """(out, final state) from the sums over all pairs of tokens; differentiable."""
    B, L, Hq, Dk = q.shape
    H, dev = log_decay.numel(), q.device
    lens = torch.full((B,), L, device=dev) if lengths is None else lengths.clamp(0, L).long()
    live = (torch.arange(L, device=dev) < lens[:, None])[:, :, None, None]
    q, k, v = (torch.where(live, t, 0.0).repeat_interleave(H // t.shape[2], 2) for t in (q, k, v))
    t = torch.arange(L, device=dev, dtype=torch.float64)

    def power(e):  # decay^e, 0 where e < 0; a decay of zero still has power 0 = 1
        ok = e >= 0
        x = torch.where(e > 0, e, 1.0)
        p = torch.exp(log_decay.view(-1, *[1] * e.dim()) * x)
        return torch.where(ok, torch.where(e > 0, p, 1.0), 0.0)

    w = power(t[:, None] - t[None, :])                                   # (H, L, L)
    o = torch.einsum("bihd,bjhd,hij,bjhe->bihe", q, k, w, v) if L else torch.zeros_like(v)
    since = power(t + 1)                                                 # (H, L)
    left = power(lens[:, None].double() - 1 - t)                         # (H, B, L)
    total = power(lens.double())                                         # (H, B)
    end = torch.einsum("hbj,bjhd,bjhe->bhde", left, k, v)
    if state is not None:
        o = o + torch.einsum("hi,bihd,bhde->bihe", since, q, state)
        end = end + total.t()[..., None, None] * state
    return o * scale, end


def decay_step(q, k, v, log_decay, state, scale):
    H = log_decay.numel()
    q, k, v = (t.repeat_interleave(H // t.shape[1], 1) for t in (q, k, v))
    new = torch.exp(log_decay).view(1, -1, 1, 1) * state + k[..., None] * v[..., None, :]
    return scale * torch.einsum("bhd,bhde->bhe", q, new), new


def beam_candidates(logits, scores, finished, end_id):
    """(B, K V) float32 candidates as the operator defines them, from float32 log sums."""
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    lse = (m.double() + (x.double() - m.double()).exp().sum(-1, keepdim=True).log()).float()
    c = scores[..., None] + (x - lse)
    if finished is not None:
        stay = torch.full_like(c, -math.inf)
        stay[..., end_id] = scores
        c = torch.where(finished[..., None], stay, c)
    return torch.where(c.isnan(), -math.inf, c).flatten(1)
