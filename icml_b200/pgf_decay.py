"""Decay attention as a layer: its autograd functions, a mixer and a PGF block around it.

The reference's mixers (pgf_mamba.py, train_singlemamba_optimized.py) carry a diagonal state; this one
carries a matrix per head, S_t = a S_{t-1} + k_t v_t^T, read by o_t = scale q_t S_t, with queries and keys
normed for each head and rotated by position.  `PGFDecayBlock` keeps the reference block's structure and PGF
API (pgf_mamba_block.py:16-249: pgf_forward, pgf_backward returning {"grads", "grad_input"}) around it:
a layer keeps its input and its backward runs the layer again.  `prefill` and `step` are the serving forms.
"""
from __future__ import annotations

import math
from typing import Any, Dict, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import ops
from .pgf_ffn import FFNFunction
from .pgf_rmsnorm import RMSNorm


class _RotateFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, turns, positions, kw):
        ctx.save_for_backward(q, k, wq, wk, turns, positions)
        ctx.kw = kw
        return ops.qk_norm_rotate_fwd(q, k, wq, wk, turns, positions=positions, **kw)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, turns, positions = ctx.saved_tensors
        r = ops.qk_norm_rotate_bwd(q, k, gq, gk, wq, wk, turns, positions=positions, **ctx.kw)
        return r["grad_q"], r["grad_k"], r.get("grad_wq"), r.get("grad_wk"), None, None, None


def qk_norm_rotate(q, k, wq=None, wk=None, turns=None, *, positions=None, **kw):
    """ops.qk_norm_rotate_fwd with its gradient (of q, k, wq and wk)."""
    return _RotateFn.apply(q, k, wq, wk, turns, positions, kw)


class _DecayFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale):
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return ops.decay_attn_fwd(q, k, v, log_decay, scale=scale, state=state, lengths=lengths)

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_state):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        if g is None:
            g = v.new_zeros((*v.shape[:2], log_decay.numel(), v.shape[3]))
        r = ops.decay_attn_bwd(q, k, v, log_decay, g, scale=ctx.scale, state=state, g_state=g_state, lengths=lengths,
                               need_g_log_decay=ctx.needs_input_grad[3])
        return (r["grad_q"], r["grad_k"], r["grad_v"], r.get("grad_log_decay"),
                r["grad_state"] if ctx.needs_input_grad[4] else None, None, None)


def decay_attention(q, k, v, log_decay, *, scale: Optional[float] = None, state=None, lengths=None):
    """ops.decay_attn_fwd with its gradient (of q, k, v, log_decay and state)."""
    return _DecayFn.apply(q, k, v, log_decay, state, lengths, scale)


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W):
        ctx.save_for_backward(x, W)
        return _linear(x, W)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, W = ctx.saved_tensors
        gW, gx = _linear_bwd(x, g, W)
        return gx, gW


def _linear(x, W, addend=None):
    """x W^T (+ addend), in x's type."""
    y = ops.gemm(x.reshape(-1, x.shape[-1]), W.to(x.dtype), out_dtype=x.dtype,
                 addend=None if addend is None else addend.reshape(-1, W.shape[0]))
    return y.view(*x.shape[:-1], W.shape[0])


def _linear_bwd(x, g, W):
    x2, g2 = x.reshape(-1, x.shape[-1]), g.reshape(-1, g.shape[-1])
    gW = ops.gemm(g2, x2, a_trans=True, b_trans=True)
    return gW, ops.gemm(g2, W.to(x.dtype), b_trans=True, out_dtype=x.dtype).view(x.shape)


class DecayMixer(nn.Module):
    """Projection to n_heads queries and n_kv_heads keys (d_state wide) and values (d_model / n_heads wide),
    norm and rotation, decay attention, a norm of the heads' outputs and the projection back."""

    def __init__(self, d_model: int, d_state: int = 64, n_heads: Optional[int] = None, n_kv_heads: Optional[int] = None,
                 rotary_dim: Optional[int] = None, rotary_base: float = 10000.0, eps: float = 1e-6):
        super().__init__()
        H = n_heads or max(1, d_model // 64)
        Hk = n_kv_heads or H
        if d_model % H or H % Hk:
            raise ValueError(f"DecayMixer: {H} heads must divide d_model {d_model}, and {Hk} must divide them")
        R = d_state // 2 * 2 if rotary_dim is None else rotary_dim
        if R < 0 or R % 2 or R > d_state:
            raise ValueError(f"DecayMixer: rotary_dim {R} must be even and at most d_state {d_state}")
        self.d_model, self.d_state, self.n_heads, self.n_kv_heads, self.eps = d_model, d_state, H, Hk, eps
        self.d_value = d_model // H
        self.widths = (H * d_state, Hk * d_state, Hk * self.d_value)
        self.qkv_proj = nn.Linear(d_model, sum(self.widths), bias=False)
        self.q_norm = nn.Parameter(torch.ones(d_state))
        self.k_norm = nn.Parameter(torch.ones(d_state))
        # a head forgets over 8 tokens (the first) to 512 (the last): a = 1 - 1/8 .. 1 - 1/512
        gap = 2.0 ** -torch.linspace(3, 9, H)
        self.decay = nn.Parameter(torch.log((1 - gap) / gap))  # a = sigmoid(decay)
        self.out_norm = RMSNorm(d_model, eps)
        self.out_proj = nn.Linear(d_model, d_model, bias=False)
        self.register_buffer("turns", ops.rotary_turns(R, rotary_base, "cpu"), persistent=False)

    def log_decay(self) -> torch.Tensor:
        return F.logsigmoid(self.decay)

    def heads(self, qkv: torch.Tensor):
        """q, k, v as (..., heads, width) views of the projection's rows."""
        q, k, v = qkv.split(self.widths, -1)
        return (q.unflatten(-1, (self.n_heads, self.d_state)), k.unflatten(-1, (self.n_kv_heads, self.d_state)),
                v.unflatten(-1, (self.n_kv_heads, self.d_value)))

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        q, k, v = self.heads(_LinearFn.apply(x, self.qkv_proj.weight))
        q, k = qk_norm_rotate(q, k, self.q_norm, self.k_norm, self.turns, eps=self.eps)
        o, _ = decay_attention(q, k, v, self.log_decay(), lengths=lengths)
        return _LinearFn.apply(self.out_norm(o.flatten(-2)), self.out_proj.weight)

    @torch.no_grad()
    def attend(self, x, state=None, lengths=None, start: int = 0, want_state: bool = True):
        """(heads' outputs (B, L, d_model), state behind them) of x (B, L, d_model) that begins at position
        `start`; `state` came before it."""
        q, k, v = self.heads(_linear(x, self.qkv_proj.weight))
        q, k = ops.qk_norm_rotate_fwd(q, k, self.q_norm, self.k_norm, self.turns, start=start, eps=self.eps)
        o, end = ops.decay_attn_fwd(q, k, v, self.log_decay(), state=state, lengths=lengths, want_state=want_state)
        return o.flatten(-2), end

    @torch.no_grad()
    def attend_step(self, x, state, positions, rows=None, out_state=None):
        """One token of every row: x (B, d_model) at positions (B); row b goes on from state row rows[b]."""
        q, k, v = self.heads(_linear(x, self.qkv_proj.weight))
        q, k = ops.qk_norm_rotate_fwd(q.unsqueeze(1), k.unsqueeze(1), self.q_norm, self.k_norm, self.turns,
                                      positions=positions.view(-1, 1), eps=self.eps)
        o, state = ops.decay_attn_step(q.squeeze(1), k.squeeze(1), v, self.log_decay(), state, rows=rows,
                                       out_state=out_state)
        return o.flatten(-2), state

    @torch.no_grad()
    def project(self, o, residual=None):
        return _linear(ops.rmsnorm_fwd(o, self.out_norm.weight, self.out_norm.eps), self.out_proj.weight, residual)

    @torch.no_grad()
    def backward(self, x, o, g):
        """({parameter: gradient}, gradient of x) from the mixer's input, its heads' outputs and g."""
        on = ops.rmsnorm_fwd(o, self.out_norm.weight, self.out_norm.eps)
        g_out_w, g = _linear_bwd(on, g, self.out_proj.weight)
        g_on_w, g = ops.rmsnorm_bwd(o, g, self.out_norm.weight, self.out_norm.eps)
        q, k, v = self.heads(_linear(x, self.qkv_proj.weight))
        qr, kr = ops.qk_norm_rotate_fwd(q, k, self.q_norm, self.k_norm, self.turns, eps=self.eps)
        a = ops.decay_attn_bwd(qr, kr, v, self.log_decay(), g.unflatten(-1, (self.n_heads, self.d_value)),
                               need_g_log_decay=True)
        r = ops.qk_norm_rotate_bwd(q, k, a["grad_q"], a["grad_k"], self.q_norm, self.k_norm, self.turns, eps=self.eps)
        g = torch.cat([r["grad_q"].flatten(-2), r["grad_k"].flatten(-2), a["grad_v"].flatten(-2)], -1)
        g_w, gx = _linear_bwd(x, g, self.qkv_proj.weight)
        return {"qkv_proj.weight": g_w, "q_norm": r["grad_wq"], "k_norm": r["grad_wk"],
                "decay": a["grad_log_decay"] * torch.sigmoid(-self.decay), "out_norm.weight": g_on_w,
                "out_proj.weight": g_out_w}, gx


class PGFDecayBlock(nn.Module):
    """x -> RMSNorm -> decay attention -> +x -> RMSNorm -> FFN -> +x with the PGF API of PGFMambaBlock."""

    def __init__(self, d_model: int, d_state: int = 64, d_ff: Optional[int] = None, block_size: int = 128,
                 n_heads: Optional[int] = None, n_kv_heads: Optional[int] = None, ffn_activation: str = "gelu", **mixer):
        super().__init__()
        self.d_model, self.d_ff, self.block_size = d_model, d_ff or 4 * d_model, block_size
        self.ffn_activation = ffn_activation
        self.norm1 = RMSNorm(d_model)
        self.mixer = DecayMixer(d_model, d_state, n_heads, n_kv_heads, **mixer)
        self.norm2 = RMSNorm(d_model)
        self.W1 = nn.Parameter(torch.empty(self.d_ff, d_model))
        self.b1 = nn.Parameter(torch.zeros(self.d_ff))
        self.W2 = nn.Parameter(torch.empty(d_model, self.d_ff))
        self.b2 = nn.Parameter(torch.zeros(d_model))
        nn.init.xavier_uniform_(self.W1)
        nn.init.xavier_uniform_(self.W2)

    def forward(self, x):
        x1 = self.mixer(self.norm1(x)) + x
        D = x.shape[-1]
        f = FFNFunction.apply(self.norm2(x1).reshape(-1, D), self.W1, self.b1, self.W2, self.b2, self.ffn_activation)
        return f.view(x.shape) + x1

    def _finish(self, o, x):
        """(layer output, residual sum) from the heads' outputs and the layer's input."""
        D = self.d_model
        x1 = self.mixer.project(o, x)
        y = ops.ffn_fwd(self.norm2.pgf_forward(x1).reshape(-1, D), self.W1, self.b1, self.W2, self.b2,
                        self.ffn_activation, residual=x1.reshape(-1, D))
        return y.view(x.shape), x1

    @torch.no_grad()
    def pgf_forward(self, x: torch.Tensor, return_ssm_states: bool = False, keep_scan: bool = False):
        """With keep_scan (and return_ssm_states) also the heads' outputs and the residual sum: pgf_backward
        then runs neither the attention nor the projection behind it again."""
        o, _ = self.mixer.attend(self.norm1.pgf_forward(x), want_state=False)
        y, x1 = self._finish(o, x)
        return (y, {"o": o, "x1": x1} if keep_scan else None) if return_ssm_states else y

    @torch.no_grad()
    def pgf_backward(self, x: torch.Tensor, g_out: torch.Tensor, fp32_accum: bool = True,
                     ssm_states: Optional[Any] = None) -> Dict[str, Any]:
        D = self.d_model
        g_out = g_out.to(x.dtype)
        xn = self.norm1.pgf_forward(x)
        if ssm_states is not None:
            o, x1 = ssm_states["o"], ssm_states["x1"]
        else:
            o, _ = self.mixer.attend(xn, want_state=False)
            x1 = self.mixer.project(o, x)
        f = ops.ffn_bwd(self.norm2.pgf_forward(x1).reshape(-1, D), g_out.reshape(-1, D), self.W1, self.b1, self.W2,
                        self.ffn_activation)
        gw2, g1 = ops.rmsnorm_bwd(x1, f["grad_x"].view(x.shape), self.norm2.weight, self.norm2.eps, g_add=g_out)
        gm, gxn = self.mixer.backward(xn, o, g1)
        gw1, gx = ops.rmsnorm_bwd(x, gxn, self.norm1.weight, self.norm1.eps, g_add=g1)
        grads = {"W1": f["grad_W1"], "b1": f["grad_b1"], "W2": f["grad_W2"], "b2": f["grad_b2"], "norm1.weight": gw1,
                 "norm2.weight": gw2}
        grads.update({"mixer." + k: v for k, v in gm.items()})
        return {"grads": grads, "grad_input": gx}

    @torch.no_grad()
    def prefill(self, x, state=None, lengths=None, start: int = 0):
        """(layer output, state (B, H, d_state, d_value) float32 behind each row's `lengths` tokens)."""
        o, state = self.mixer.attend(self.norm1.pgf_forward(x), state, lengths, start)
        return self._finish(o, x)[0], state

    @torch.no_grad()
    def step(self, x, state, positions, rows=None, out_state=None):
        """prefill for one token of every row: x (B, d_model) at positions (B).  rows (B): the state row that
        row b goes on from; out_state: where the new state goes (`state` itself updates in place, without rows)."""
        o, state = self.mixer.attend_step(self.norm1.pgf_forward(x), state, positions, rows, out_state)
        return self._finish(o, x)[0], state


__all__ = ["DecayMixer", "PGFDecayBlock", "decay_attention", "qk_norm_rotate"]
