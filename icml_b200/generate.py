"""Beam search with a decay-attention language model (lm.PGFLanguageModel, variant "decay").

A prompt runs once through the layers' chunked form, which leaves one state per layer and row; every further
token is one single-token call per layer.  A selected beam goes on from its parent's state by reading it (the
step's `rows`), so states are never copied to reorder them; only the short token histories are.

    python -m icml_b200.generate         trains a small model on synthetic sequences and continues some
"""
from __future__ import annotations

import argparse
from typing import Optional

import torch

from . import ops
from .lm import PGFLanguageModel


def _logits(model: PGFLanguageModel, x: torch.Tensor) -> torch.Tensor:
    if model.final_norm is not None:
        x = model.final_norm.pgf_forward(x)
    return ops.lm_head_fwd(x, model.lm_head_weight)


@torch.no_grad()
def prefill(model: PGFLanguageModel, prompt: torch.Tensor, lengths: Optional[torch.Tensor] = None):
    """(logits (B, V) behind each row's last token, [state of each layer]) of a prompt (B, L) whose row b has
    lengths[b] tokens (default all), 1 or more."""
    B, L = prompt.shape
    least, most = (L, L) if lengths is None or B == 0 else torch.stack(lengths.aminmax()).tolist()
    if L < 1 or least < 1 or most > L:
        raise ValueError(f"prefill: lengths from {least} to {most}, every row has 1 to {L} tokens")
    x = ops.embedding_fwd(prompt, model.emb_weight, dtype=model.act_dtype)
    states = []
    for layer in model.backbone.layers:
        x, s = layer.prefill(x, lengths=lengths)
        states.append(s)
    last = x[:, -1] if lengths is None else x[torch.arange(B, device=x.device), lengths.to(x.device).long() - 1]
    return _logits(model, last), states


@torch.no_grad()
def beam_search(model: PGFLanguageModel, prompt: torch.Tensor, steps: int, beams: int = 4,
                lengths: Optional[torch.Tensor] = None, end_id: Optional[int] = None):
    """(tokens (B, beams, steps), scores (B, beams), finished (B, beams)): the best continuations of each row,
    best first.  A score is the sum of its tokens' log probabilities; a beam that has chosen end_id is finished
    and repeats it at no cost."""
    if model.variant != "decay":
        raise ValueError(f"beam_search: variant {model.variant!r} has no single-token form (decay)")
    if steps < 1 or not 1 <= beams <= min(32, model.vocab_size):
        raise ValueError(f"beam_search: {steps} steps of {beams} beams (at most 32) over {model.vocab_size} tokens")
    B, L = prompt.shape
    dev = prompt.device
    logits, states = prefill(model, prompt, lengths)
    # the first selection: all beams of a row are its prompt, of which one counts
    scores = torch.full((B, beams), float("-inf"), device=dev)
    scores[:, 0] = 0
    logits = logits.unsqueeze(1).expand(B, beams, -1)
    done = None
    at = torch.full((B,), L, device=dev) if lengths is None else lengths.to(dev).long()
    at = at.repeat_interleave(beams)
    tokens = torch.zeros(B * beams, steps, dtype=torch.int64, device=dev)
    other = torch.empty_like(tokens)
    spare = [None] * len(states)
    for t in range(steps):
        scores, rows, chosen, done = ops.beam_select(logits, scores, done if end_id is not None else None,
                                                     end_id=end_id)
        flat = rows.view(-1)
        ops.beam_reorder([tokens], flat, out=[other])
        tokens, other = other, tokens
        tokens[:, t] = chosen.view(-1)
        if t == steps - 1:
            break
        if t == 0:
            flat = flat // beams               # the prompt's states have one row per sequence
        x = ops.embedding_fwd(chosen.view(-1), model.emb_weight, dtype=model.act_dtype)
        for i, layer in enumerate(model.backbone.layers):
            # two buffers per layer take turns: parents are read from one, children written to the other
            x, new = layer.step(x, states[i], at, rows=flat, out_state=spare[i])
            spare[i], states[i] = (states[i] if t else None), new
        at = at + 1
        logits = _logits(model, x).view(B, beams, -1)
    return tokens.view(B, beams, steps), scores, done


def synthetic_batch(B: int, L: int, vocab: int, device, seed: int) -> torch.Tensor:
    """(B, L) ids that count upwards by a step of 1 to 3 for each row, modulo the vocabulary."""
    g = torch.Generator().manual_seed(seed)
    first, by = torch.randint(vocab, (B, 1), generator=g), torch.randint(1, 4, (B, 1), generator=g)
    return ((first + by * torch.arange(L)) % vocab).to(device)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--train-steps", type=int, default=300)
    ap.add_argument("--vocab", type=int, default=64)
    ap.add_argument("--d-model", type=int, default=128)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--steps", type=int, default=12)
    ap.add_argument("--dtype", choices=("float32", "bfloat16"), default="bfloat16")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = PGFLanguageModel(a.vocab, a.d_model, 64, 2 * a.d_model, a.layers, 128, "cuda",
                             act_dtype=getattr(torch, a.dtype), lr=2e-3, variant="decay", final_norm=True)
    first = last = None
    for s in range(a.train_steps):
        ids = synthetic_batch(16, 97, a.vocab, "cuda", s)
        loss = model.step(ids[:, :-1].contiguous(), ids[:, 1:].contiguous())
        first = loss.clone() if first is None else first
        last = loss
    ids = synthetic_batch(4, 24 + a.steps, a.vocab, "cuda", 10 ** 6)
    lengths = torch.tensor([24, 17, 9, 24], device="cuda")
    tokens, scores, _ = beam_search(model, ids[:, :24], a.steps, a.beams, lengths)
    want = torch.stack([ids[b, n:n + a.steps] for b, n in enumerate(lengths.tolist())])
    right = (tokens[:, 0] == want).float().mean().item()
    if last is not None:
        print(f"loss {first.item():.3f} -> {last.item():.3f} in {a.train_steps} steps")
    for b, n in enumerate(lengths.tolist()):
        print(f"prompt ...{ids[b, n - 4:n].tolist()} -> {tokens[b, 0].tolist()} (log probability {scores[b, 0].item():.2f})")
    print(f"{100 * right:.0f}% of the best beams' tokens continue their sequence")
    return right


__all__ = ["beam_search", "prefill"]

if __name__ == "__main__":
    main()
