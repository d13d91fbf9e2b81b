"""The decay-attention layer's host side, without a GPU."""
import pytest
import torch

from icml_b200.lm import PGFLanguageModel
from icml_b200.pgf_decay import DecayMixer, PGFDecayBlock


def test_mixer_layout():
    m = DecayMixer(96, 24, 6, 2)
    assert m.widths == (144, 48, 32) and m.d_value == 16
    assert [p.shape for p in (m.qkv_proj.weight, m.q_norm, m.decay, m.out_proj.weight)] == [(224, 96), (24,), (6,), (96, 96)]
    q, k, v = m.heads(torch.arange(2 * 3 * 224).view(2, 3, 224))
    assert q.shape == (2, 3, 6, 24) and k.shape == (2, 3, 2, 24) and v.shape == (2, 3, 2, 16)
    assert q[1, 2, 5, 23] == 5 * 224 + 143 and k[0, 0, 1, 0] == 168 and v[0, 1, 0, 0] == 224 + 192
    a = m.log_decay().exp()
    assert torch.allclose(a[[0, -1]], torch.tensor([1 - 2.0 ** -3, 1 - 2.0 ** -9])) and bool((a[1:] > a[:-1]).all())


def test_odd_widths_and_rotation():
    assert DecayMixer(64, 33, 1).turns.numel() == 16
    assert DecayMixer(64, 32, 1, rotary_dim=0).turns.numel() == 0


@pytest.mark.parametrize("kw", [dict(n_heads=5), dict(n_heads=4, n_kv_heads=3), dict(rotary_dim=66), dict(rotary_dim=7),
                                dict(rotary_dim=-2)])
def test_mixer_refusals(kw):
    with pytest.raises(ValueError):
        DecayMixer(64, 64, **kw)


def test_model_variant():
    m = PGFLanguageModel(31, 64, 16, 128, 2, 64, "cpu", variant="decay", n_heads=4, n_kv_heads=2)
    assert all(isinstance(b, PGFDecayBlock) and b.mixer.n_kv_heads == 2 for b in m.backbone.layers)
    with pytest.raises(ValueError):
        PGFLanguageModel(31, 64, 16, 128, 1, 64, "cpu", variant="none")
