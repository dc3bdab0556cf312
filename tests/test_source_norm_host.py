"""cfg["source_norm"]: where the store may take the source activations from (no GPU needed: the norm is a stand-in)."""
import pytest
import torch

from matryoshka_transcoder_amd import _lib
from matryoshka_transcoder_amd.activation_store import TranscoderActivationsStore


class _Doubling(torch.nn.Module):
    """Stands in for a norm on the CPU: what went through it is seen at once."""
    def forward(self, x):
        return 2.0 * x


class _Model:
    """Exposes the hooks it is given; the block's norm has the scale 3."""
    def __init__(self, *hooks):
        self.hooks = hooks
        self.asked = None
        ln2 = type("Norm", (), {"w": torch.full((8,), 3.0)})()
        self.blocks = [type("Block", (), {"ln2": ln2})()]

    def run_with_cache(self, tokens, names_filter, stop_at_layer):
        self.asked = list(names_filter)
        return None, {h: torch.ones(*tokens.shape, 8) for h in self.hooks if h in names_filter}


def _store(model, norm, source="blocks.0.hook_mlp_in"):
    cfg = dict(act_size=8, batch_size=4, device="cpu", dtype=torch.float32, seq_len=5, layer=0, source_hook_point=source,
               target_hook_point="blocks.0.hook_mlp_out")
    if norm is not None:
        cfg["source_norm"] = norm
    return TranscoderActivationsStore(model, cfg)


TOKENS = torch.zeros(2, 5, dtype=torch.long)


def test_the_residual_in_front_of_the_norm_is_normed_once():
    model = _Model("blocks.0.hook_mlp_in", "blocks.0.ln2.hook_normalized", "blocks.0.hook_mlp_out")
    src, tgt = _store(model, _Doubling()).get_paired_activations(TOKENS)
    assert torch.equal(src, torch.full((2, 5, 8), 2.0)) and torch.equal(tgt, torch.ones(2, 5, 8))
    model = _Model("blocks.0.hook_resid_mid", "blocks.0.hook_mlp_out")
    src, _ = _store(model, _Doubling(), "blocks.0.hook_resid_mid").get_paired_activations(TOKENS)
    assert torch.equal(src, torch.full((2, 5, 8), 2.0))


def test_an_already_normed_fallback_is_refused():
    """A model without hook_mlp_in: the store falls back to what the block's norm left, which must not be normed again."""
    hooks = ("blocks.0.ln2.hook_normalized", "blocks.0.hook_mlp_out")
    src, _ = _store(_Model(*hooks), None).get_paired_activations(TOKENS)
    assert torch.equal(src, torch.full((2, 5, 8), 3.0))                      # without a source norm: the fallback, scaled
    with pytest.raises(_lib.MtcError, match="residual"):
        _store(_Model(*hooks), _Doubling()).get_paired_activations(TOKENS)


def test_a_source_point_behind_the_norm_is_refused():
    with pytest.raises(_lib.MtcError, match="hook_normalized"):
        _store(_Model(), _Doubling(), "blocks.0.ln2.hook_normalized")
    _store(_Model(), None, "blocks.0.ln2.hook_normalized")                   # without a source norm it is a point like any other
