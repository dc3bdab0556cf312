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
    from matryoshka_transcoder_amd.activation_store import TensorPairSource
    cfg = dict(act_size=8, batch_size=4, num_batches_in_buffer=1, device="cpu", dtype=torch.float32, source_norm=_Doubling(),
               source_hook_point="blocks.0.ln2.hook_normalized")
    store = TranscoderActivationsStore(None, cfg, source=TensorPairSource([(torch.ones(4, 8), torch.ones(4, 8))]))
    assert torch.equal(store.next_batch()[0], torch.full((4, 8), 2.0))       # rows that are handed over are residual rows, whatever the name


# ---------------------------------------------------------------- a saved run keeps its norm, an adapter takes it along
def _run_cfg(**kw):
    return dict(dict(seed=3, prefix_sizes=[16, 64], dict_size=64, act_size=8, top_k=4, top_k_aux=8, aux_penalty=1 / 32, n_batches_to_dead=20,
                     l1_coeff=0.0, dtype=torch.float32, device="cpu", model_name="gpt2-small", layer=0, source_site="resid_mid",
                     source_hook_point="blocks.0.hook_resid_mid", seq_len=64), **kw)


def _norm():
    from matryoshka_transcoder_amd.block_norm import BlockNorm
    n = BlockNorm(8, kind="layer", eps=3e-4, weight_offset=1.0)
    with torch.no_grad():
        n.weight.copy_(torch.arange(8.0))
        n.bias.copy_(-torch.arange(8.0))
    return n


def _saved_run(tmp_path, norm):
    from matryoshka_transcoder_amd.results import CleanResultsManager
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    cfg = _run_cfg(source_norm=norm)
    results = CleanResultsManager(str(tmp_path))
    run = results.create_experiment_dir("m", 0, 1)
    results.save_checkpoint(run, MatryoshkaTranscoder(cfg), cfg, 1, is_final=True)
    return run / "checkpoints" / "final.pt"


def _same_norm(a, b):
    assert (a.width, a.kind, a.eps, a.weight_offset) == (b.width, b.kind, b.eps, b.weight_offset)
    assert list(a.state_dict()) == list(b.state_dict())
    for k, v in a.state_dict().items():
        assert torch.equal(v, b.state_dict()[k])


def test_a_saved_run_keeps_its_norm(tmp_path):
    import json
    from matryoshka_transcoder_amd.sae_bench import build_matryoshka_adapter
    norm = _norm()
    path = _saved_run(tmp_path, norm)
    saved = json.loads((path.parents[1] / "config.json").read_text())["source_norm"]
    for cfg in (_run_cfg(source_norm=saved), _run_cfg(), _run_cfg(source_norm=norm)):       # as read back, rebuilt by hand, live
        adapter = build_matryoshka_adapter(cfg, state_dict_path=path)
        _same_norm(adapter.source_norm, norm)
        assert list(adapter.state_dict()) == ["b_enc", "W_enc", "W_dec", "b_dec", "threshold"]      # the layout stays the reference's
        assert len(list(adapter.parameters())) == 4
    assert adapter.source_norm is not norm and not any(p.requires_grad for p in adapter.source_norm.parameters())
    assert adapter.to(dtype=torch.bfloat16).source_norm.weight.dtype == torch.bfloat16
    assert build_matryoshka_adapter(_run_cfg(source_norm=None), state_dict_path=path).source_norm is None      # said so: none


def test_a_later_run_without_a_norm_leaves_none(tmp_path):
    from matryoshka_transcoder_amd.sae_bench import build_matryoshka_adapter
    _saved_run(tmp_path, _norm())
    path = _saved_run(tmp_path, None)
    assert build_matryoshka_adapter(_run_cfg(), state_dict_path=path).source_norm is None


def test_the_adapter_norms_what_the_hook_yields(monkeypatch):
    from matryoshka_transcoder_amd import sae_bench
    from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder
    seen = []
    for name in ("encode", "reconstruct", "compute_activations"):
        monkeypatch.setattr(MatryoshkaTranscoder, name, lambda self, x: seen.append(x))
    monkeypatch.setattr(MatryoshkaTranscoder, "_run_forward", lambda self, x, *rest: seen.append(x))
    x = torch.ones(2, 8)
    for norm, want in ((_Doubling(), 2.0), (None, 1.0)):
        adapter = sae_bench.build_matryoshka_adapter(_run_cfg(source_norm=norm))
        for call in (adapter.encode, adapter.reconstruct, adapter.compute_activations):
            call(x)
        adapter._run_forward(x, x, None, None, None, None, False)
        assert len(seen) == 4 and all(torch.equal(s, want * x) for s in seen)
        seen.clear()


def test_an_adapter_without_its_norm_is_refused(tmp_path):
    from matryoshka_transcoder_amd.block_norm import BlockNorm
    from matryoshka_transcoder_amd.sae_bench import build_matryoshka_adapter
    with pytest.raises(_lib.MtcError, match="source_norm"):                  # a description and no file that holds the norm
        build_matryoshka_adapter(_run_cfg(source_norm="BlockNorm(8, ...)"))
    path = _saved_run(tmp_path, _Doubling())
    with pytest.raises(_lib.MtcError, match="source_norm"):                  # a module that the file cannot bring back
        build_matryoshka_adapter(_run_cfg(), state_dict_path=path)
    assert build_matryoshka_adapter(_run_cfg(source_norm=_Doubling()), state_dict_path=path).source_norm is not None
    with pytest.raises(_lib.MtcError, match="hook_normalized"):
        build_matryoshka_adapter(_run_cfg(source_norm=_norm()), hook_point="blocks.0.ln2.hook_normalized")
    with pytest.raises(_lib.MtcError, match="width"):
        build_matryoshka_adapter(_run_cfg(source_norm=BlockNorm(4)))
