"""A run with cfg["source_norm"], used through its adapter: raw residual rows in, the numbers of the run out."""
import pytest
import torch

from matryoshka_transcoder_amd.block_norm import BlockNorm
from matryoshka_transcoder_amd.results import CleanResultsManager
from matryoshka_transcoder_amd.sae_bench import build_matryoshka_adapter
from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_the_adapter_of_a_saved_run_sees_what_the_run_saw(dt, tmp_path):
    norm = BlockNorm(64, kind="layer", weight_offset=1.0, dtype=dt, device=DEV)
    with torch.no_grad():
        norm.weight.copy_(0.3 * torch.randn(64, generator=torch.Generator("cpu").manual_seed(1)))
        norm.bias.copy_(0.2 * torch.randn(64, generator=torch.Generator("cpu").manual_seed(2)))
    cfg = dict(seed=3, prefix_sizes=[64, 256], dict_size=256, act_size=64, top_k=8, top_k_aux=16, aux_penalty=1 / 32, n_batches_to_dead=20,
               l1_coeff=0.0, dtype=dt, device=DEV, model_name="gpt2-small", layer=0, source_site="resid_mid",
               source_hook_point="blocks.0.hook_resid_mid", seq_len=64, input_unit_norm=True, source_norm=norm)
    run = MatryoshkaTranscoder(cfg)
    with torch.no_grad():
        run.threshold.fill_(0.2)
        run.W_dec.div_(run.W_dec.norm(dim=-1, keepdim=True).clamp_min(1e-12))       # what the adapter does once more on loading
    results = CleanResultsManager(str(tmp_path))
    where = results.create_experiment_dir("m", 0, 1)
    results.save_checkpoint(where, run, cfg, 1, is_final=True)
    rebuilt = {k: v for k, v in cfg.items() if k != "source_norm"}
    adapter = build_matryoshka_adapter(rebuilt, state_dict_path=where / "checkpoints" / "final.pt").eval()
    run.eval()
    raw = (torch.randn(3, 11, 64, generator=torch.Generator("cpu").manual_seed(4)) * 3 + 1).to(dt).to(DEV)
    target = torch.randn(33, 64, generator=torch.Generator("cpu").manual_seed(5)).to(dt).to(DEV)
    with torch.no_grad():
        normed = norm(raw)
        assert torch.equal(adapter.encode(raw), run.encode(normed))
        assert not torch.equal(adapter.encode(raw), run.encode(raw))
        assert torch.equal(adapter.compute_activations(raw[0])[1], run.compute_activations(normed[0])[1])
        adapter.W_dec.copy_(run.W_dec)                                              # to the bit, for the reconstructions
        assert torch.equal(adapter.reconstruct(raw), run.reconstruct(normed))
        a, b = adapter(raw.reshape(33, 64), target), run(normed.reshape(33, 64), target)
        assert torch.equal(a["transcoder_out"], b["transcoder_out"]) and torch.equal(a["fvu"], b["fvu"])
    leaf = raw.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(adapter.reconstruct(leaf).sum(), [leaf])             # the gradient passes through the norm
    leaf2 = raw.clone().requires_grad_(True)
    (g2,) = torch.autograd.grad(run.reconstruct(norm(leaf2)).sum(), [leaf2])
    assert torch.equal(g, g2) and bool(g.any())
