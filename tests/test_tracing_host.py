"""Recorders of torch operations see an output's allocation and not the kernel that fills it: a trace of these calls would return
memory nobody wrote.  They are refused (no GPU needed: the refusal comes before everything else)."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from matryoshka_transcoder_amd import _lib
from matryoshka_transcoder_amd.block_norm import BlockNorm, block_norm, residual_block_norm
from matryoshka_transcoder_amd.grad_clip import clip_by_global_norm_, coef_of_power_sum, global_norm, norm_and_coef, power_sum
from matryoshka_transcoder_amd.transcoder import MatryoshkaTranscoder


def _reconstruct(x):
    cfg = dict(seed=3, prefix_sizes=[16, 64], dict_size=64, act_size=8, top_k=4, top_k_aux=8, aux_penalty=1 / 32, n_batches_to_dead=20,
               l1_coeff=0.0, dtype=torch.float32, device="cpu")
    model = getattr(_reconstruct, "model", None) or MatryoshkaTranscoder(cfg)
    _reconstruct.model = model
    return model.reconstruct(x)


CALLS = {
    "block_norm": lambda x: block_norm(x),
    "residual_block_norm": lambda x: residual_block_norm(x, x),
    "global_norm": lambda x: global_norm([x]),
    "norm_and_coef": lambda x: norm_and_coef([x], 1.0),
    "power_sum": lambda x: power_sum([x]),
    "coef_of_power_sum": lambda x: coef_of_power_sum(x.sum().double(), 1.0),
    "clip": lambda x: clip_by_global_norm_([x], 1.0),
    "reconstruct": _reconstruct,
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused(name):
    x = torch.randn(3, 8)
    call = lambda x: CALLS[name](x)                                          # noqa: E731
    for record in (lambda f: torch.jit.trace(f, (x,)), lambda f: make_fx(f)(x), lambda f: make_fx(f, pre_dispatch=True)(x)):
        with pytest.raises(_lib.MtcError, match="trace"):
            record(call)
    with pytest.raises(_lib.MtcError, match="GPU"):                          # and nothing stays behind: the ordinary refusal again
        CALLS[name](x)


@pytest.mark.filterwarnings("ignore")
def test_a_module_cannot_be_traced():
    with pytest.raises(_lib.MtcError, match="trace"):
        torch.jit.trace(BlockNorm(8), (torch.randn(3, 8),))
    with pytest.raises(_lib.MtcError, match="trace"):
        torch.export.export(BlockNorm(8), (torch.randn(3, 8),), strict=False)
