"""What the block norms refuse before any launch (no GPU needed)."""
import ctypes as C
import json
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from matryoshka_transcoder_amd import _lib
from matryoshka_transcoder_amd.block_norm import BlockNorm, block_norm, residual_block_norm


def _desc(**kw):
    base = dict(rows=4, A=64, dtype=_lib.MTC_F32, has_branch=1, post_kind=_lib.MTC_NORM_RMS, pre_kind=_lib.MTC_NORM_RMS,
                residual_scale=1.0, branch_scale=1.0, ld_residual=64, ld_branch=64, ld_hidden=64, ld_normed=64)
    base.update(kw)
    return _lib.BlockNormDesc(**base)


def _fwd(d, residual=1, branch=1, gate=None, hidden=1, normed=1):
    """Pointers are made up: every call here has to be refused on the host."""
    fake = lambda v: C.c_void_p(0x10000) if v else None      # noqa: E731
    return _lib.load().mtc_block_norm_fwd(C.byref(d), fake(residual), fake(branch), fake(gate), None, None, None, None, fake(hidden),
                                          fake(normed), None, None)


@pytest.mark.parametrize("kw,call,text", [
    (dict(dtype=7), {}, "dtype"), (dict(A=0), {}, "width"), (dict(A=8193), {}, "width"), (dict(rows=-1), {}, "row count"),
    (dict(post_kind=5), {}, "norm kind"), (dict(pre_kind=-1), {}, "norm kind"), (dict(gate_kind=9), {}, "gate kind"),
    (dict(has_branch=0), {}, "need a branch"), (dict(has_branch=0, post_kind=0, residual_scale=0.5), {}, "need a branch"),
    (dict(has_branch=0, post_kind=0, pre_kind=0), {}, "neither"), (dict(ld_branch=-64), {}, "negative"),
    ({}, dict(residual=None), "null residual"), ({}, dict(branch=None), "has_branch disagree"),
    ({}, dict(gate=1), "gate_kind disagree"), (dict(gate_kind=1), {}, "gate_kind disagree"),
    ({}, dict(hidden=None), "hidden"), ({}, dict(normed=None), "normed"), (dict(ld_hidden=8), {}, "overlap"),
])
def test_c_refusals(kw, call, text):
    assert _fwd(_desc(**kw), **call) != 0
    assert text in _lib.load().mtc_last_error().decode()


def test_c_backward_refusals():
    lib = _lib.load()
    f = C.c_void_p(0x10000)

    def bwd(d, stats=f, d_normed=f, outs=(f,) * 7, ws=f, nbytes=1 << 30):
        return lib.mtc_block_norm_bwd(C.byref(d), f, f if d.has_branch else None, f if d.gate_kind else None, None, None, None, None,
                                      stats, f if d.has_branch else None, 64, d_normed, 64, *outs, ws, nbytes, None)

    none_gate = (f, f, None, f, f, f, f)
    for d, kw, text in ((_desc(), {}, "absent gate"), (_desc(), dict(outs=none_gate, stats=None), "null stats"),
                        (_desc(), dict(outs=none_gate, d_normed=None), "d_normed"),
                        (_desc(), dict(outs=none_gate, nbytes=64), "workspace too small"),
                        (_desc(), dict(outs=none_gate, ws=None), "workspace too small"),
                        (_desc(), dict(outs=none_gate, ws=C.c_void_p(0x10004)), "16-byte"),
                        (_desc(post_kind=0), dict(outs=none_gate), "absent post norm"),
                        (_desc(pre_kind=0), dict(outs=none_gate, d_normed=None), "absent pre norm"),
                        (_desc(has_branch=0, post_kind=0), dict(outs=none_gate), "absent branch"),
                        (_desc(rows=0), dict(outs=none_gate), "no rows")):
        assert bwd(d, **kw) != 0, text
        assert text in lib.mtc_last_error().decode(), (text, lib.mtc_last_error())
    assert lib.mtc_block_norm_bwd_workspace_bytes(C.byref(_desc())) > 0
    assert lib.mtc_block_norm_bwd_workspace_bytes(C.byref(_desc(A=-3))) == 0
    assert lib.mtc_block_norm_fwd(C.byref(_desc(rows=0)), *([None] * 11)) == 0      # nothing to do, nothing touched


def test_python_refusals():
    x = torch.randn(4, 64)
    for call in (lambda: block_norm(x), lambda: residual_block_norm(x, x), lambda: BlockNorm(64)(x)):
        with pytest.raises(_lib.MtcError, match="no CPU fallback"):
            call()
    with pytest.raises(_lib.MtcError, match="norm kind"):
        BlockNorm(64, kind="group")
    for width in (0, 8193):
        with pytest.raises(_lib.MtcError, match="outside"):
            BlockNorm(width)
    with pytest.raises(_lib.MtcError, match="affine"):
        BlockNorm(64, affine=False, bias=True)


def test_module_parameters():
    m = BlockNorm(64, kind="rms", weight_offset=1.0, dtype=torch.bfloat16)
    assert list(m.state_dict()) == ["weight"] and not bool(m.weight.any()) and m.weight.dtype == torch.bfloat16
    m = BlockNorm(64, kind="layer")
    assert list(m.state_dict()) == ["weight", "bias"] and bool((m.weight == 1).all()) and not bool(m.bias.any())
    assert list(BlockNorm(64, affine=False).state_dict()) == []


def test_a_run_with_a_source_norm_can_be_saved(tmp_path):
    """The configuration of a run is written as JSON with every checkpoint: a module in it appears by its description."""
    from matryoshka_transcoder_amd.activation_store import TranscoderActivationsStore
    from matryoshka_transcoder_amd.results import CleanResultsManager
    results = CleanResultsManager(str(tmp_path))
    run = results.create_experiment_dir("m", 0, 1)
    cfg = {"dtype": torch.bfloat16, "act_size": 64, "device": "cpu", "source_norm": BlockNorm(64)}
    results.save_checkpoint(run, torch.nn.Linear(2, 2), cfg, 1)
    saved = json.loads((run / "config.json").read_text())
    assert saved["source_norm"].startswith("BlockNorm(64, kind='rms'")
    with pytest.raises(_lib.MtcError, match="source_norm"):                 # what was saved is no module any more
        TranscoderActivationsStore(None, dict(cfg, source_norm=saved["source_norm"]))


def test_the_binding_loads_in_a_process_without_torch():
    """`_lib` itself imports no torch: the binding brings the libraries it links against."""
    code = "from matryoshka_transcoder_amd import _lib; assert _lib.torch_binding() is _lib.torch_binding()"
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=str(Path(__file__).resolve().parents[1]))


def test_a_residual_without_a_branch_is_refused():
    """residual_block_norm adds a branch; a norm of the residual alone is block_norm's (and hidden would be nothing)."""
    x = torch.randn(4, 64)
    for kw in ({}, dict(pre=BlockNorm(64)), dict(post=BlockNorm(64)), dict(gate=torch.ones(()))):
        with pytest.raises(_lib.MtcError, match="branch"):
            residual_block_norm(x, None, **kw)
