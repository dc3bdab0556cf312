"""What the gradient clipping refuses before any launch (no GPU needed)."""
import ctypes as C
import math

import pytest
import torch

from matryoshka_transcoder_amd import _lib
from matryoshka_transcoder_amd.grad_clip import clip_by_global_norm_, clip_grad_norm_, global_norm, norm_and_coef

GOOD = 0x10000


def _arrays(ptrs, elems, dtypes):
    n = len(ptrs)
    return (C.c_void_p * n)(*ptrs), (C.c_uint64 * n)(*elems), (C.c_int32 * n)(*dtypes)


def _clip(ptrs, outs, elems, dtypes, p=2.0, max_norm=1.0, ws=GOOD, nbytes=1 << 20):
    """Pointers are made up: every call here has to be refused on the host."""
    src, el, dt = _arrays(ptrs, elems, dtypes)
    dst = (C.c_void_p * len(outs))(*outs) if outs is not None else None
    rc = _lib.load().mtc_grad_clip(len(ptrs), src, dst, el, dt, p, max_norm, ws, nbytes, None, None)
    return rc, _lib.load().mtc_last_error().decode()


@pytest.mark.parametrize("kw,text", [
    (dict(p=3.0), "order"), (dict(p=float("nan")), "order"), (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"),
    (dict(dtypes=[5]), "bad dtype"), (dict(ptrs=[None]), "null or misaligned"), (dict(ptrs=[GOOD + 1]), "null or misaligned"),
    (dict(outs=[None]), "null or misaligned"), (dict(outs=None), "null output"), (dict(elems=[1 << 41]), "too many"),
    (dict(ws=None), "workspace"), (dict(ws=GOOD + 4), "workspace"), (dict(nbytes=4), "workspace"),
])
def test_c_refusals(kw, text):
    base = dict(ptrs=[GOOD * 16], outs=[GOOD * 16], elems=[100], dtypes=[_lib.MTC_F32])
    base.update(kw)
    rc, msg = _clip(**base)
    assert rc != 0 and text in msg, msg


@pytest.mark.parametrize("ptrs,outs,elems", [
    ([0x100000, 0x100000], [0x100000, 0x100000], [100, 100]),               # one tensor twice
    ([0x100000, 0x100100], [0x100000, 0x100100], [100, 100]),               # two views of one buffer that overlap
    ([0x100000], [0x100004], [100]),                                        # an output shifted against its input
    ([0x100000, 0x200000], [0x200000, 0x300000], [100, 100]),               # an output on another input
    ([0x100000, 0x200000], [0x300000, 0x300000], [100, 100]),               # one output twice
    ([0x100000, 0x200000, 0x100040], [0x100000, 0x200000, 0x400000], [1000, 10, 1]),    # a small input inside an output
])
def test_c_refuses_shared_memory(ptrs, outs, elems):
    rc, msg = _clip(ptrs, outs, elems, [_lib.MTC_F32] * len(ptrs))
    assert rc != 0 and "shares memory" in msg


def test_c_norm_refusals():
    lib = _lib.load()
    src, el, dt = _arrays([GOOD], [100], [_lib.MTC_F32])
    f = C.c_void_p(GOOD)
    assert lib.mtc_grad_norm(1, src, el, dt, 2.0, f, 1 << 20, None, 1.0, None, None) != 0 and b"no output" in lib.mtc_last_error()
    assert lib.mtc_grad_norm(1, src, el, dt, 0.0, f, 1 << 20, f, 1.0, f, None) != 0 and b"order" in lib.mtc_last_error()
    assert lib.mtc_grad_norm(1, src, el, dt, 2.0, f, 0, f, 1.0, f, None) != 0 and b"workspace" in lib.mtc_last_error()
    assert lib.mtc_grad_norm(-1, None, None, None, 2.0, f, 0, f, 1.0, f, None) != 0 and b"list" in lib.mtc_last_error()
    assert lib.mtc_grad_norm_coef(None, 2.0, 1.0, f, None) != 0 and b"null" in lib.mtc_last_error()
    assert lib.mtc_grad_norm_coef(f, 2.5, 1.0, f, None) != 0 and b"order" in lib.mtc_last_error()
    assert lib.mtc_grad_norm_workspace_bytes(-1, None, None) == 0
    h = _lib.AdamHyper()
    h.step = 1
    assert lib.mtc_adam_flat_scaled(_lib.MTC_F32, 8, f, f, f, f, C.byref(h), None, None) != 0 and b"grad_scale" in lib.mtc_last_error()
    d = _lib.make_desc(1, 32, 32, 256, [256], _lib.MTC_F32, False)
    assert lib.mtc_unitnorm_adam_rows_scaled(C.byref(d), f, f, f, f, C.byref(h), 0, None, None) != 0
    assert b"grad_scale" in lib.mtc_last_error()


def test_workspace_covers_any_list():
    """At least one fp64 partial per workgroup of every launch of up to 128 tensors."""
    lib = _lib.load()
    for elems in ([1], [0, 0], [16384], [16385], [10 ** 9] * 3, [1] * 1000, [10 ** 7] * 300, [0] * 500 + [5]):
        el, dt = (C.c_uint64 * len(elems))(*elems), (C.c_int32 * len(elems))(*[1] * len(elems))
        live = [e for e in elems if e]
        parts = 0
        for i in range(0, len(live), 128):
            parts += min(2048, sum((e + 8191) // 8192 for e in live[i:i + 128]))
        assert lib.mtc_grad_norm_workspace_bytes(len(elems), el, dt) >= 8 * (parts + 1)


def test_python_refusals():
    t = torch.ones(4)
    for call in (lambda: global_norm([t]), lambda: clip_by_global_norm_([t], 1.0), lambda: norm_and_coef(t, 1.0)):
        with pytest.raises(_lib.MtcError, match="no CPU fallback"):
            call()
    for p in (0, 3, float("nan"), -2):
        with pytest.raises(_lib.MtcError, match="order"):
            global_norm([], p)
        with pytest.raises(_lib.MtcError, match="order"):
            clip_by_global_norm_([], 1.0, p)
    for m in (-1.0, float("nan")):
        with pytest.raises(_lib.MtcError, match="max_norm"):
            clip_by_global_norm_([], m)
    assert float(global_norm([])) == 0.0 and float(clip_by_global_norm_([], 1.0, math.inf)) == 0.0
    assert float(clip_grad_norm_([torch.nn.Parameter(t)], 1.0)) == 0.0           # no .grad anywhere
