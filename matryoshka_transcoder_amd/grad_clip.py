"""One norm over all gradients, and clipping by it: the `max_grad_norm` of the configuration (config.py:70), which the
reference defines and never applies.

    norm = (sum over all tensors of |g|^p)^(1/p),   p in {1, 2, inf}        coef = min(1, max_norm / (norm + 1e-6))
    g <- round(g * coef)

`clip_grad_norm_` takes parameters like `torch.nn.utils.clip_grad_norm_`; `clip_by_global_norm_` and `global_norm` take the
gradients themselves.  float32 and bfloat16 tensors may be mixed; the norm is a float32 scalar on their GPU (sums are held in 64
bits), and nothing is read back to the host.  A NaN anywhere makes the norm and every clipped gradient NaN, an infinity makes
coef 0, as in torch.  `FusedAdam(max_grad_norm=...)` applies the coefficient while it reads the gradients instead.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Iterable, List, Optional, Union

import torch

from . import _lib
from ._lib import MtcError, check
from .block_norm import _on
from .engine import _stream

_CODES = {torch.float32: _lib.MTC_F32, torch.bfloat16: _lib.MTC_BF16}
Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]


def _order(norm_type) -> float:
    p = float(norm_type)
    if p not in (1.0, 2.0, math.inf):
        raise MtcError(f"the norm's order must be 1, 2 or inf, got {norm_type}")
    return p


def _limit(max_norm) -> float:
    m = float(max_norm)
    if not m >= 0.0:
        raise MtcError(f"max_norm must not be negative or NaN, got {max_norm}")
    return m


def _dense(t: torch.Tensor) -> bool:
    """Every element once, without gaps, in some order of the dimensions (a transposed view, a channels-last gradient)."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _listed(tensors: Tensors) -> List[torch.Tensor]:
    ts = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    dev = None
    for t in ts:
        if not t.is_cuda:
            raise MtcError(f"gradient clipping runs on the GPU only (HIP kernels); got a {t.device} tensor and there is no CPU fallback")
        if t.dtype not in _CODES:
            raise MtcError(f"gradients must be float32 or bfloat16, got {t.dtype}")
        if t.layout is not torch.strided:
            raise MtcError(f"gradients must be dense tensors, got {t.layout}")
        if dev is None:
            dev = t.get_device()
        elif t.get_device() != dev:
            raise MtcError(f"all gradients must live on one GPU, got cuda:{dev} and {t.device}")
    return ts


class _Call:
    """Host arrays and workspace of one call over a list of dense tensors."""
    __slots__ = ("n", "src", "elems", "dtype", "ws", "ws_bytes", "lib")

    def __init__(self, ts: List[torch.Tensor]):
        self.lib = _lib.load()
        n = self.n = len(ts)
        self.src = (C.c_void_p * n)(*[t.data_ptr() for t in ts])
        self.elems = (C.c_uint64 * n)(*[t.numel() for t in ts])
        self.dtype = (C.c_int32 * n)(*[_CODES[t.dtype] for t in ts])
        self.ws_bytes = self.lib.mtc_grad_norm_workspace_bytes(n, self.elems, self.dtype)
        self.ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=ts[0].device)

    def norm(self, p, total=None, max_norm=math.inf, norm_coef=None):
        ptr = lambda t: None if t is None else C.c_void_p(t.data_ptr())       # noqa: E731
        check(self.lib.mtc_grad_norm(self.n, self.src, self.elems, self.dtype, p, C.c_void_p(self.ws.data_ptr()), self.ws_bytes,
                                     ptr(total), max_norm, ptr(norm_coef), _stream()), "mtc_grad_norm")

    def clip(self, p, dst: List[torch.Tensor], max_norm, norm):
        out = (C.c_void_p * self.n)(*[t.data_ptr() for t in dst])
        check(self.lib.mtc_grad_clip(self.n, self.src, out, self.elems, self.dtype, p, max_norm, C.c_void_p(self.ws.data_ptr()),
                                     self.ws_bytes, C.c_void_p(norm.data_ptr()), _stream()), "mtc_grad_clip")


@torch.no_grad()
def norm_and_coef(tensors: Tensors, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """float32 [2] on the GPU: the norm and the factor that clips to max_norm."""
    ts = [t if _dense(t) else t.contiguous() for t in _listed(tensors)]
    p, max_norm = _order(norm_type), _limit(max_norm)
    if not ts:
        raise MtcError("no gradients to take a norm of")
    with _on(ts[0].device):
        out = torch.empty(2, dtype=torch.float32, device=ts[0].device)
        _Call(ts).norm(p, max_norm=max_norm, norm_coef=out)
    return out


@torch.no_grad()
def power_sum(tensors: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """float64 scalar on the GPU: the norm's sum before its root (p = inf: the maximum), to be combined over ranks."""
    ts = [t if _dense(t) else t.contiguous() for t in _listed(tensors)]
    if not ts:
        raise MtcError("no gradients to take a norm of")
    with _on(ts[0].device):
        out = torch.empty((), dtype=torch.float64, device=ts[0].device)
        _Call(ts).norm(_order(norm_type), total=out)
    return out


@torch.no_grad()
def coef_of_power_sum(total: torch.Tensor, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """`norm_and_coef` of gradients whose combined `power_sum` is `total`."""
    if not total.is_cuda or total.dtype != torch.float64 or total.numel() != 1:
        raise MtcError("total must be one float64 value on the GPU")
    with _on(total.device):
        out = torch.empty(2, dtype=torch.float32, device=total.device)
        check(_lib.load().mtc_grad_norm_coef(C.c_void_p(total.data_ptr()), _order(norm_type), _limit(max_norm),
                                             C.c_void_p(out.data_ptr()), _stream()), "mtc_grad_norm_coef")
    return out


def global_norm(tensors: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm over all elements of all tensors: a float32 scalar on their GPU (0 on the CPU for an empty list)."""
    ts = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not ts:
        _order(norm_type)
        return torch.zeros(())
    return norm_and_coef(ts, math.inf, norm_type)[0]


@torch.no_grad()
def clip_by_global_norm_(tensors: Tensors, max_norm: float, norm_type: float = 2.0, *, error_if_nonfinite: bool = False,
                         out: Optional[Iterable[torch.Tensor]] = None) -> torch.Tensor:
    """Scale the tensors in place so that their common norm is at most max_norm; returns the norm before (float32 scalar).

    out: tensors of the same shapes and dtypes that receive the scaled values instead; the inputs then stay as they are.
    Dense tensors (and outputs) that share memory with one another are refused.  Nothing is written, in place, when the norm is
    within the limit.  error_if_nonfinite: raise before anything is changed if the norm is not finite (reads it back: a
    synchronisation)."""
    p, max_norm = _order(norm_type), _limit(max_norm)
    src = _listed(tensors)
    dst = src if out is None else _listed(out)
    if not src:
        if dst:
            raise MtcError("out has tensors but there are none to clip")
        return torch.zeros(())
    if dst is not src:
        if len(dst) != len(src):
            raise MtcError(f"{len(src)} tensors but {len(dst)} outputs")
        for i, (s, o) in enumerate(zip(src, dst)):
            if s.shape != o.shape or s.dtype != o.dtype or s.device != o.device:
                raise MtcError(f"output {i} must be {list(s.shape)} of {s.dtype} on {s.device}, got {list(o.shape)} of {o.dtype} on {o.device}")
    for o in dst:
        if any(st == 0 and sz > 1 for st, sz in zip(o.stride(), o.shape)):
            raise MtcError("a tensor that repeats its memory (expanded) cannot be clipped in place")
    dev = src[0].device
    with _on(dev):
        # the kernel walks over memory: inputs with gaps, or outputs laid out another way, go through a dense copy
        a, b, back = [], [], []
        for s, o in zip(src, dst):
            if not _dense(s):
                s = s.contiguous()
            if o.stride() != s.stride() and s.numel():
                back.append((o, torch.empty_like(s)))
                o = back[-1][1]
            a.append(s)
            b.append(o)
        call = _Call(a)
        if error_if_nonfinite:
            check_norm = torch.empty(2, dtype=torch.float32, device=dev)
            call.norm(p, norm_coef=check_norm)
            if not math.isfinite(float(check_norm[0])):
                raise RuntimeError(f"the total norm of order {norm_type} of the gradients is non-finite, so it cannot be clipped")
        norm = torch.empty((), dtype=torch.float32, device=dev)
        call.clip(p, b, max_norm, norm)
        for o, tmp in back:
            o.copy_(tmp)
    return norm


def clip_grad_norm_(parameters: Tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """`torch.nn.utils.clip_grad_norm_` for parameters on one GPU: clips every `.grad` that is there, returns the norm."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_by_global_norm_([q.grad for q in params if q.grad is not None], max_norm, norm_type,
                                error_if_nonfinite=error_if_nonfinite)
