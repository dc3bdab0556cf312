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
from .engine import _stream

Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]


def _list(tensors: Tensors) -> List[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def norm_and_coef(tensors: Tensors, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """float32 [2] on the GPU: the norm and the factor that clips to max_norm."""
    return _lib.torch_binding().norm_of(_list(tensors), float(norm_type), float(max_norm), False)


def power_sum(tensors: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """float64 scalar on the GPU: the norm's sum before its root (p = inf: the maximum), to be combined over ranks."""
    return _lib.torch_binding().norm_of(_list(tensors), float(norm_type), math.inf, True)


def coef_of_power_sum(total: torch.Tensor, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """`norm_and_coef` of gradients whose combined `power_sum` is `total`."""
    _lib.torch_binding().refuse_tracing("a gradient norm")
    if not total.is_cuda or total.dtype != torch.float64 or total.numel() != 1:
        raise MtcError("total must be one float64 value on the GPU")
    with torch.cuda.device(total.device):
        out = torch.empty(2, dtype=torch.float32, device=total.device)
        check(_lib.load().mtc_grad_norm_coef(C.c_void_p(total.data_ptr()), float(norm_type), float(max_norm),
                                             C.c_void_p(out.data_ptr()), _stream()), "mtc_grad_norm_coef")
    return out


def global_norm(tensors: Tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm over all elements of all tensors: a float32 scalar on their GPU (0 on the CPU for an empty list)."""
    ts = _list(tensors)
    return norm_and_coef(ts, math.inf, norm_type)[0] if ts else clip_by_global_norm_(ts, math.inf, norm_type)


def clip_by_global_norm_(tensors: Tensors, max_norm: float, norm_type: float = 2.0, *, error_if_nonfinite: bool = False,
                         out: Optional[Iterable[torch.Tensor]] = None) -> torch.Tensor:
    """Scale the tensors in place so that their common norm is at most max_norm; returns the norm before (float32 scalar).

    out: tensors of the same shapes and dtypes that receive the scaled values instead; the inputs then stay as they are.
    Dense tensors (and outputs) that share memory with one another are refused; outputs laid out unlike their inputs are written by
    a copy, and must not span the same memory as any other output.  Nothing is written, in place, when the norm
    is within the limit.  error_if_nonfinite: raise before anything is changed if the norm is not finite (reads it back: a
    synchronisation)."""
    src = _list(tensors)
    if error_if_nonfinite and src and not math.isfinite(float(global_norm(src, norm_type))):
        raise RuntimeError(f"the total norm of order {norm_type} of the gradients is non-finite, so it cannot be clipped")
    return _lib.torch_binding().clip(src, None if out is None else _list(out), float(norm_type), float(max_norm))


def clip_grad_norm_(parameters: Tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """`torch.nn.utils.clip_grad_norm_` for parameters on one GPU: clips every `.grad` that is there, returns the norm."""
    return clip_by_global_norm_([q.grad for q in _list(parameters) if q.grad is not None], max_norm, norm_type,
                                error_if_nonfinite=error_if_nonfinite)
