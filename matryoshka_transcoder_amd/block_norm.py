"""The norms around a block of a language model, fused with the block's gate and the residual add.

A transcoder replaces a model's MLP.  In the model that MLP sits between a norm that makes its input from the residual
stream (the transcoder's source activations, `hook_mlp_in`) and, in models with sandwich norms such as Gemma 2, a norm of its
output on the way back into the stream.  Both, with the residual add, an optional gate and constant scales, are one libmtc
launch (`mtc_block_norm_fwd`), and so is their gradient (`mtc_block_norm_bwd`, plus one small launch for the weights'):

    hidden = residual_scale * residual + branch_scale * gate * post(branch)
    normed = pre(hidden)                                            norm(x) = u * (weight_offset + weight) + bias

`BlockNorm` holds a norm's parameters, `block_norm` is one norm alone, `residual_block_norm` is the rest.  The reference
has no counterpart: it reads what these compute out of the model's cache (transcoder_activation_store.py:116-142).
Arithmetic is fp32; each output is rounded once to the model dtype.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _lib
from ._lib import MtcError

_KINDS = {"rms": _lib.MTC_NORM_RMS, "layer": _lib.MTC_NORM_LAYER}
MAX_WIDTH = 8192


def _kind_code(kind: str) -> int:
    try:
        return _KINDS[kind]
    except KeyError:
        raise MtcError(f"norm kind must be 'rms' or 'layer', got {kind!r}") from None


class BlockNorm(nn.Module):
    """Parameters of one norm over the last dimension (`width`).

    kind "rms": x / sqrt(mean(x^2) + eps); "layer": (x - mean) / sqrt(biased variance + eps); then
    `* (weight_offset + weight) + bias`.  weight_offset = 1 is Gemma's convention (weights around zero).
    affine = False: no weight; bias (default: only layer norms have one) needs affine = True."""

    def __init__(self, width: int, *, kind: str = "rms", eps: float = 1e-6, weight_offset: float = 0.0, affine: bool = True,
                 bias: Optional[bool] = None, dtype=None, device=None):
        super().__init__()
        self._code = _kind_code(kind)
        if not 1 <= int(width) <= MAX_WIDTH:
            raise MtcError(f"norm width {width} outside 1..{MAX_WIDTH}")
        if bias is None:
            bias = affine and kind == "layer"
        if bias and not affine:
            raise MtcError("a norm with bias needs affine = True")
        self.width, self.kind, self.eps, self.weight_offset = int(width), kind, float(eps), float(weight_offset)
        self.weight = nn.Parameter(torch.full((self.width,), 1.0 - self.weight_offset, dtype=dtype, device=device)) if affine else None
        self.bias = nn.Parameter(torch.zeros(self.width, dtype=dtype, device=device)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _call(x, None, None, None, self, 1.0, 1.0)[1]

    def saved_form(self) -> dict:
        """Everything the norm consists of, for a file (numbers, text and tensors only); `from_saved` makes it again."""
        return {"spec": {"width": self.width, "kind": self.kind, "eps": self.eps, "weight_offset": self.weight_offset,
                         "affine": self.weight is not None, "bias": self.bias is not None},
                "state_dict": {k: v.detach().clone() for k, v in self.state_dict().items()}}

    @classmethod
    def from_saved(cls, saved: dict, device=None) -> "BlockNorm":
        if "spec" not in saved:
            raise MtcError("the saved source_norm is not a BlockNorm and cannot be made again from its file")
        state, spec = saved["state_dict"], dict(saved["spec"])
        norm = cls(spec.pop("width"), **spec, dtype=state["weight"].dtype if "weight" in state else None, device=device)
        norm.load_state_dict(state)
        return norm

    def extra_repr(self) -> str:
        return (f"{self.width}, kind={self.kind!r}, eps={self.eps}, weight_offset={self.weight_offset}, "
                f"affine={self.weight is not None}, bias={self.bias is not None}")


class _Norm:
    """A norm given by its tensors (the functional form)."""
    __slots__ = ("width", "_code", "eps", "weight_offset", "weight", "bias")

    def __init__(self, width, kind, eps, weight_offset, weight, bias):
        self.width, self._code, self.eps, self.weight_offset = width, _kind_code(kind), eps, weight_offset
        self.weight, self.bias = weight, bias


def block_norm(x: torch.Tensor, weight=None, bias=None, *, kind: str = "rms", eps: float = 1e-6,
               weight_offset: float = 0.0) -> torch.Tensor:
    """One norm over the last dimension of x (any leading shape), differentiable in x, weight and bias."""
    return _call(x, None, None, None, _Norm(x.shape[-1] if x.dim() else 0, kind, eps, weight_offset, weight, bias), 1.0, 1.0)[1]


def residual_block_norm(residual: torch.Tensor, branch: torch.Tensor, post: Optional[BlockNorm] = None, *, gate=None,
                        residual_scale: float = 1.0, branch_scale: float = 1.0, pre: Optional[BlockNorm] = None):
    """`hidden = residual_scale * residual + branch_scale * gate * post(branch)`; with `pre` (the norm in front of the next
    block) returns `(hidden, pre(hidden))` from the same pass, the norm taken of the sum before its rounding.

    residual and branch: one shape [..., width], one dtype (float32 or bfloat16), one GPU; leading dimensions may be strided
    or expanded.  gate: a scalar tensor, [width] (per channel), [..., 1] (per token) or the full shape; it multiplies, so an infinity or
    NaN in the branch outlives a gate of 0.
    Differentiable in residual, branch, gate and both norms' parameters, once: a backward with create_graph = True raises, and
    so do forward-mode tangents, tracing (torch.jit.trace, make_fx) and a backward recorded into a HIP graph while an eager graph of
    the same leaves is alive."""
    if branch is None:
        raise MtcError("residual_block_norm needs a branch: block_norm (or a BlockNorm) norms the residual alone")
    hidden, normed = _call(residual, branch, gate, post, pre, residual_scale, branch_scale)
    return hidden if pre is None else (hidden, normed)


def _call(residual, branch, gate, post, pre, rs, bs):
    """One pass through csrc/torch_binding.cpp (checks, outputs, launch, autograd node): (hidden or None, normed or None)."""
    norms = []
    for n in (post, pre):
        norms += (0, None, None, 0.0, 0.0, 0) if n is None else (n._code, n.weight, n.bias, n.eps, n.weight_offset, n.width)
    return _lib.torch_binding().block_norm(residual, branch, gate, *norms, rs, bs)
