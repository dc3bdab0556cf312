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

import contextlib
import ctypes as C
from typing import Optional

import torch
import torch.nn as nn

from . import _lib
from ._lib import BlockNormDesc, MtcError, check
from .engine import _p, _stream, dtype_code

_KINDS = {"rms": _lib.MTC_NORM_RMS, "layer": _lib.MTC_NORM_LAYER}
_NULL_CTX = contextlib.nullcontext()
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
        _kind_code(kind)
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
        return _apply(x, None, None, None, self, 1.0, 1.0)[1]

    def extra_repr(self) -> str:
        return (f"{self.width}, kind={self.kind!r}, eps={self.eps}, weight_offset={self.weight_offset}, "
                f"affine={self.weight is not None}, bias={self.bias is not None}")


class _Norm:
    """A norm given by its tensors (the functional form)."""
    __slots__ = ("width", "kind", "eps", "weight_offset", "weight", "bias")

    def __init__(self, width, kind, eps, weight_offset, weight, bias):
        self.width, self.kind, self.eps, self.weight_offset, self.weight, self.bias = width, kind, eps, weight_offset, weight, bias


def block_norm(x: torch.Tensor, weight=None, bias=None, *, kind: str = "rms", eps: float = 1e-6,
               weight_offset: float = 0.0) -> torch.Tensor:
    """One norm over the last dimension of x (any leading shape), differentiable in x, weight and bias."""
    return _apply(x, None, None, None, _Norm(x.shape[-1] if x.dim() else 0, kind, eps, weight_offset, weight, bias), 1.0, 1.0)[1]


def residual_block_norm(residual: torch.Tensor, branch: torch.Tensor, post: Optional[BlockNorm] = None, *, gate=None,
                        residual_scale: float = 1.0, branch_scale: float = 1.0, pre: Optional[BlockNorm] = None):
    """`hidden = residual_scale * residual + branch_scale * gate * post(branch)`; with `pre` (the norm in front of the next
    block) returns `(hidden, pre(hidden))` from the same pass, the norm taken of the sum before its rounding.

    residual and branch: one shape [..., width], one dtype (float32 or bfloat16), one GPU; leading dimensions may be strided
    or expanded.  gate: a scalar tensor, [width] (per channel), [..., 1] (per token) or the full shape.
    Differentiable in residual, branch, gate and both norms' parameters."""
    hidden, normed = _apply(residual, branch, gate, post, pre, float(residual_scale), float(branch_scale))
    return hidden if pre is None else (hidden, normed)


# ------------------------------------------------------------------------------------------------ plumbing
def _rows(t: torch.Tensor, A: int):
    """[rows, A] view (a copy only if the leading dimensions do not collapse or the columns are strided) and its row stride."""
    if t.dim() != 2:
        t = t.reshape(-1, A)
    if t.stride(1) != 1 and A > 1:
        t = t.contiguous()
    return t, t.stride(0)


def _vector(t, A: int, like: torch.Tensor, name: str):
    if t is None:
        return None
    if t.device != like.device or t.dtype != like.dtype or tuple(t.shape) != (A,):
        raise MtcError(f"{name} must be [{A}] of {like.dtype} on {like.device}, got {list(t.shape)} of {t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _gate_kind(gate, shape, like):
    """(code, gate) for a gate of one of the documented shapes."""
    if gate is None:
        return _lib.MTC_GATE_NONE, None
    if gate.device != like.device or gate.dtype != like.dtype:
        raise MtcError(f"gate must be {like.dtype} on {like.device}, got {gate.dtype} on {gate.device}")
    gs, A = tuple(gate.shape), shape[-1]
    if gs == (A,):
        return _lib.MTC_GATE_CHANNEL, gate
    if gs == () or gs == (1,):
        return _lib.MTC_GATE_SCALAR, gate
    if gs == shape:
        return _lib.MTC_GATE_FULL, gate
    if gs == shape[:-1] + (1,):
        return _lib.MTC_GATE_ROW, gate
    raise MtcError(f"gate of shape {list(gs)} fits neither a scalar, [{A}], {list(shape[:-1]) + [1]} nor {list(shape)}")


def _on(dev):
    return _NULL_CTX if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


class _Plan:
    """Shapes and constants of one call."""
    __slots__ = ("shape", "A", "code", "post", "pre", "gate_kind", "rs", "bs", "branch")

    def desc(self, rows, *, pre=True) -> BlockNormDesc:
        d = BlockNormDesc()
        d.rows, d.A, d.dtype, d.has_branch, d.gate_kind = rows, self.A, self.code, int(self.branch), self.gate_kind
        if self.post is not None:
            d.post_kind, d.post_eps, d.post_offset = self.post
        if self.pre is not None and pre:
            d.pre_kind, d.pre_eps, d.pre_offset = self.pre
        d.residual_scale, d.branch_scale = self.rs, self.bs
        return d


def _apply(residual, branch, gate, post, pre, rs, bs):
    if not residual.is_cuda:
        raise MtcError(f"the block norms run on the GPU only (HIP kernels); got a {residual.device} tensor and there is no CPU "
                       "fallback")
    if residual.dim() < 1:
        raise MtcError("a norm needs a tensor with at least one dimension")
    p = _Plan()
    p.shape, p.A, p.code = tuple(residual.shape), residual.shape[-1], dtype_code(residual.dtype)
    p.branch, p.rs, p.bs = branch is not None, rs, bs
    if not 1 <= p.A <= MAX_WIDTH:
        raise MtcError(f"norm width {p.A} outside 1..{MAX_WIDTH}")
    if p.branch and (branch.shape != residual.shape or branch.dtype != residual.dtype or branch.device != residual.device):
        raise MtcError(f"residual and branch must share shape, dtype and device: {list(residual.shape)} {residual.dtype} "
                       f"{residual.device} against {list(branch.shape)} {branch.dtype} {branch.device}")
    p.post = p.pre = None
    tensors = [residual, branch, None, None, None, None, None]
    for slot, n, what in ((3, post, "post"), (5, pre, "pre")):
        if n is None:
            continue
        if n.width != p.A:
            raise MtcError(f"{what} norm of width {n.width} on activations of width {p.A}")
        setattr(p, what, (_kind_code(n.kind), n.eps, n.weight_offset))
        tensors[slot] = _vector(n.weight, p.A, residual, what + " weight")
        tensors[slot + 1] = _vector(n.bias, p.A, residual, what + " bias")
    p.gate_kind, tensors[2] = _gate_kind(gate, p.shape, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        out = _BlockNormFn.apply(p, *tensors)
        return out if p.branch and p.pre is not None else (out, None) if p.branch else (None, out)
    return _forward(p, tensors, None)


def _operands(p: _Plan, residual, branch, gate):
    """Row views of the inputs and their strides, in the order of the C call."""
    res, ld_res = _rows(residual, p.A)
    br, ld_br = _rows(branch, p.A) if p.branch else (None, 0)
    g, ld_g = None, 0
    if p.gate_kind == _lib.MTC_GATE_CHANNEL:
        g = gate.contiguous()
    elif p.gate_kind == _lib.MTC_GATE_SCALAR:
        g = gate
    elif p.gate_kind == _lib.MTC_GATE_ROW:
        g, ld_g = _rows(gate, 1)
    elif p.gate_kind == _lib.MTC_GATE_FULL:
        g, ld_g = _rows(gate, p.A)
    return res, ld_res, br, ld_br, g, ld_g


def _forward(p: _Plan, tensors, stats):
    residual, branch, gate, post_w, post_b, pre_w, pre_b = tensors
    dev = residual.device
    hidden = torch.empty(p.shape, dtype=residual.dtype, device=dev) if p.branch else None
    normed = torch.empty(p.shape, dtype=residual.dtype, device=dev) if p.pre is not None else None
    rows = residual.numel() // p.A
    if rows:
        with _on(dev):
            res, ld_res, br, ld_br, g, ld_g = _operands(p, residual, branch, gate)
            d = p.desc(rows)
            d.ld_residual, d.ld_branch, d.ld_gate, d.ld_hidden, d.ld_normed = ld_res, ld_br, ld_g, p.A, p.A
            check(_lib.load().mtc_block_norm_fwd(C.byref(d), _p(res), _p(br), _p(g), _p(post_w), _p(post_b), _p(pre_w), _p(pre_b),
                                                 _p(hidden), _p(normed), _p(stats), _stream()), "mtc_block_norm_fwd")
    return hidden, normed


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, p, *tensors):
        residual = tensors[0]
        stats = torch.empty(residual.numel() // p.A, 4, dtype=torch.float32, device=residual.device)
        hidden, normed = _forward(p, tensors, stats)
        ctx.plan = p
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(stats, *tensors)
        return (hidden, normed) if p.branch and p.pre is not None else hidden if p.branch else normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        p = ctx.plan
        stats, residual, branch, gate, post_w, post_b, pre_w, pre_b = ctx.saved_tensors
        d_hidden = grads[0] if p.branch else None
        d_normed = None if p.pre is None else grads[-1]
        if d_hidden is None and d_normed is None:
            return (None,) * 8
        need = ctx.needs_input_grad[1:]
        dev, dt, rows = residual.device, residual.dtype, residual.numel() // p.A
        use_pre = d_normed is not None

        def new(i, shape, used=True):
            if not need[i]:
                return None
            return torch.empty(shape, dtype=dt, device=dev) if used and rows else torch.zeros(shape, dtype=dt, device=dev)

        with _on(dev):
            out = [new(0, p.shape), new(1, p.shape), new(2, None if gate is None else gate.shape), new(3, p.A), new(4, p.A),
                   new(5, p.A, use_pre), new(6, p.A, use_pre)]
            if rows:
                res, ld_res, br, ld_br, g, ld_g = _operands(p, residual, branch, gate)
                d = p.desc(rows, pre=use_pre)
                d.ld_residual, d.ld_branch, d.ld_gate = ld_res, ld_br, ld_g
                dh, ld_dh = (None, 0) if d_hidden is None else _rows(d_hidden, p.A)
                dn, ld_dn = _rows(d_normed, p.A) if use_pre else (None, 0)
                lib = _lib.load()
                ws, ws_bytes = None, 0
                if any(need[3:]) or (need[2] and p.gate_kind in (_lib.MTC_GATE_CHANNEL, _lib.MTC_GATE_SCALAR)):
                    ws_bytes = lib.mtc_block_norm_bwd_workspace_bytes(C.byref(d))
                    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
                ptrs = [_p(t) for t in out]
                if not use_pre:
                    ptrs[5] = ptrs[6] = None
                check(lib.mtc_block_norm_bwd(C.byref(d), _p(res), _p(br), _p(g), _p(post_w), _p(post_b), _p(pre_w), _p(pre_b),
                                             _p(stats), _p(dh), ld_dh, _p(dn), ld_dn, *ptrs, _p(ws), ws_bytes, _stream()),
                      "mtc_block_norm_bwd")
        return (None, *out)
