"""A transcoder in its model's block, where the MLP was.

    x      = pre(h)                                              the block's norm in front of its MLP: the transcoder's source
    h_next = residual_scale * h + branch_scale * gate * post(T(x))        and, in models with sandwich norms, the one behind it

(Gemma 2: pre = RMS norm with weight offset 1, post likewise; GPT-2: pre = layer norm, no post.)  With the attention's
output given, the residual add in front of the MLP and the norm of its sum are one pass as well:

    h = h_in + attn_post(attn_out),  x = pre(h)

The norms, gate and adds run as block norms (block_norm.py); T is `MatryoshkaTranscoder.reconstruct`.  Everything is
differentiable, so the transcoder, the gate and the norms can be trained on the model's own loss; clip_grad_norm_
(grad_clip.py) takes all their gradients at once.  The reference only compares reconstructions outside the model
(eval/sae_bench/wrappers.py:100-109).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from ._lib import MtcError
from .block_norm import BlockNorm, residual_block_norm
from .transcoder import MatryoshkaTranscoder


class SplicedTranscoder(nn.Module):
    """Stands in for the second half of a transformer block.

    pre / post / attn_post: the model's own norms as BlockNorm (copy their weights in); post and attn_post only where the model
    has them.  gate: None, or "scalar" / "channel" for a learned gate that starts at 1.  Freeze what should not train with
    requires_grad_(False)."""

    def __init__(self, transcoder: MatryoshkaTranscoder, pre: BlockNorm, post: Optional[BlockNorm] = None, *,
                 attn_post: Optional[BlockNorm] = None, gate: Optional[str] = None, residual_scale: float = 1.0,
                 branch_scale: float = 1.0):
        super().__init__()
        width = transcoder.source_act_size
        if transcoder.target_act_size != width:
            raise MtcError(f"a spliced transcoder writes to the stream it reads: widths {width} and {transcoder.target_act_size} differ")
        for name, n in (("pre", pre), ("post", post), ("attn_post", attn_post)):
            if n is not None and n.width != width:
                raise MtcError(f"{name} norm of width {n.width} around a transcoder of width {width}")
        if pre is None:
            raise MtcError("a spliced transcoder needs the norm in front of it")
        self.transcoder, self.pre, self.post, self.attn_post = transcoder, pre, post, attn_post
        self.residual_scale, self.branch_scale = float(residual_scale), float(branch_scale)
        shape = {None: None, "scalar": (), "channel": (width,)}.get(gate, "?")
        if shape == "?":
            raise MtcError(f"gate must be None, 'scalar' or 'channel', got {gate!r}")
        self.gate = None if shape is None else nn.Parameter(torch.ones(shape, dtype=transcoder.dtype, device=transcoder.W_dec.device))

    def forward(self, residual: torch.Tensor, attn_out: Optional[torch.Tensor] = None, *, token_gate=None) -> torch.Tensor:
        """residual [..., width] -> the stream behind the block.  attn_out: the attention's output, added (through attn_post) in
        the same pass as the norm in front of the transcoder.  token_gate [..., 1]: a gate per token (0 keeps a token out of
        the splice), instead of the learned one."""
        if token_gate is not None and self.gate is not None:
            raise MtcError("give either a learned gate or token_gate, not both")
        if attn_out is None:
            if self.attn_post is not None:
                raise MtcError("attn_post needs attn_out")
            x = self.pre(residual)
        else:
            residual, x = residual_block_norm(residual, attn_out, self.attn_post, pre=self.pre)
        y = self.transcoder.reconstruct(x)
        return residual_block_norm(residual, y, self.post, gate=self.gate if token_gate is None else token_gate,
                                   residual_scale=self.residual_scale, branch_scale=self.branch_scale)
