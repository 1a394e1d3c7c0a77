"""The feed-forward sublayer of a language model on the omarchy_mac_torch device, for training and for serving:

    h = x + residual                                 (the stream, handed on)
    y = h / sqrt(mean(h^2) + eps) * weight           RMSNorm
    out = (act(y Wg^T) * (y Wu^T)) Wd^T              GatedFeedForward

Differentiable functions (rms_norm, glu) and modules over torch.ops.omt's operators; the down projection is the device's
own linear layer. Training keeps the block's activations in 8 bits by default (checkpoint="fp8": one byte and 4/128 for
each value of x and of both projections, where float32 takes 4), or whole ("full"). serve() gives the sublayer with its
weights in 8 bits, whose activations are quantized where they are produced: three launches and their sums for a token.

No counterpart in the reference. hip_ops has the same operators as plain functions, for torch.cuda tensors too.
"""

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from omarchy_mac_torch import hip_ops

__all__ = ["FeedForward", "GatedFeedForward", "RMSNorm", "ServedFeedForward", "glu", "rms_norm"]


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = hip_ops.rms_norm(x, weight, residual, eps)
        ctx.save_for_backward(h, weight, rstd)
        ctx.added = residual is not None
        return (y, h) if ctx.added else y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gh=None):
        h, weight, rstd = ctx.saved_tensors
        gx, gw = hip_ops.rms_norm_backward(gy, h, weight, rstd, gh=gh, weight_grad=ctx.needs_input_grad[1])
        return gx, gw, gx if ctx.added else None, None


class _Glu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act, checkpoint):
        h, kept = hip_ops.glu(x, w_gate, w_up, act, checkpoint)
        ctx.save_for_backward(w_gate, w_up, *kept)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, gh):
        w_gate, w_up, *kept = ctx.saved_tensors
        need_x, *need_w = ctx.needs_input_grad[:3]
        gx, gwg, gwu = hip_ops.glu_backward(gh, kept, w_gate, w_up, ctx.act, input_grad=need_x,
                                            weight_grad=any(need_w))
        return gx, gwg if need_w[0] else None, gwu if need_w[1] else None, None, None


@torch.compiler.disable  # one operator each way: nothing for a compiler to fuse
def rms_norm(x, weight, residual=None, eps=1e-6):
    """hip_ops.rms_norm, differentiable: y, or (y, h) with a residual."""
    return _RmsNorm.apply(x, weight, residual, eps)


@torch.compiler.disable
def glu(x, w_gate, w_up, act="silu", checkpoint="fp8"):
    """hip_ops.glu's h, differentiable; `checkpoint` says how x and both projections are kept for the backward: "fp8" or
    "full". Nothing is kept where no gradient can be asked for."""
    if checkpoint not in ("fp8", "full"):
        raise ValueError(f"checkpoint: expected 'fp8' or 'full', got {checkpoint!r}")
    # (inside the function grad mode is always off, and ctx.needs_input_grad says what the inputs require whatever the mode)
    if not torch.is_grad_enabled() or not any(t.requires_grad for t in (x, w_gate, w_up)):
        return hip_ops.glu(x, w_gate, w_up, act)[0]
    return _Glu.apply(x, w_gate, w_up, act, checkpoint)


class RMSNorm(nn.Module):
    """rms_norm over the last dimension with a learned weight: forward(x) gives y, forward(x, residual) gives (y, h)."""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual, self.eps)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}"


class GatedFeedForward(nn.Module):
    """(act(x gate^T) * (x up^T)) down^T, no biases."""

    def __init__(self, dim, hidden, act="silu", checkpoint="fp8"):
        super().__init__()
        self.gate = nn.Parameter(torch.empty(hidden, dim))
        self.up = nn.Parameter(torch.empty(hidden, dim))
        self.down = nn.Linear(hidden, dim, bias=False)
        self.act, self.checkpoint = act, checkpoint
        for w in (self.gate, self.up):
            nn.init.normal_(w, std=dim ** -0.5)
        nn.init.normal_(self.down.weight, std=hidden ** -0.5)

    def forward(self, x):
        return self.down(glu(x, self.gate, self.up, self.act, self.checkpoint))

    def extra_repr(self):
        return f"act={self.act!r}, checkpoint={self.checkpoint!r}"


class FeedForward(nn.Module):
    """The sublayer: forward(x, residual) adds x, the last sublayer's output, to the residual stream and returns (this
    sublayer's output, the stream); forward(x) starts the stream with x."""

    def __init__(self, dim, hidden, act="silu", checkpoint="fp8", eps=1e-6):
        super().__init__()
        self.norm = RMSNorm(dim, eps)
        self.ffn = GatedFeedForward(dim, hidden, act, checkpoint)

    def forward(self, x, residual=None):
        y, h = (self.norm(x), x) if residual is None else self.norm(x, residual)
        return self.ffn(y), h

    def serve(self):
        return ServedFeedForward(self)


class ServedFeedForward(nn.Module):
    """A FeedForward with its weights in 8 bits, scales by 128 x 128, for inference: forward as FeedForward's. The norm and
    the block give their results in 8 bits, scales by 128 along each row; the output is of the stream's type."""

    def __init__(self, block):
        super().__init__()
        self.eps, self.act = block.norm.eps, block.ffn.act
        self.register_buffer("weight", block.norm.weight.detach().clone())
        for name, w in (("gate", block.ffn.gate), ("up", block.ffn.up), ("down", block.ffn.down.weight)):
            q, scale = hip_ops.quantize_fp8_weight(w.detach())
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", scale)

    def _apply(self, fn, recurse=True):
        # a change of type (to(dtype), float(), bfloat16()) is for the norm's weight: values in 8 bits and their scales move only
        def apply(t):
            if t is not self.weight:
                like = fn(t.new_empty(0))
                if like.dtype != t.dtype:
                    return t.to(like.device)
            return fn(t)
        return super()._apply(apply, recurse)

    @torch.compiler.disable
    @torch.no_grad()
    def forward(self, x, residual=None):
        q, scale, h = hip_ops.rms_norm_fp8(x, self.weight, residual, self.eps)
        q, scale = hip_ops.glu_fp8(q, scale, self.gate, self.gate_scale, self.up, self.up_scale, self.act)
        return hip_ops.matmul_fp8(q, scale, self.down, self.down_scale, dtype=x.dtype), h
