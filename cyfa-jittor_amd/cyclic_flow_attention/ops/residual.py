"""The join between two blocks of a model on the gfx950 HIP path: a block's
output norm and gate, the scaled residual add and the next block's norm
(CyFABlock.execute, models/cyfa/modeling_cyfa.py:48-51 of Chyxx/CyFA-Jittor
v0.1.2, with the two options the reference's blocks leave out)."""

import torch

from .. import _native
from .vocab import _recorded, _torch_backward


def residual_norm(x, y, weight, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """(s, h) of the residual ``x`` and a block's output ``y`` [..., D]:

        b = y [* rsqrt(mean(y^2) + eps) * post_weight] [* sigmoid(gate)]
        s = x + scale * b
        h = s * rsqrt(mean(s^2) + eps) * weight

    s is the next residual, h the next block's input. x, y and gate share one
    shape and dtype (bf16, fp16 or fp32), the weights are [D], D at most 8192.
    All in fp32, s and h rounded once (h is that of s before its rounding).
    Differentiable in every tensor; a backward pass that is itself recorded runs
    in torch operations."""
    if x.dtype not in _native.LM_DTYPES:
        raise NotImplementedError(f"residual_norm: x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"residual_norm: x must be [..., width], got {tuple(x.shape)}")
    D = x.shape[-1]
    if D > _native.RESIDUAL_MAX_D:
        raise NotImplementedError(f"residual_norm: at most {_native.RESIDUAL_MAX_D} columns, got {D}")
    for name, t in (("y", y), ("gate", gate)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"residual_norm: {name} must be {tuple(x.shape)} {x.dtype}, got {tuple(t.shape)} {t.dtype}")
    for name, t in (("weight", weight), ("post_weight", post_weight)):
        if t is not None and (tuple(t.shape) != (D,) or not t.dtype.is_floating_point):
            raise ValueError(f"residual_norm: {name} must be a float tensor of shape ({D},), got {tuple(t.shape)} {t.dtype}")
    if isinstance(scale, torch.Tensor):
        raise ValueError("residual_norm: the scale must be a number (a tensor's gradient would be lost)")
    given = (x.contiguous(), y.contiguous(), weight.float().contiguous(),
             None if post_weight is None else post_weight.float().contiguous(),
             None if gate is None else gate.contiguous())
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given):
        return _ResidualNorm.apply(*given, float(scale), float(eps))
    return _native.residual_norm(*given, float(scale), float(eps))[:2]


def _plain(x, y, weight, post, gate, scale, eps):
    """residual_norm in torch operations."""
    b = y.float()
    if post is not None:
        b = b * torch.rsqrt(b.pow(2).mean(-1, keepdim=True) + eps) * post
    if gate is not None:
        b = b * torch.sigmoid(gate.float())
    s = x.float() + scale * b
    return s.to(x.dtype), (s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + eps) * weight).to(x.dtype)


class _ResidualNorm(torch.autograd.Function):
    """residual_norm with its gradients; keeps the inputs and the two
    reciprocal roots of each row."""

    @staticmethod
    def forward(ctx, x, y, weight, post, gate, scale, eps):
        s, h, stats = _native.residual_norm(x, y, weight, post, gate, scale, eps, stats=True)
        ctx.save_for_backward(x, y, weight, post, gate, stats)
        ctx.args = (scale, eps)
        ctx.set_materialize_grads(False)
        return s, h

    @staticmethod
    def backward(ctx, d_s, d_h):
        *inputs, stats = ctx.saved_tensors
        needed = ctx.needs_input_grad[:5]
        if _recorded(d_s, d_h):
            return _torch_backward(lambda *a: _plain(*a, *ctx.args), inputs, needed, (d_s, d_h)) + (None, None)
        d_s, d_h = (None if t is None else t.contiguous() for t in (d_s, d_h))
        return _native.residual_norm_grad(*inputs, *ctx.args, stats, d_s, d_h, needed) + (None, None)
