"""The join between two blocks of a model on the gfx950 HIP path: a block's
output norm and gate, the scaled residual add and the next block's norm
(CyFABlock.execute, models/cyfa/modeling_cyfa.py:48-51 of Chyxx/CyFA-Jittor
v0.1.2, with the two options the reference's blocks leave out)."""

import torch

from .. import _native
from .._autograd import kernel_ok, through_torch, torch_grads


def residual_norm(x, y, weight, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    """(s, h) of the residual ``x`` and a block's output ``y`` [..., D]:

        b = y [* rsqrt(mean(y^2) + eps) * post_weight] [* sigmoid(gate)]
        s = x + scale * b
        h = s * rsqrt(mean(s^2) + eps) * weight

    s is the next residual, h the next block's input. x, y and gate share one
    shape and dtype (bf16, fp16 or fp32), the weights are [D], D at most 8192.
    All in fp32, s and h rounded once (h is that of s before its rounding).
    Differentiable in every tensor; a backward pass that is itself recorded, and
    a call that torch has to see (torch.func transforms, forward-mode
    derivatives, tracing, compiling, dispatch modes, subclasses of tensors), run
    in torch operations."""
    shape, dtype = x.shape, x.dtype
    if dtype not in _native.LM_DTYPES:
        raise NotImplementedError(f"residual_norm: x must be bf16, fp16 or fp32, got {dtype}")
    if not shape or shape[-1] == 0:
        raise ValueError(f"residual_norm: x must be [..., width], got {tuple(shape)}")
    D = shape[-1]
    if D > _native.RESIDUAL_MAX_D:
        raise NotImplementedError(f"residual_norm: at most {_native.RESIDUAL_MAX_D} columns, got {D}")
    for name, t in (("y", y), ("gate", gate)):
        if t is not None and (t.shape != shape or t.dtype != dtype):
            raise ValueError(f"residual_norm: {name} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    for name, t in (("weight", weight), ("post_weight", post_weight)):
        if t is not None and (t.dim() != 1 or t.shape[0] != D or not t.dtype.is_floating_point):
            raise ValueError(f"residual_norm: {name} must be a float tensor of shape ({D},), got {tuple(t.shape)} {t.dtype}")
    if isinstance(scale, torch.Tensor):
        raise ValueError("residual_norm: the scale must be a number (a tensor's gradient would be lost)")
    scale, eps = float(scale), float(eps)
    x, y, weight = x.contiguous(), y.contiguous(), _fp32(weight)
    if post_weight is not None:
        post_weight = _fp32(post_weight)
    if gate is not None:
        gate = gate.contiguous()
    if not kernel_ok(x, y, weight, post_weight, gate):
        _native.require_device(x, y, weight, post_weight, gate)
        return _plain(x, y, weight, post_weight, gate, scale, eps)
    if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad or weight.requires_grad
                                    or (post_weight is not None and post_weight.requires_grad)
                                    or (gate is not None and gate.requires_grad)):
        return _ResidualNorm.apply(x, y, weight, post_weight, gate, scale, eps)
    return _native.residual_norm(x, y, weight, post_weight, gate, scale, eps)[:2]


def _fp32(t):
    return t.contiguous() if t.dtype is torch.float32 else t.float().contiguous()


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
        needed = ctx.needs_input_grad
        if through_torch(d_s, d_h):
            return torch_grads(lambda *a: _plain(*a, *ctx.args), inputs, needed[:5], (d_s, d_h)) + (None, None)
        if d_s is not None:
            d_s = d_s.contiguous()
        if d_h is not None:
            d_h = d_h.contiguous()
        return _native.residual_norm_grad(*inputs, *ctx.args, stats, d_s, d_h, needed) + (None, None)
