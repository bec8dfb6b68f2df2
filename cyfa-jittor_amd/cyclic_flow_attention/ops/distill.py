"""The training loss of a student against a teacher's most probable tokens on
the gfx950 HIP path, beside the loss against labels in ops.vocab (the reference
trains on labels alone: models/cyfa/modeling_cyfa.py:96-108 of
Chyxx/CyFA-Jittor v0.1.2)."""

import torch

from .. import _native
from .._autograd import kernel_ok, through_torch, torch_grads


def distill_loss(logits, top_ids, top_logprobs, temperature=1.0, tail=False, weights=None):
    """The mean divergence sum p (log p - log q) of q = softmax(``logits`` [..., V]
    / temperature) from a teacher's distribution p known at ``top_ids`` [..., k]
    (int64 or int32, k at most 256), an fp32 scalar.

    p is the softmax of ``top_logprobs`` [..., k] / temperature over a row's tokens
    (the teacher's logits serve as well as its log probabilities). With ``tail``
    p is exp(top_logprobs) itself and the rest of either distribution, the mass of
    all other tokens, one more outcome (temperature 1; V at most 2^19; nothing
    where the student's other logits are all -inf). Entries with an id outside
    [0, V) or a log probability of -inf are left out.

    The sum is over the entries, each with its own p and the q of its id, not over
    the tokens. Teachers as score(top_k) gives them name a token once, and the two
    are the same. Of a token that a row names several times, with p_1, p_2, ...
    that add up to P, the gradient is that of one entry of P, and the loss is less
    than the divergence by the constant sum p_i log(P / p_i): it may be negative.

    ``weights`` [...], float: each row's in the mean, 1 without. A row without
    entries or with weight 0 does not count, gets a gradient of zeros and is not
    read; no row that counts: NaN. A row of nothing but -inf, or with NaN or +inf,
    has no probabilities: NaN. Differentiable in the logits. (The loss is not
    multiplied by temperature^2.) A backward pass that is itself recorded, and a
    call that torch has to see (torch.func transforms, forward-mode derivatives,
    tracing, compiling, dispatch modes, subclasses of tensors), run in torch
    operations."""
    what = "distill_loss"
    if logits.dtype not in _native.LM_DTYPES:
        raise NotImplementedError(f"{what}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits must be [..., vocabulary], got {tuple(logits.shape)}")
    lead, V = logits.shape[:-1], logits.shape[-1]
    if top_ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: top_ids must be int64 or int32, got {top_ids.dtype}")
    if top_ids.dim() != logits.dim() or top_ids.shape[:-1] != lead or top_ids.shape[-1] == 0:
        raise ValueError(f"{what}: top_ids must be {tuple(lead)} + (k,), got {tuple(top_ids.shape)}")
    if top_logprobs.shape != top_ids.shape or not top_logprobs.dtype.is_floating_point:
        raise ValueError(f"{what}: top_logprobs must be a float tensor of shape {tuple(top_ids.shape)}, got "
                         f"{tuple(top_logprobs.shape)} {top_logprobs.dtype}")
    if top_ids.shape[-1] > _native.DISTILL_MAX_K:
        raise NotImplementedError(f"{what}: at most {_native.DISTILL_MAX_K} tokens, got {top_ids.shape[-1]}")
    if weights is not None and (weights.shape != lead or not weights.dtype.is_floating_point):
        raise ValueError(f"{what}: weights must be a float tensor of shape {tuple(lead)}, got {tuple(weights.shape)} {weights.dtype}")
    if isinstance(temperature, torch.Tensor):
        raise ValueError(f"{what}: the temperature must be a number (a tensor's gradient would be lost)")
    temperature, tail = float(temperature), bool(tail)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"{what}: temperature must be positive, got {temperature}")
    if tail and temperature != 1.0:
        raise ValueError(f"{what}: with the tail the temperature is 1, got {temperature}")
    if V > (_native.DISTILL_MAX_TAIL_V if tail else _native.LOGPROBS_MAX_V):
        raise NotImplementedError(f"{what}: at most {_native.DISTILL_MAX_TAIL_V if tail else _native.LOGPROBS_MAX_V} columns, got {V}")
    for name, t in (("top_logprobs", top_logprobs), ("weights", weights)):
        if t is not None and torch.is_grad_enabled() and t.requires_grad:
            raise NotImplementedError(f"{what}: {name} gets no gradient here; give it detached")
    ids = top_ids.contiguous() if top_ids.dtype is torch.int64 else top_ids.long().contiguous()
    values = _float32(top_logprobs)
    if weights is not None:
        weights = _float32(weights)
    _native.require_device(logits, ids, values, weights)
    if not kernel_ok(logits, ids, values, weights):
        return _plain(logits, ids, values, weights, temperature, tail)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillLoss.apply(logits, ids, values, weights, temperature, tail)
    return _native.distill_loss(logits, ids, values, weights, temperature, tail)[0]


def _float32(t):
    if t.requires_grad:
        t = t.detach()
    return (t if t.dtype is torch.float32 else t.float()).contiguous()


def _plain(logits, ids, values, weights, temperature, tail):
    """distill_loss in torch operations; rows that do not count are not read."""
    V = logits.shape[-1]
    valid = (ids >= 0) & (ids < V) & (values != float("-inf"))
    count = valid.any(-1).float() if weights is None else valid.any(-1) * weights
    live = count != 0
    x = torch.where(live[..., None], logits.float(), 0.0)
    at = ids.clamp(0, V - 1)
    x = x - x.detach().amax(-1, keepdim=True)  # (before the temperature, which may take the lowest values past fp32)
    x_at = x.gather(-1, at).double() / temperature
    x = x / temperature
    lse = x.exp().sum(-1, keepdim=True).log()
    t = torch.where(valid, values.double(), 0.0)
    if tail:
        log_p = t
    else:
        t = t.masked_fill(~valid, float("-inf"))
        t = (t - torch.where(live[..., None], t.amax(-1, keepdim=True), 0.0)) / temperature
        log_p = t - t.masked_fill(~live[..., None], 0.0).logsumexp(-1, keepdim=True)
    p = torch.where(valid & live[..., None], log_p.exp(), 0.0)
    given = p > 0
    log_p = torch.where(given, log_p, 0.0)
    log_q = torch.where(given, x_at - lse, 0.0)
    loss = (p * (log_p - log_q)).sum(-1)
    if tail:
        entry = torch.zeros(logits.shape, dtype=torch.int32, device=logits.device).scatter_add(-1, at, valid.int()) > 0
        others = x.masked_fill(entry, float("-inf"))
        most = others.detach().amax(-1)
        some = most > float("-inf")
        most = torch.where(some, most, 0.0)
        others = torch.where(some[..., None] | ~entry, others - most[..., None], 0.0)
        sums = torch.where(some, others.exp().sum(-1), 1.0)
        rest = torch.where(some & live, (1 - p.sum(-1)).clamp(min=0), 0.0)
        loss = loss + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - (sums.log() + most - lse[..., 0])), 0.0)
    return (torch.where(live, loss * count, 0.0).sum() / count.double().sum()).float()


class _DistillLoss(torch.autograd.Function):
    """distill_loss with its gradient: keeps the logits and ten numbers a row."""

    @staticmethod
    def forward(ctx, logits, ids, values, weights, temperature, tail):
        loss, kept = _native.distill_loss(logits, ids, values, weights, temperature, tail)
        ctx.save_for_backward(logits, ids, values, weights, kept)
        ctx.args = (temperature, tail)
        return loss

    @staticmethod
    def backward(ctx, d_loss):
        logits, ids, values, weights, kept = ctx.saved_tensors
        if through_torch(d_loss):
            return torch_grads(lambda x: _plain(x, ids, values, weights, *ctx.args), (logits,), (True,), (d_loss,)) + (None,) * 5
        return (_native.distill_loss_grad(logits, ids, values, weights, *ctx.args, kept, d_loss.contiguous()),) + (None,) * 5
