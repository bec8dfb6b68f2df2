"""The vocabulary's two ends of a causal language model on the gfx950 HIP path:
the scaled embedding lookup, and log probabilities of tokens with their mean as
the training loss (the reference's nn.Embedding and cross_entropy_loss,
models/cyfa/modeling_cyfa.py:63-71, 96-108 of Chyxx/CyFA-Jittor v0.1.2).

Each computes in fp32 whatever the dtype (bf16, fp16 or fp32) and rounds its
results once. Where an input requires a gradient the call is recorded for
autograd and its backward runs as HIP kernels too; a backward pass that is
itself recorded (``create_graph=True``) runs in torch operations, and so does a
call that torch has to see (torch.func transforms, forward-mode derivatives,
tracing, compiling, dispatch modes, subclasses of tensors).
"""

from typing import NamedTuple

import torch
import torch.nn.functional as F

from .. import _native
from .._autograd import batched, kernel_ok, through_torch, torch_grads


class TokenLogprobs(NamedTuple):
    """token_logprobs' results; the last two are None without alternatives."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None
    top_ids: torch.Tensor | None


def _check_logits(what, logits, tokens, name):
    if logits.dtype not in _native.LM_DTYPES:
        raise NotImplementedError(f"{what}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits must be [..., vocabulary], got {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: {name} must have shape {tuple(logits.shape[:-1])}, got {tuple(tokens.shape)}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: {name} must be int64 or int32, got {tokens.dtype}")
    return _int64(tokens)


def _int64(t):
    return t.contiguous() if t.dtype is torch.int64 else t.to(torch.int64).contiguous()


def token_logprobs(logits, tokens, top_k=0, ignore_index=-100):
    """Log probabilities of ``tokens`` [...] under softmax(``logits`` [..., V]),
    the entropy of each row, and its ``top_k`` (at most 32) most probable tokens.

    Returns TokenLogprobs(logprob [...], entropy [...], top_logprobs
    [..., top_k], top_ids [..., top_k]), fp32 and int64; the alternatives in
    falling order, the lower id first among equal logits. The logits may be
    strided (a slice of the time axis is read in place). A token equal to
    ``ignore_index`` has logprob 0 and gives no gradient through it; one outside
    [0, V) otherwise has logprob NaN. Logits of -inf have probability 0 and add
    nothing to the entropy; a row of nothing else has no probabilities, and its
    results are NaN, as those of a row that holds a NaN or +inf.

    Differentiable in the logits through logprob, entropy and top_logprobs; a
    row whose cotangents are all zero gets a gradient of zeros, whatever it holds.
    """
    tokens = _check_logits("token_logprobs", logits, tokens, "tokens")
    top_k = int(top_k)
    if not 0 <= top_k <= logits.shape[-1]:
        raise ValueError(f"token_logprobs: top_k must be in [0, {logits.shape[-1]}], got {top_k}")
    if top_k > _native.LOGPROBS_MAX_TOP:
        raise NotImplementedError(f"token_logprobs: at most {_native.LOGPROBS_MAX_TOP} alternatives, got {top_k}")
    if not kernel_ok(logits, tokens):
        _native.require_device(logits, tokens)
        ids = logits.detach().sort(dim=-1, descending=True, stable=True).indices[..., :top_k] if top_k else None
        return TokenLogprobs(*_plain_logprobs(logits, tokens, ids, int(ignore_index)), *(() if top_k else (None,)), ids)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top_k, int(ignore_index)))
    return TokenLogprobs(*_native.logprobs(logits, tokens, top_k, int(ignore_index))[:4])


def _plain_logprobs(logits, tokens, ids, ignore_index):
    """(logprob, entropy, top_logprobs) in torch operations."""
    lp = F.log_softmax(logits.float(), -1)
    V = logits.shape[-1]
    logprob = lp.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0]
    ignored = tokens == ignore_index
    logprob = logprob * torch.where(ignored | ((tokens >= 0) & (tokens < V)), 1.0, float("nan"))
    logprob = logprob.masked_fill(ignored, 0.0)
    p = lp.exp()
    entropy = -(p * lp.masked_fill(p == 0, 0.0)).sum(-1)
    return (logprob, entropy) if ids is None else (logprob, entropy, lp.gather(-1, ids))


def _live_rows(logits, tokens, ignore_index, d_logprob, d_entropy, d_top):
    """[..., 1]: rows that have probabilities or that a cotangent other than
    zero reaches; the others get a gradient of zeros, whatever they hold."""
    live = logits.detach().float().logsumexp(-1).isfinite()
    if d_logprob is not None:
        live = live | ((d_logprob != 0) & (tokens != ignore_index))
    if d_entropy is not None:
        live = live | (d_entropy != 0)
    if d_top is not None:
        live = live | (d_top != 0).any(-1)
    return live[..., None]


class _TokenLogprobs(torch.autograd.Function):
    """token_logprobs with its gradient: keeps the logits and, of each row, the
    maximum, the log of the sum and the entropy."""

    @staticmethod
    def forward(ctx, logits, tokens, top_k, ignore_index):
        logprob, entropy, top, ids, stats = _native.logprobs(logits, tokens, top_k, ignore_index, stats=True)
        ctx.save_for_backward(logits, tokens, stats, entropy, ids)
        ctx.args = (top_k, ignore_index)
        ctx.set_materialize_grads(False)
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        return logprob, entropy, top, ids

    @staticmethod
    def backward(ctx, d_logprob, d_entropy, d_top, _):
        logits, tokens, stats, entropy, ids = ctx.saved_tensors
        top_k, ignore_index = ctx.args
        cots = (d_logprob, d_entropy, d_top)
        if through_torch(*cots):
            live = _live_rows(logits, tokens, ignore_index, *cots)

            def plain(x):
                return _plain_logprobs(x, tokens, ids, ignore_index)

            if batched(*cots):
                (dx,) = torch_grads(plain, (logits,), (True,), cots)
                dx = torch.where(live, dx, 0.0)
            else:  # (other rows stay out of the higher derivatives too)
                (dx,) = torch_grads(lambda x: plain(torch.where(live, x, 0.0)), (logits,), (True,), cots)
            return dx, None, None, None
        cots = [None if c is None else c.contiguous() for c in cots]
        return _native.logprobs_grad(logits, tokens, top_k, ignore_index, stats, entropy, ids, *cots), None, None, None


def token_loss(logits, labels, ignore_index=-100):
    """The mean of -log softmax(``logits`` [..., V])[label] over the ``labels``
    [...] that are not ``ignore_index``, an fp32 scalar: F.cross_entropy of the
    logits in fp32, without forming them, and with NaN for a label outside
    [0, V). No label that counts: NaN, as F.cross_entropy. Differentiable in the
    logits; rows of ignored labels get zeros. The labels are those of the rows
    as they are (a causal model shifts them: label t is the token after t)."""
    labels = _check_logits("token_loss", logits, labels, "labels")
    if not kernel_ok(logits, labels):
        _native.require_device(logits, labels)
        return _plain_loss(logits, labels, int(ignore_index))[0]
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLoss.apply(logits, labels, int(ignore_index))
    return _native.token_loss(logits, labels, int(ignore_index))[0]


def _plain_loss(logits, labels, ignore_index):
    """token_loss in torch operations; rows of ignored labels are not read."""
    kept = labels != ignore_index
    logits = torch.where(kept[..., None], logits, 0.0)
    return (-_plain_logprobs(logits, labels, None, ignore_index)[0].sum() / kept.sum(),)


class _TokenLoss(torch.autograd.Function):
    """token_loss with its gradient."""

    @staticmethod
    def forward(ctx, logits, labels, ignore_index):
        loss, kept = _native.token_loss(logits, labels, ignore_index, stats=True)
        ctx.save_for_backward(logits, labels, kept)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    def backward(ctx, d_loss):
        logits, labels, kept = ctx.saved_tensors
        if through_torch(d_loss):
            return torch_grads(lambda x: _plain_loss(x, labels, ctx.ignore_index), (logits,), (True,), (d_loss,)) + (None, None)
        return _native.token_loss_grad(logits, labels, ctx.ignore_index, kept, d_loss.contiguous()), None, None


def embed_tokens(ids, weight, scale=1.0, padding_idx=None):
    """scale weight[ids]: rows of ``weight`` [V, D] for integer ``ids`` [...],
    [..., D] in the weight's dtype. An id outside [0, V) gives a row of NaN.

    The gradient of the weight is dense and adds each id's cotangents in fp32,
    in an association that the ids alone fix, and rounds once, so that two
    backward passes give the same bits; the row of ``padding_idx`` (negative: from the
    end) and ids outside [0, V) get none."""
    if weight.dtype not in _native.LM_DTYPES:
        raise NotImplementedError(f"embed_tokens: the weight must be bf16, fp16 or fp32, got {weight.dtype}")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"embed_tokens: the weight must be [vocabulary, width], got {tuple(weight.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"embed_tokens: ids must be int64 or int32, got {ids.dtype}")
    if isinstance(scale, torch.Tensor):
        raise ValueError("embed_tokens: the scale must be a number (a tensor's gradient would be lost)")
    V = weight.shape[0]
    if padding_idx is None:
        padding_idx = -1
    elif not -V <= padding_idx < V:
        raise ValueError(f"embed_tokens: padding_idx must be in [-{V}, {V}), got {padding_idx}")
    else:
        padding_idx = int(padding_idx) % V
    ids = _int64(ids)
    weight = weight.contiguous()
    if not kernel_ok(ids, weight):
        _native.require_device(ids, weight)
        return _plain_embed(ids, weight, float(scale), padding_idx)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _EmbedTokens.apply(ids, weight, float(scale), padding_idx)
    return _native.embed(ids, weight, float(scale))


def _plain_embed(ids, weight, scale, padding_idx):
    """embed_tokens in torch operations."""
    V = weight.shape[0]
    rows = weight.float()[ids.clamp(0, V - 1)]
    rows = torch.where((ids == padding_idx)[..., None], rows.detach(), rows) * scale
    return torch.where(((ids >= 0) & (ids < V))[..., None], rows, float("nan")).to(weight.dtype)


class _EmbedTokens(torch.autograd.Function):
    """embed_tokens with its gradient."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx)
        return _native.embed(ids, weight, scale)

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        V, scale, padding_idx = ctx.args
        if through_torch(dy):  # (linear in dy)
            kept = ((ids >= 0) & (ids < V) & (ids != padding_idx)).reshape(-1, 1)
            rows = torch.where(kept, dy.float().reshape(-1, dy.shape[-1]) * scale, 0.0)
            dw = rows.new_zeros(V, dy.shape[-1]).index_add(0, ids.reshape(-1).clamp(0, V - 1), rows)
            return None, dw.to(dy.dtype), None, None
        return None, _native.embed_grad(ids, V, dy.contiguous(), scale, padding_idx), None, None
