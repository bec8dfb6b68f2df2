"""From a causal language model's logits to its next tokens on the gfx950 HIP
path: penalties for repeated tokens, biases and grammar masks, and the choice
of a token by temperature, top-k, top-p and min-p. (The reference chooses on the
host, from the logits as they are: generation.py:23-62 of Chyxx/CyFA-Jittor
v0.1.2.)

Options are numbers, the same for every row, or tensors with a value for each. A
call that torch has to see (torch.func transforms, forward-mode derivatives,
tracing, compiling, dispatch modes, subclasses of tensors) runs in torch
operations."""

from typing import NamedTuple

import torch

from .. import _native
from .._autograd import kernel_ok, through_torch


class SampledTokens(NamedTuple):
    """sample_tokens' results."""

    ids: torch.Tensor
    logprob: torch.Tensor


def _check_logits(what, logits):
    if logits.dtype not in _native.LM_DTYPES:
        raise NotImplementedError(f"{what}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits must be [..., vocabulary], got {tuple(logits.shape)}")
    if logits.shape[-1] > _native.LOGPROBS_MAX_V:
        raise NotImplementedError(f"{what}: at most {_native.LOGPROBS_MAX_V} columns, got {logits.shape[-1]}")


def _constant(what, name, t):
    if not t.requires_grad:
        return t
    if torch.is_grad_enabled():
        raise NotImplementedError(f"{what}: {name} gets no gradient here; give it detached")
    return t.detach()


def _expanded(what, name, t, shape):
    """t broadcast to shape, not copied."""
    if t.shape == shape:
        return t
    try:
        return t.expand(shape)
    except RuntimeError:
        raise ValueError(f"{what}: {name} must broadcast to {tuple(shape)}, got {tuple(t.shape)}") from None


def _per_row(what, name, v, lead, dtype=torch.float32):
    """An option: a number, or a contiguous tensor of dtype for the rows ``lead``."""
    if not isinstance(v, torch.Tensor):
        return float(v) if dtype is torch.float32 else int(v)
    if v.dtype is dtype and v.shape == lead and not v.requires_grad and v.is_contiguous():
        return v
    if dtype is torch.float32 and not v.dtype.is_floating_point or dtype is torch.int64 and v.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: {name} must be {'a float' if dtype is torch.float32 else 'an int64 or int32'} tensor, got {v.dtype}")
    v = _constant(what, name, v)
    if v.dtype is not dtype:
        v = v.to(dtype)
    return _expanded(what, name, v, lead).contiguous()


def _integers(what, name, t, lead):
    if t.dtype is torch.int64 and t.shape == lead and t.is_contiguous():
        return t
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: {name} must be int64 or int32, got {t.dtype}")
    if t.dtype is torch.int32:
        t = t.long()
    return _expanded(what, name, t, lead).contiguous()


def _float32(what, name, t):
    if not t.dtype.is_floating_point:
        raise ValueError(f"{what}: {name} must be a float tensor, got {t.dtype}")
    t = _constant(what, name, t)
    return t if t.dtype is torch.float32 else t.float()


def _share(a, b):
    """Whether the memory between a's first and last element meets b's."""
    if not isinstance(b, torch.Tensor) or not a.numel() or not b.numel() or a.device != b.device:
        return False
    first, end = zip(*((t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size())
                       for t in (a, b)))
    return max(first) < min(end)


def adjust_logits(logits, history=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0,
                  bias=None, token_bias=None, allowed=None, out=None):
    """``logits`` [..., V] with penalties for the tokens a sequence holds already,
    biases and a mask, in fp32 and rounded once to the logits' dtype:

        y = x / repetition (x repetition below zero)     tokens of the history
        y -= frequency count + presence                  those behind the prompt, count their number
        y += bias + token_bias
        y = -inf                                         tokens that are not allowed

    ``history`` [..., L], int64 or int32: each row's tokens so far, its first
    ``lengths`` [...] of them (all without; clamped to [0, L]), of which the first
    ``prompt_lengths`` [...] (none without) are the prompt's. Tokens outside
    [0, V) are passed over. ``repetition``, ``presence``, ``frequency``: numbers or
    float tensors [...]. ``bias``: float [..., V]. ``token_bias``: (ids [..., n],
    values [..., n]), n at most 1024; the values of equal ids are added up, in
    their order, before the logit, ids outside [0, V) are passed over.
    ``allowed``: bool [..., V], or int32 [..., ceil(V / 32)] with token j at bit
    j % 32 of word j // 32. Each of them may have any shape that broadcasts to the
    logits' leading one, and is read in place where it does.
    ``out``: a tensor of the logits' shape and dtype, or the logits themselves
    (with a bias or a mask an element at a time, up to three times as slow).

    Differentiable in the logits (not with ``out``): a row without allowed tokens is
    all -inf and gets a gradient of zeros, as every token that is not allowed."""
    what = "adjust_logits"
    _check_logits(what, logits)
    lead, V = logits.shape[:-1], logits.shape[-1]
    if history is None:
        if lengths is not None or prompt_lengths is not None:
            raise ValueError(f"{what}: lengths are those of a history")
    else:
        if history.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"{what}: history must be int64 or int32, got {history.dtype}")
        if history.dim() == 0:
            raise ValueError(f"{what}: history must be [..., length], got a scalar")
        history = _expanded(what, "history", history, lead + history.shape[-1:])
        if lengths is not None:
            lengths = _integers(what, "lengths", lengths, lead)
        if prompt_lengths is not None:
            prompt_lengths = _integers(what, "prompt_lengths", prompt_lengths, lead)
    repetition = _per_row(what, "repetition", repetition, lead)
    presence = _per_row(what, "presence", presence, lead)
    frequency = _per_row(what, "frequency", frequency, lead)
    if not isinstance(repetition, torch.Tensor) and not repetition > 0:
        raise ValueError(f"{what}: repetition must be positive, got {repetition}")
    if bias is not None:
        bias = _expanded(what, "bias", _float32(what, "bias", bias), logits.shape)
    if token_bias is not None:
        ids, values = token_bias
        if ids.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"{what}: token_bias' ids must be int64 or int32, got {ids.dtype}")
        if ids.dim() == 0 or values.dim() == 0 or ids.shape[-1] != values.shape[-1]:
            raise ValueError(f"{what}: token_bias must be ids [..., n] and values [..., n], got {tuple(ids.shape)} {tuple(values.shape)}")
        n = ids.shape[-1]
        if n > _native.ADJUST_MAX_TOKENS:
            raise NotImplementedError(f"{what}: at most {_native.ADJUST_MAX_TOKENS} token biases, got {n}")
        token_bias = (_expanded(what, "token_bias' ids", ids.long(), lead + (n,)),
                      _expanded(what, "token_bias' values", _float32(what, "token_bias' values", values), lead + (n,)))
    if allowed is not None:
        if allowed.dtype not in (torch.bool, torch.int32):
            raise ValueError(f"{what}: allowed must be bool, or int32 words of bits, got {allowed.dtype}")
        columns = V if allowed.dtype is torch.bool else (V + 31) // 32
        if allowed.dim() == 0 or allowed.shape[-1] != columns:
            raise ValueError(f"{what}: allowed must be [..., {columns}] in {allowed.dtype}, got {tuple(allowed.shape)}")
        allowed = _expanded(what, "allowed", allowed, lead + (columns,))
    penalties = (repetition, presence, frequency)
    args = (history, lengths, prompt_lengths, penalties, bias, token_bias, allowed)
    recorded = torch.is_grad_enabled() and logits.requires_grad
    if out is not None:
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
            raise ValueError(f"{what}: out must be {tuple(logits.shape)} {logits.dtype} on {logits.device}, got {tuple(out.shape)} "
                             f"{out.dtype} on {out.device}")
        if recorded or (torch.is_grad_enabled() and out.requires_grad):
            raise NotImplementedError(f"{what}: a call that is recorded for autograd has no out")
        if out.shape[-1] > 1 and out.stride(-1) != 1 or out.dim() > 3:
            raise ValueError(f"{what}: out needs contiguous rows and at most three dimensions")
        if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise ValueError(f"{what}: out has to be one element of memory for each of its own")
        if _share(out, logits) and (out.data_ptr(), out.stride()) != (logits.data_ptr(), logits.stride()):
            raise ValueError(f"{what}: out has to be the logits themselves or apart from them")
        if any(_share(out, t) for t in (*args[:3], *penalties, bias, *(token_bias or ()), allowed)):
            raise ValueError(f"{what}: out has to be apart from what is read with the logits")
    tensors = [t for t in (logits, out, history, lengths, prompt_lengths, bias, allowed, *(token_bias or ()), *penalties)
               if isinstance(t, torch.Tensor)]
    _native.require_device(*tensors)
    if not kernel_ok(*tensors):
        y = _plain_adjust(logits, *args)
        return y if out is None else out.copy_(y)
    if recorded:
        return _AdjustLogits.apply(logits, args)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif not out.is_inference():
        torch.autograd.graph.increment_version(out)  # (a graph that kept it finds it edited)
    if logits.numel():
        _native.adjust(logits, out, *args)
    return out


def _tables(logits, history, lengths, prompts, allowed):
    """(occurrences or None, those behind the prompt or None, mask or None) [..., V]."""
    V = logits.shape[-1]
    n = m = None
    if history is not None and history.shape[-1]:
        at = torch.arange(history.shape[-1], device=logits.device)
        inside = (history >= 0) & (history < V)
        if lengths is not None:
            inside = inside & (at < lengths[..., None])
        ids = history.long().clamp(0, V - 1)
        zero = torch.zeros(logits.shape, dtype=torch.int32, device=logits.device)
        n = zero.scatter_add(-1, ids, inside.int())
        m = n if prompts is None else zero.scatter_add(-1, ids, (inside & (at >= prompts[..., None])).int())
    if allowed is not None and allowed.dtype is torch.int32:
        bits = (allowed[..., None] >> torch.arange(32, device=allowed.device, dtype=torch.int32)) & 1
        allowed = bits.flatten(-2)[..., :V] != 0
    return n, m, allowed


def _column(v):
    return v[..., None] if isinstance(v, torch.Tensor) else v


def _plain_adjust(logits, history, lengths, prompts, penalties, bias, tokens, allowed):
    """adjust_logits in torch operations."""
    repetition, presence, frequency = (_column(v) for v in penalties)
    if not isinstance(repetition, torch.Tensor):  # (torch divides by a number by a product with its reciprocal)
        repetition = torch.full((), repetition, dtype=torch.float32, device=logits.device)
    n, m, allowed = _tables(logits, history, lengths, prompts, allowed)
    y = logits.float()
    if n is not None:
        y = torch.where(n > 0, torch.where(y > 0, y / repetition, y * repetition), y)
        y = torch.where(m > 0, y - (m * frequency + presence), y)
    if bias is not None:
        y = y + bias
    if tokens is not None:
        ids, values = tokens
        inside, at = (ids >= 0) & (ids < logits.shape[-1]), ids.clamp(0, logits.shape[-1] - 1)
        named = torch.zeros(y.shape, dtype=torch.int32, device=y.device).scatter_add(-1, at, inside.int()) > 0
        sums = torch.zeros(y.shape, dtype=y.dtype, device=y.device).scatter_add(-1, at, torch.where(inside, values, 0.0))
        y = torch.where(named, y + sums, y)
    if allowed is not None:
        y = torch.where(allowed, y, float("-inf"))
    return y.to(logits.dtype)


class _AdjustLogits(torch.autograd.Function):
    """adjust_logits with its gradient; linear in the cotangent but for the
    logits' signs."""

    @staticmethod
    def forward(ctx, logits, args):
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if logits.numel():
            _native.adjust(logits, out, *args)
        history, lengths, prompts, penalties, _, _, allowed = args
        repetition = penalties[0] if isinstance(penalties[0], torch.Tensor) else None
        ctx.save_for_backward(logits, history, lengths, prompts, repetition, allowed)
        ctx.repetition = penalties[0] if repetition is None else None
        return out

    @staticmethod
    def backward(ctx, dy):
        logits, history, lengths, prompts, repetition, allowed = ctx.saved_tensors
        if repetition is None:
            repetition = ctx.repetition
        if through_torch(dy):
            n, _, allowed = _tables(logits.detach(), history, lengths, prompts, allowed)
            dx = dy.float()
            if n is not None:
                r = torch.as_tensor(_column(repetition), dtype=torch.float32, device=logits.device)
                dx = torch.where(n > 0, dx * torch.where(logits.detach() > 0, 1 / r, r), dx)
            if allowed is not None:
                dx = torch.where(allowed, dx, 0.0)
            return dx.to(logits.dtype), None
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if logits.numel():
            _native.adjust(logits, dx, history, lengths, prompts, (repetition, 0.0, 0.0), None, None, allowed, dy.contiguous())
        return dx, None


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A token for each row of ``logits`` [..., V], drawn with the numbers
    ``uniform`` [...] (fp32 or fp64, in [0, 1)): SampledTokens(ids [...] int64,
    logprob [...] fp32), logprob under the distribution that the token was drawn
    from.

    With weights w = exp((x - max) / temperature), in the order of falling logits,
    the lower id first among equals, kept are the first ``top_k`` tokens (0: all),
    of those the ones before which less than ``top_p`` of their mass lies (the
    first always), of those the ones with w >= ``min_p``. The token is the first
    kept one, by id, at which the running mass of the kept passes uniform times
    their mass, so that equal inputs give equal tokens: weights are held as
    multiples of 2^-46 of the largest (past 2^16 columns of 2^(ceil(log2 V) - 62))
    and added up exactly.

    Each option is a number or a tensor [...] (top_k int64 or int32, the others
    float, read in fp32). Temperature 0, or below in a tensor: the first largest
    logit, logprob 0. A min_p above 1 in a tensor counts as 1. A row that holds
    a NaN or +inf, or nothing but -inf, has no probabilities: its first largest
    logit (a NaN before all others), logprob NaN.
    A choice has no gradient: logits that require one are read as they are."""
    what = "sample_tokens"
    _check_logits(what, logits)
    lead, V = logits.shape[:-1], logits.shape[-1]
    if uniform.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"{what}: uniform must be fp32 or fp64, got {uniform.dtype}")
    if uniform.shape != lead:
        raise ValueError(f"{what}: uniform must have shape {tuple(lead)}, got {tuple(uniform.shape)}")
    temperature = _per_row(what, "temperature", temperature, lead)
    top_k = _per_row(what, "top_k", top_k, lead, torch.int64)
    top_p = _per_row(what, "top_p", top_p, lead)
    min_p = _per_row(what, "min_p", min_p, lead)
    if not isinstance(temperature, torch.Tensor) and not temperature >= 0:
        raise ValueError(f"{what}: temperature must not be negative, got {temperature}")
    if not isinstance(top_k, torch.Tensor) and top_k < 0:
        raise ValueError(f"{what}: top_k must not be negative, got {top_k}")
    if not isinstance(top_p, torch.Tensor) and not 0 < top_p <= 1:
        raise ValueError(f"{what}: top_p must be in (0, 1], got {top_p}")
    if not isinstance(min_p, torch.Tensor) and not 0 <= min_p <= 1:
        raise ValueError(f"{what}: min_p must be in [0, 1], got {min_p}")
    tensors = [t for t in (logits, uniform, temperature, top_k, top_p, min_p) if isinstance(t, torch.Tensor)]
    _native.require_device(*tensors)
    if not kernel_ok(*tensors):
        return _plain_sample(logits.detach(), uniform.detach(), temperature, top_k, top_p, min_p)
    return SampledTokens(*_native.sample(logits, uniform.contiguous(), temperature, top_k, top_p, min_p))


def _plain_sample(logits, uniform, temperature, top_k, top_p, min_p):
    """sample_tokens in torch operations."""
    V = logits.shape[-1]
    x = logits.double()

    def column(v, dtype=torch.float64):
        return torch.as_tensor(_column(v), dtype=dtype, device=x.device)

    T, k, p = column(temperature), column(top_k, torch.int64), column(top_p)
    nan = x.isnan()
    top = x.masked_fill(nan, float("inf")).amax(-1, keepdim=True)
    none = nan.any(-1, keepdim=True) | ~top.isfinite()
    greedy = none | ~(T > 0)
    first = torch.where(nan.any(-1, keepdim=True), nan, x == top).int().argmax(-1)
    x = torch.where(none, 0.0, x)
    top = torch.where(none, 0.0, top)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, T))).masked_fill(x == float("-inf"), 0.0)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(-1, order)
    rank = torch.arange(V, device=x.device)
    mass_of = torch.where((k <= 0) | (rank < k), sorted_w, 0.0)
    before = mass_of.cumsum(-1) - mass_of
    keep = (mass_of > 0) & ((rank == 0) | ~(p < 1) | (before < p * mass_of.sum(-1, keepdim=True)))
    keep = keep & ((rank == 0) | ~(sorted_w < column(min_p).clamp(max=1.0)))
    kept = w * torch.zeros_like(w).scatter(-1, order, keep.to(w.dtype))
    mass = kept.cumsum(-1)
    total = mass[..., -1:]
    passed = (mass <= uniform.double().nan_to_num(0.0).clamp(0, 1 - 2.0**-53)[..., None] * total).sum(-1)
    last = torch.where(kept > 0, rank, 0).amax(-1)
    ids = torch.minimum(passed, last)
    logprob = (kept.gather(-1, ids[..., None]) / total).log()[..., 0]
    logprob = torch.where(greedy[..., 0], torch.where(none[..., 0], float("nan"), 0.0), logprob)
    return SampledTokens(torch.where(greedy[..., 0], first, ids), logprob.float())
