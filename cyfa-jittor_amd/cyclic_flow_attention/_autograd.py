"""What the autograd functions of the layers and of the operators share: which
calls and which backward passes run in torch operations, and how."""

import torch
from torch.autograd import forward_ad

# (looked up once: a small call's time is the host's)
_peek = torch._C._functorch.peek_interpreter_stack
_is_batched = torch._C._functorch.is_legacy_batchedtensor
_compiling, _tracing, _modes = torch.compiler.is_compiling, torch._C._is_tracing, torch._C._len_torch_dispatch_stack
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))


def kernel_ok(*tensors):
    """Whether a call with these tensors (or Nones) may go to a kernel, of which
    torch sees nothing: plain tensors, and no torch.func transform, forward-mode
    derivative, tracing, compiling or dispatch mode (make_fx, operation
    counters), each of which would lose what the kernel computes."""
    if _compiling() or _peek() is not None or forward_ad._current_level >= 0 or _tracing() or _modes():
        return False
    for t in tensors:
        if type(t) not in _PLAIN:
            return False
    return True


def batched(*cotangents):
    """Whether this backward pass runs over several cotangents at once (vmap). A
    cotangent may be None."""
    if _peek() is not None:
        return True
    for t in cotangents:
        if t is not None and _is_batched(t):
            return True
    return False


def through_torch(*cotangents):
    """Whether a backward pass has to run in torch operations: one that is
    itself recorded (``create_graph=True``), or batched."""
    return torch.is_grad_enabled() or batched(*cotangents)


def torch_grads(fn, inputs, needed, cotangents):
    """Gradients of fn(*inputs) (a tensor or a tuple of them) by autograd, None
    where ``needed`` is false and zeros where no given cotangent reaches an
    input, as the adjoint kernels give them; recorded when this backward pass is.

    fn is differentiated at aliases of the inputs: one input may have been
    computed from another (a block's output from the residual it joins) or be
    the same tensor, and a gradient of the inputs themselves would follow, and
    free, the caller's graph between them."""
    recorded = torch.is_grad_enabled()
    with torch.enable_grad():
        aliases = [t.view_as(t) if n else t for t, n in zip(inputs, needed)]
        outs = fn(*aliases)
        pairs = [(o, c) for o, c in zip(outs if isinstance(outs, tuple) else (outs,), cotangents)
                 if c is not None and o.requires_grad]
        wanted = [t for t, n in zip(aliases, needed) if n]
        grads = [None] * len(wanted)
        if pairs and wanted:
            outs, cots = zip(*pairs)
            grads = torch.autograd.grad(outs, wanted, cots, create_graph=recorded, allow_unused=True)
        grads = iter([torch.zeros_like(t) if g is None else g for t, g in zip(wanted, grads)])
    return tuple(next(grads) if n else None for n in needed)
