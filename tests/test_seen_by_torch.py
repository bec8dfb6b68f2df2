"""Calls of the operators around a model's blocks that torch has to see run in
torch operations: forward-mode derivatives, torch.func transforms, tracing,
compiling, dispatch modes and subclasses of tensors. No launch may happen."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from cyclic_flow_attention import _native, ops

INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    def launch(*args, **kwargs):
        raise AssertionError("a kernel was launched")

    monkeypatch.setattr(_native, "require_device", lambda *tensors: tensors[0].device)
    for name in ("logprobs", "logprobs_grad", "token_loss", "token_loss_grad", "embed", "embed_grad", "residual_norm",
                 "residual_norm_grad"):
        monkeypatch.setattr(_native, name, launch)


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


TOKENS = torch.tensor([3, -100, 0, 10, 7])
IDS = torch.tensor([[1, 4, 2], [4, 2, 0]])


def _logprobs(x):
    r = ops.token_logprobs(x, TOKENS, top_k=3)
    return r.logprob, r.entropy, r.top_logprobs


def _logprobs64(x):
    lp = torch.log_softmax(x, -1)
    at = lp.gather(1, TOKENS.clamp(min=0)[:, None])[:, 0]
    return torch.where(TOKENS < 0, 0.0, at), -(lp.exp() * lp).sum(-1), lp.topk(3, -1).values


# name: (call, the same in 64 bits, shapes of the inputs)
CALLS = {
    "token_logprobs": (_logprobs, _logprobs64, [(5, 11)]),
    "token_loss": (lambda x: (ops.token_loss(x, TOKENS),), lambda x: (torch.nn.functional.cross_entropy(x, TOKENS),), [(5, 11)]),
    "embed_tokens": (lambda w: (ops.embed_tokens(IDS, w, scale=2.0),), lambda w: (2 * w[IDS],), [(5, 6)]),
    "residual_norm": (lambda x, y, w, p, g: ops.residual_norm(x, y, w, p, g, scale=0.5, eps=1e-3),
                      lambda x, y, w, p, g: _join64(x, y, w, p, g), [(4, 6), (4, 6), (6,), (6,), (4, 6)]),
}


def _join64(x, y, w, p, g):
    s = x + 0.5 * y * (y.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * p * torch.sigmoid(g)
    return s, s * (s.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * w


def _inputs(name, seed=0):
    return [_randn(seed + i, *shape) for i, shape in enumerate(CALLS[name][2])]


def _close(got, want, what):
    assert len(got) == len(want)
    for a, b in zip(got, want):  # fp32 through reductions of at most 11 terms
        assert (a.double() - b).abs().max() <= 2.0**-18 * (1 + b.abs().max()), what


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_derivatives(name):
    fn, fn64, _ = CALLS[name]
    inputs, tangents = _inputs(name), _inputs(name, 20)
    want = torch.func.jvp(fn64, tuple(t.double() for t in inputs), tuple(t.double() for t in tangents))[1]
    _close(torch.func.jvp(fn, tuple(inputs), tuple(tangents))[1], want, name)
    with torch.no_grad(), forward_ad.dual_level():  # inputs that require no gradient
        outs = fn(*(forward_ad.make_dual(t, d) for t, d in zip(inputs, tangents)))
        got = [forward_ad.unpack_dual(o).tangent for o in outs]
    _close(got, want, name)


@pytest.mark.parametrize("name", CALLS)
def test_transforms(name):
    fn, fn64, _ = CALLS[name]
    inputs = _inputs(name)
    more = [torch.stack([t, 2 * t, t - 1]) for t in inputs]
    got = torch.vmap(fn)(*more)
    for i in range(3):
        _close([o[i] for o in got], fn64(*(t[i].double() for t in more)), name)

    def total(f):
        return lambda *a: sum((i + 1) * o.sum() for i, o in enumerate(f(*a)))

    at = tuple(range(len(inputs)))
    _close(torch.func.grad(total(fn), at)(*inputs), torch.func.grad(total(fn64), at)(*(t.double() for t in inputs)), name)


@pytest.mark.filterwarnings("ignore")  # (tracing warns of the checks of arguments)
@pytest.mark.parametrize("name", CALLS)
def test_traced_and_compiled_calls_compute(name):
    """A graph made from some inputs gives other inputs' results."""
    fn, fn64, _ = CALLS[name]
    other = _inputs(name, 40)
    want = fn64(*(t.double() for t in other))
    with torch.no_grad():
        _close(make_fx(fn)(*_inputs(name))(*other), want, name)
        _close(torch.jit.trace(fn, tuple(_inputs(name)), check_trace=False)(*other), want, name)
        graph = torch.compile(fn, backend="eager", fullgraph=True)
        graph(*_inputs(name))
        _close(graph(*other), want, name)


@pytest.mark.parametrize("name", CALLS)
def test_modes_and_subclasses_see_the_operations(name):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.n += 1
            return func(*args, **(kwargs or {}))

    class Own(torch.Tensor):
        pass

    fn, fn64, _ = CALLS[name]
    inputs = _inputs(name)
    want = fn64(*(t.double() for t in inputs))
    with Count() as mode:
        _close(fn(*inputs), want, name)
    assert mode.n > 2
    got = fn(*(t.as_subclass(Own) for t in inputs))
    assert all(type(o) is Own for o in got)
    _close([o.as_subclass(torch.Tensor) for o in got], want, name)


def test_alternatives_impossible_tokens_and_padding_keep_their_meaning():
    x = torch.tensor([[1.0, 3.0, 3.0, -0.0, 0.0, 3.0], [NAN, 1.0, INF, 0.0, NAN, 2.0], [-INF] * 6])
    tokens = torch.tensor([6, 0, -100])
    w = torch.arange(12.0).reshape(4, 3).requires_grad_(True)
    ids = torch.tensor([2, -1, 4, 0, 2, 1])
    with forward_ad.dual_level():
        got = ops.token_logprobs(x, tokens, top_k=5)
        none = ops.token_logprobs(x, tokens)
        out = ops.embed_tokens(ids, w, scale=2.0, padding_idx=-2)
        (dw,) = torch.autograd.grad(out[[0, 3, 4, 5]].sum(), [w])
    assert got.top_ids.tolist() == [[1, 2, 5, 0, 3], [0, 4, 2, 5, 1], [0, 1, 2, 3, 4]]
    assert got.logprob[0].isnan() and got.logprob[1].isnan() and got.logprob[2] == 0 and got.entropy[1:].isnan().all()
    assert none.top_logprobs is None and none.top_ids is None
    assert out[[1, 2]].isnan().all() and torch.equal(out[[0, 3]], 2 * w.detach()[[2, 0]])
    assert torch.equal(dw, torch.tensor([2.0, 2.0, 0.0, 0.0])[:, None].expand(4, 3))


def test_host_tensors_are_refused_there_too(monkeypatch):
    monkeypatch.undo()
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        for call in (lambda: ops.token_logprobs(x, t), lambda: ops.token_loss(x, t), lambda: ops.embed_tokens(t, x),
                     lambda: ops.residual_norm(x, x, torch.ones(8))):
            with pytest.raises(ValueError, match="GPU"):
                call()
