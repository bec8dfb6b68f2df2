"""Backward passes that are themselves recorded, or batched over cotangents, run
in torch operations: their gradients where one input was computed from another,
with the forward kernels' results formed by stand-ins (no GPU compute)."""

import pytest
import torch

from cyclic_flow_attention import _native, ops
from cyclic_flow_attention.layers import autograd as layer_autograd
from cyclic_flow_attention.ops.residual import _plain
from cyclic_flow_attention.ops.vocab import _plain_logprobs, _plain_loss


@pytest.fixture
def stand_ins(monkeypatch):
    """The forward launches in torch operations; the adjoint kernels may not be called."""
    def residual_norm(x, y, weight, post, gate, scale, eps, stats=False):
        s, h = _plain(x, y, weight, post, gate, scale, eps)
        return s, h, torch.zeros(x.shape[0], 2) if stats else None

    def norm_train(x, weight, gate, eps, prescale):
        assert prescale == 1.0
        return _norm(x, weight, gate, eps)

    def logprobs(logits, tokens, k, ignore, stats=False):
        ids = logits.topk(k, -1).indices if k else None
        out = _plain_logprobs(logits, tokens, ids, ignore)
        return (*out, *(() if k else (None,)), ids, torch.zeros(logits.shape[:-1] + (2,)) if stats else None)

    def token_loss(logits, labels, ignore, stats=False):
        return _plain_loss(logits, labels, ignore)[0], torch.zeros(1)

    def launch(*args, **kwargs):
        raise AssertionError("an adjoint kernel was called")

    monkeypatch.setattr(_native, "residual_norm", residual_norm)
    monkeypatch.setattr(_native, "norm_train", norm_train)
    monkeypatch.setattr(_native, "logprobs", logprobs)
    monkeypatch.setattr(_native, "token_loss", token_loss)
    for name in ("residual_norm_grad", "norm_grad", "logprobs_grad", "token_loss_grad"):
        monkeypatch.setattr(_native, name, launch)


def _norm(x, weight, gate, eps):
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight
    return y if gate is None else y * torch.sigmoid(gate)


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


# y and gate as functions of x; fp32 through two reductions of 24 terms: 2^-18 of the largest value
DEPENDENT = {"y of x": (torch.tanh, None), "y is x": (lambda x: x, None), "gate of x": (lambda x: 2 * x, torch.sin),
             "gate of y": (torch.tanh, torch.tanh)}


@pytest.mark.parametrize("case", DEPENDENT)
def test_join_of_a_block_computed_from_its_residual(stand_ins, case):
    make_y, make_gate = DEPENDENT[case]
    x0, w0, p0 = _randn(1, 5, 24), 1 + 0.1 * _randn(2, 24), 1 + 0.1 * _randn(3, 24)
    cots = [_randn(4, 5, 24), _randn(5, 5, 24)]
    results = []
    for dtype in (torch.float32, torch.float64):
        x, w, p = (t.to(dtype).requires_grad_(True) for t in (x0, w0, p0))
        y = make_y(x)
        gate = None if make_gate is None else make_gate(y if case == "gate of y" else x)
        join = ops.residual_norm if dtype == torch.float32 else lambda a, b, c, d, g, s, e: _plain_double(a, b, c, d, g, s, e)
        s, h = join(x, y, w, p, gate, 0.5, 1e-3)
        grads = torch.autograd.grad([s, h], [x, w, p], [c.to(dtype) for c in cots], create_graph=True)
        again = torch.autograd.grad(sum(g.square().sum() for g in grads), [x, w, p])
        results.append([*grads, *again])
    for got, want in zip(*results):
        assert (got.double() - want).abs().max() <= 2.0**-18 * want.abs().max(), case


def _plain_double(x, y, weight, post, gate, scale, eps):
    b = y * (y.square().mean(-1, keepdim=True) + eps).rsqrt() * post
    s = x + scale * (b if gate is None else b * torch.sigmoid(gate))
    return s, s * (s.square().mean(-1, keepdim=True) + eps).rsqrt() * weight


def test_batched_cotangents_leave_the_graph_before_the_join(stand_ins):
    x, w = _randn(1, 5, 24).requires_grad_(True), _randn(2, 24)
    cots = _randn(3, 3, 5, 24)
    s, h = ops.residual_norm(x, torch.tanh(x), w)
    (batched,) = torch.autograd.grad(h, [x], cots, is_grads_batched=True, retain_graph=True)
    again = torch.autograd.grad(h, [x], cots, is_grads_batched=True)[0]  # the graph of tanh is still there
    z = x.detach().double().requires_grad_(True)
    t = z + torch.tanh(z)
    ref = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    for i in range(3):
        (want,) = torch.autograd.grad(ref, [z], cots[i].double(), retain_graph=True)
        assert (batched[i].double() - want).abs().max() <= 2.0**-18 * want.abs().max()
    assert torch.equal(batched, again)


@pytest.mark.parametrize("gate_of", [torch.sin, lambda x: x])
def test_norm_whose_gate_was_computed_from_its_input(stand_ins, gate_of):
    def general(x, weight, gate):
        return _norm(x, weight, gate, 1e-3)

    results = []
    for dtype in (torch.float32, torch.float64):
        x = _randn(1, 5, 24).to(dtype).requires_grad_(True)
        w = _randn(2, 24).to(dtype)
        if dtype == torch.float32:
            y = layer_autograd.rms_norm(x, w, gate_of(x), 1e-3, 1.0, general)
        else:
            y = general(x, w, gate_of(x))
        (dx,) = torch.autograd.grad(y, [x], _randn(3, 5, 24).to(dtype), create_graph=True)
        results.append([dx, torch.autograd.grad(dx.square().sum(), [x])[0]])
    for got, want in zip(*results):
        assert (got.double() - want).abs().max() <= 2.0**-18 * want.abs().max()


def test_inputs_that_no_cotangent_reaches(stand_ins):
    """s does not depend on the next norm's weight: zeros, as the kernels give."""
    x0, w0 = _randn(1, 5, 24), _randn(2, 24)
    for x_grad in (False, True):
        x, w = x0.clone().requires_grad_(x_grad), w0.clone().requires_grad_(True)
        s, _ = ops.residual_norm(x, 2 * x0, w)
        wanted = [x, w] if x_grad else [w]
        grads = torch.autograd.grad(s, wanted, torch.ones_like(s), create_graph=True)
        assert not grads[-1].any()
        if x_grad:
            assert torch.equal(grads[0], torch.ones_like(s))


INF, NAN = float("inf"), float("nan")


def test_rows_without_probabilities_that_no_cotangent_reaches(stand_ins):
    """Zeros, whatever the row holds; the other rows' gradients as ever."""
    x0 = _randn(1, 6, 9)
    x0[0], x0[1, 2], x0[2, 3], x0[3, 4:] = -INF, NAN, INF, -INF
    tokens = torch.tensor([0, 1, 2, 3, -100, 5])
    keep = torch.tensor([0.0, 0.0, 0.0, 1.0, 1.0, 0.0])
    cots = [keep * _randn(2, 6), (keep * _randn(3, 6)), keep[:, None] * _randn(4, 6, 2)]
    x = x0.clone().requires_grad_(True)
    got = ops.token_logprobs(x, tokens, top_k=2)
    (dx,) = torch.autograd.grad(got[:3], [x], cots, create_graph=True)
    z = x0[3:5].double().requires_grad_(True)
    want = _plain_logprobs(z, tokens[3:5], got.top_ids[3:5], -100)
    (dz,) = torch.autograd.grad(want, [z], [c[3:5].double() for c in cots])
    assert not dx[:3].any() and not dx[5].any() and (dx[3:5] - dz).abs().max() <= 2.0**-18 * dz.abs().max()
    for i in range(3):  # one that a cotangent reaches
        (dx,) = torch.autograd.grad(got[:2], [x], [torch.eye(6)[i], torch.zeros(6)], create_graph=True)
        assert dx[i].isnan().all() and not dx[[r for r in range(6) if r != i]].any()
    ignored = tokens.masked_fill(tokens == 0, -100)  # the first row's label is ignored
    (dx,) = torch.autograd.grad(ops.token_logprobs(x, ignored).logprob, [x], torch.eye(6)[0], create_graph=True)
    assert not dx.any()


def test_loss_beside_rows_without_probabilities(stand_ins):
    x0 = _randn(1, 4, 9)
    x0[0], x0[1, 2] = -INF, NAN
    labels = torch.tensor([-100, -100, 3, 8])
    x, z = x0.clone().requires_grad_(True), x0[2:].double().requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.token_loss(x, labels), [x], create_graph=True)
    (dz,) = torch.autograd.grad(torch.nn.functional.cross_entropy(z, labels[2:]), [z])
    assert not dx[:2].any() and (dx[2:] - dz).abs().max() <= 2.0**-18 * dz.abs().max()


def test_derivative_with_respect_to_cotangents_of_zero(stand_ins):
    """The forward derivative as the adjoint of the adjoint at cotangents of zero."""
    x, u = _randn(1, 3, 9).requires_grad_(True), _randn(2, 3, 9)
    v = torch.zeros(3, requires_grad=True)
    tokens = torch.tensor([1, 2, 8])
    (dx,) = torch.autograd.grad(ops.token_logprobs(x, tokens).logprob, [x], v, create_graph=True)
    (got,) = torch.autograd.grad(dx, [v], u)
    p = x.detach().double().softmax(-1)
    want = u.double().gather(1, tokens[:, None])[:, 0] - (p * u).sum(-1)
    assert (got - want).abs().max() <= 2.0**-18 * want.abs().max()


def test_batched_cotangents_of_log_probabilities(stand_ins):
    x = _randn(1, 4, 9)
    x[1] = -INF
    x.requires_grad_(True)
    tokens = torch.tensor([0, 1, -100, 8])
    got = ops.token_logprobs(x, tokens, top_k=2)[:3]
    cots = [_randn(i, 5, *o.shape) for i, o in enumerate(got)]
    for c in cots:
        c[:, 1] = 0
    batched = torch.autograd.grad(got, [x], cots, is_grads_batched=True, retain_graph=True)[0]
    for i in range(5):
        (one,) = torch.autograd.grad(got, [x], [c[i] for c in cots], create_graph=True)
        assert (batched[i] - one).abs().max() <= 2.0**-20 * one.abs().max() and not one[1].any()
    loss = ops.token_loss(x, tokens.masked_fill(torch.arange(4) == 1, -100))
    batched = torch.autograd.grad(loss, [x], torch.tensor([1.0, -2.0]), is_grads_batched=True, retain_graph=True)[0]
    (one,) = torch.autograd.grad(loss, [x], create_graph=True)
    assert torch.equal(batched, torch.stack([one, -2 * one]))
