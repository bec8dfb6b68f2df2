"""The torch operations behind the operators on a model's logits where ids
repeat and options leave their range (no GPU compute)."""

import math

import pytest
import torch

from cyclic_flow_attention import _native, ops
from cyclic_flow_attention.ops import distill, sampling

INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def in_torch(monkeypatch):
    monkeypatch.setattr(_native, "require_device", lambda *tensors: tensors[0].device)
    for module in (distill, sampling):
        monkeypatch.setattr(module, "kernel_ok", lambda *tensors: False)


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("tail", [False, True])
def test_a_token_named_several_times(tail):
    """Entries of 0.1, 0.2 and 0.3 for one token against one of 0.6: the loss by
    entries is less by the constant sum p_i log(P / p_i), the gradient the same."""
    x = _randn(1, 1, 9).requires_grad_(True)
    split, whole = torch.tensor([[0.1, 0.2, 0.3, 0.25]]), torch.tensor([[0.6, 0.25]])
    losses, grads = [], []
    for ids, p in ((torch.tensor([[5, 5, 5, 2]]), split), (torch.tensor([[5, 2]]), whole)):
        losses.append(ops.distill_loss(x, ids, p.log(), tail=tail))
        grads.append(torch.autograd.grad(losses[-1], [x])[0])
    scale = 1.0 if tail else 1 / 0.85
    less = scale * sum(p * math.log(0.6 / p) for p in (0.1, 0.2, 0.3))
    # fp32 values of order one through sums of nine terms
    assert abs(losses[1].item() - losses[0].item() - less) < 2.0**-19
    assert (grads[0] - grads[1]).abs().max() < 2.0**-20


def test_a_number_that_is_none_takes_the_first_kept_token():
    x = torch.tensor([[1.0, 3, 3, 0, 2, 5], [-math.inf, 1, 0, 2, 2, 2], [0, 0, 0, 0, 0, 0]])
    got = ops.sample_tokens(x, torch.full((3,), NAN), top_k=torch.tensor([1, 5, 0]), top_p=torch.tensor([1.0, 0.9, 1.0]))
    zero = ops.sample_tokens(x, torch.zeros(3), top_k=torch.tensor([1, 5, 0]), top_p=torch.tensor([1.0, 0.9, 1.0]))
    assert got.ids.tolist() == zero.ids.tolist() == [5, 1, 0] and torch.equal(got.logprob, zero.logprob)


def test_a_min_p_above_one_is_one():
    """The tokens as large as the largest are kept, all of them."""
    x = torch.tensor([[3.0, 0, 3, 3]]).expand(4, 4)
    u, least = torch.tensor([0.1, 0.5, 0.9, 0.9]), torch.tensor([2.0, math.inf, 1.0, 1.5])
    got = ops.sample_tokens(x, u, min_p=least)
    assert got.ids.tolist() == [0, 2, 3, 3] and (got.logprob + math.log(3)).abs().max() < 1e-6
    got = ops.sample_tokens(x, u, min_p=least, top_k=torch.tensor([2, 2, 1, 0]))
    assert got.ids.tolist() == [0, 2, 0, 3]


@pytest.mark.parametrize("least", [0.0, 0.5, 1.0])
def test_an_infinite_temperature_weighs_the_finite_alike(least):
    x = torch.tensor([[1.0, -math.inf, 3, -math.inf, 2, -1e30]]).expand(4, 6)
    u = torch.tensor([0.0, 0.3, 0.5, 0.9])
    got = ops.sample_tokens(x, u, temperature=math.inf, min_p=least)
    assert got.ids.tolist() == [0, 2, 4, 5] and (got.logprob + math.log(4)).abs().max() < 1e-6
    got = ops.sample_tokens(x, u, temperature=math.inf, top_k=3)
    assert got.ids.tolist() == [0, 0, 2, 4] and (got.logprob + math.log(3)).abs().max() < 1e-6


def test_equal_token_biases_are_added_up_before_the_logit():
    """As the kernel does it: 1 + (2^-24 + 2^-24) is one step above 1 in fp32, (1 + 2^-24) + 2^-24 is 1."""
    step = 2.0**-24
    x = torch.tensor([[1.0, -0.0, 1.0, 0.5], [1.0, 1.0, 1.0, -INF]]).requires_grad_(True)
    y = ops.adjust_logits(x, token_bias=(torch.tensor([[0, 2, 0, 9], [3, 1, 3, 1]]), torch.tensor([[step, 1.0, step, 5.0], [1.0, step, 1.0, step]])))
    assert y.tolist() == [[1 + 2 * step, -0.0, 2.0, 0.5], [1.0, 1 + 2 * step, 1.0, -INF]] and y[0, 1].signbit()
    (dx,) = torch.autograd.grad(y, [x], torch.ones(2, 4))
    assert dx.tolist() == [[1.0] * 4] * 2


@pytest.mark.parametrize("T", [0.25, 1.0, 4.0])
def test_rows_of_the_lowest_value_at_any_temperature(T):
    """They are rows of zeros: divided by a temperature below 1 first, they were of -inf."""
    x, ids, values = torch.full((2, 6), torch.finfo(torch.float32).min), torch.tensor([[1, 3], [0, 2]]), torch.tensor([[-0.5, -1.0], [0.0, -2.0]])
    results = []
    for logits in (x, torch.zeros(2, 6)):
        logits = logits.clone().requires_grad_(True)
        loss = ops.distill_loss(logits, ids, values, temperature=T)
        results.append((loss, torch.autograd.grad(loss, [logits])[0]))
    assert results[0][0].isfinite() and torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    if T < 1:  # a quarter of the mass at a token that the mask took
        x[0, 0] = 5.0
        loss = ops.distill_loss(x[:1], torch.tensor([[0, 1]]), torch.tensor([[math.log(3.0), 0.0]]) * T, temperature=T)
        assert loss == INF or abs(loss.item() / (0.25 / T * torch.finfo(torch.float32).max) - 1) < 2.0**-20


def test_a_numbers_penalty_is_the_tensors():
    """torch divides by a number by a product with its reciprocal on a GPU; either way the kernel divides."""
    x = _randn(3, 4, 50)
    history = torch.arange(50)[None]
    y = ops.adjust_logits(x, history, repetition=1.3, presence=0.1, frequency=0.7)
    per_row = {n: torch.full((4,), v) for n, v in (("repetition", 1.3), ("presence", 0.1), ("frequency", 0.7))}
    assert torch.equal(y, ops.adjust_logits(x, history, **per_row))
