"""The operators on a model's logits where ids repeat and options leave their
range: the kernels, on every path that chooses a token."""

import math

import pytest
import torch

from cyclic_flow_attention import ops

pytestmark = pytest.mark.gpu

BF, F32, INF, NAN = torch.bfloat16, torch.float32, float("inf"), float("nan")
# rows of a wave's, of a workgroup's and of parts' columns
SIZES = [(5, 9), (5, 5003), (700, 8200), (5, 50001)]


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def _four(V):
    """Four columns, far apart, of a row of V."""
    return [0, V // 3, V // 2, V - 1]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V", SIZES)
def test_an_infinite_temperature_weighs_the_finite_alike(rows, V, dtype):
    at = _four(V)
    x = torch.full((rows, V), -INF)
    x[:, at] = torch.tensor([1.0, 3.0, -1e30, 2.0])
    x, u = x.to(dtype).cuda(), torch.full((rows,), 0.6).cuda()
    for least in (0.0, 0.5, 1.0):
        for T in (INF, torch.full((rows,), INF).cuda()):
            got = ops.sample_tokens(x, u, temperature=T, min_p=least)
            assert (got.ids == at[2]).all() and (got.logprob + math.log(4)).abs().max() < 1e-6, least
            got = ops.sample_tokens(x, u, temperature=T, min_p=least, top_k=3)  # without the least
            assert (got.ids == at[1]).all() and (got.logprob + math.log(3)).abs().max() < 1e-6, least
            got = ops.sample_tokens(x, u, temperature=T, min_p=least, top_p=0.5)
            assert (got.ids == at[3]).all() and (got.logprob + math.log(2)).abs().max() < 1e-6, least


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("V", [9, 8200, 50001])
def test_equal_token_biases_are_added_up_before_the_logit(V, inplace):
    """1 + (2^-24 + 2^-24) is one step above 1 in fp32, (1 + 2^-24) + 2^-24 is 1."""
    step, x = 2.0**-24, torch.ones(3, V).cuda()
    ids, values = torch.tensor([V - 1, 2, V - 1, V, 0]).cuda(), torch.tensor([step, 1.0, step, 5.0, step]).cuda()
    want = x.clone()
    want[:, V - 1], want[:, 2] = 1 + 2 * step, 2.0
    y = ops.adjust_logits(x, token_bias=(ids, values), out=x if inplace else None)
    assert torch.equal(y, want)


@pytest.mark.parametrize("V", [1000, 9000, 50000])
def test_numbers_on_the_borders_of_equal_shares(V):
    """500 tokens of one weight: number u takes token floor(500 u), for every u by itself."""
    x = torch.full((8, V), -INF)
    x[:, :500] = 0.0
    u = torch.tensor([0.0, 0.25, 0.5, 0.998, 1 - 2.0**-24, 0.002, 0.75, 0.001])
    want = (u.double() * 500).floor().long()  # (the weights and their sum are exact)
    assert want.tolist() == [0, 125, 250, 499, 499, 1, 375, 0]
    for k, p in ((0, 1.0), (500, 1.0), (0, 0.9999)):
        got = ops.sample_tokens(x.cuda(), u.cuda(), top_k=k, top_p=p)
        assert got.ids.tolist() == want.tolist() and (got.logprob + math.log(500)).abs().max() < 2.0**-20, (k, p)


@pytest.mark.parametrize("rows,V", SIZES)
def test_numbers_that_are_none_and_min_p_above_one(rows, V):
    at = _four(V)
    x = torch.full((rows, V), -1.0)
    x[:, at] = torch.tensor([0.0, 3.0, 1.0, 3.0])
    nan, u = torch.full((rows,), NAN).cuda(), torch.full((rows,), 0.75).cuda()
    for kw in (dict(top_k=1), dict(top_k=2), dict(top_p=0.001), dict(top_k=200, top_p=0.001), dict(min_p=0.9)):
        assert (ops.sample_tokens(x.cuda(), nan, **kw).ids == at[1]).all(), kw
    for kw in (dict(), dict(top_k=min(V - 1, 300)), dict(top_k=3), dict(top_p=0.9999)):
        got = ops.sample_tokens(x.cuda(), u, min_p=torch.full((rows,), 1.5).cuda(), **kw)
        assert (got.ids == at[3]).all() and (got.logprob + math.log(2)).abs().max() < 1e-6, kw


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V,dtype", [(9, F32), (5003, F32), (5003, BF)])
def test_a_token_named_several_times(V, dtype, tail):
    """Entries of 0.1, 0.2 and 0.3 for one token against one of 0.6: the loss by
    entries is less by the constant sum p_i log(P / p_i), the gradient the same."""
    x = _randn(1, 4, V).to(dtype).cuda().requires_grad_(True)
    losses, grads = [], []
    for ids, p in (([5, 5, 5, 2], [0.1, 0.2, 0.3, 0.25]), ([5, 2], [0.6, 0.25])):
        losses.append(ops.distill_loss(x, torch.tensor([ids] * 4).cuda(), torch.tensor([p] * 4).log().cuda(), tail=tail))
        grads.append(torch.autograd.grad(losses[-1], [x])[0].double())
    less = (1.0 if tail else 1 / 0.85) * sum(p * math.log(0.6 / p) for p in (0.1, 0.2, 0.3))
    # fp32 values of order ten
    assert abs(losses[1].item() - losses[0].item() - less) < 16 * 2.0**-22
    # fp32 masses of order one, off by a few steps, over four rows; each rounded once
    assert (grads[0] - grads[1]).abs().max() < 2.0**-22 + torch.finfo(dtype).eps * grads[1].abs().max()


@pytest.mark.parametrize("V", [9, 5003])
def test_large_divergences_whose_mean_fits(V):
    """Tokens that a mask of the type's lowest value takes from the student: a row's
    loss past fp32, or its logarithms over the temperature, beside a mean that is not."""
    low = torch.finfo(F32).min
    x = torch.full((3, V), low)
    x[:, 0] = 5.0
    x[1:, 4] = 5.0
    # 0.5 e^1e-6 twice: with the tail row 0 costs 1.000001 times the largest value, the others log 2 and a little
    ids, values = torch.tensor([[1, 2], [0, 4], [0, 4]]), torch.full((3, 2), math.log(0.5) + 1e-6)
    loss = ops.distill_loss(x.cuda(), ids.cuda(), values.cuda(), tail=True)
    assert abs(loss.item() / (-low / 3 * (1 + 1e-6)) - 1) < 2.0**-20
    # a quarter of the mass at 2 x the lowest value below the largest
    ids, values = torch.tensor([[0, 1]]), torch.tensor([[math.log(3.0), 0.0]]) * 0.5
    loss = ops.distill_loss(x[:1].cuda(), ids.cuda(), values.cuda(), temperature=0.5)
    assert abs(loss.item() / (0.25 * 2 * -low) - 1) < 2.0**-20
    assert ops.distill_loss(x[:1].cuda(), ids.cuda() + 1, values.cuda(), temperature=0.5).item() == INF  # past fp32


@pytest.mark.parametrize("dtype", [BF, torch.float16, F32])
def test_a_numbers_penalty_in_torch_operations(dtype, monkeypatch):
    """The torch form divides by a number as the kernel does, not by a product with its reciprocal."""
    from cyclic_flow_attention.ops import sampling

    x, history = (_randn(3, 4, 5003) * 3).to(dtype).cuda(), torch.arange(5003).cuda()[None]
    y = ops.adjust_logits(x, history, repetition=1.3, presence=0.1, frequency=0.7)
    monkeypatch.setattr(sampling, "kernel_ok", lambda *tensors: False)
    assert torch.equal(y, ops.adjust_logits(x, history, repetition=1.3, presence=0.1, frequency=0.7))
