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
