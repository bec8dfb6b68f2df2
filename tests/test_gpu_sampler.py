"""A Sampler's random numbers and sequences without a next token, on the GPU."""

import pytest
import torch

import cyclic_flow_attention.sampling as module
from cyclic_flow_attention import Sampler, Sampling

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 64, 301, 5000])
def test_numbers_of_a_seed(rows, monkeypatch):
    """The fp32 numbers that the seed's generator gives, a call for each choice,
    and less than 2^-24 more, in [0, 1)."""
    numbers, sample_tokens = [], module.sample_tokens
    monkeypatch.setattr(module, "sample_tokens", lambda logits, uniform, **kw: numbers.append(uniform) or sample_tokens(logits, uniform, **kw))
    sampler = Sampler(Sampling(seed=7), torch.zeros(rows, 2, dtype=torch.int64).cuda(), 3)
    generator = torch.Generator("cuda").manual_seed(7)
    for n in range(3):
        sampler.next(torch.zeros(rows, 9).cuda())
        u = numbers[-1]
        more = u - torch.rand(rows, device="cuda", generator=generator).double()
        assert u.dtype is torch.float64 and (u < 1).all() and (more >= 0).all() and (more < 2.0**-24).all() and more.any(), n
    assert torch.cat(numbers).unique().numel() == 3 * rows
