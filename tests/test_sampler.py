"""A Sampler's random numbers, masks and sequences without a next token, and the
generation calls that meet them, through the torch operations (no GPU compute)."""

import pytest
import torch

import cyclic_flow_attention.sampling as module
from cyclic_flow_attention import Sampler, Sampling, _native
from cyclic_flow_attention.ops import sampling


@pytest.fixture(autouse=True)
def in_torch(monkeypatch):
    monkeypatch.setattr(_native, "require_device", lambda *tensors: tensors[0].device)
    monkeypatch.setattr(sampling, "kernel_ok", lambda *tensors: False)


def _sampler(rows=3, room=4, **options):
    return Sampler(Sampling(**options), torch.zeros(rows, 2, dtype=torch.int64), room)


def test_numbers_finer_than_the_smallest_probabilities(monkeypatch):
    """Multiples of 2^-48 in [0, 1), of which the seed's fp32 numbers are the first 24 bits."""
    numbers, sample_tokens = [], module.sample_tokens
    monkeypatch.setattr(module, "sample_tokens", lambda logits, uniform, **kw: numbers.append(uniform) or sample_tokens(logits, uniform, **kw))
    sampler = _sampler(rows=1000, seed=7)
    for _ in range(3):
        sampler.next(torch.zeros(1000, 9))
    first = torch.rand(1000, generator=torch.Generator().manual_seed(7))
    assert torch.equal((numbers[0] * 2**24).floor(), first.double() * 2**24)
    u = torch.cat(numbers)
    assert u.dtype is torch.float64 and (u >= 0).all() and (u < 1).all()
    assert ((u * 2.0**48) % 1 == 0).all() and u.unique().numel() == 3000
    low = (u * 2.0**24) % 1  # uniform themselves: means of 3000, variances 1/12 and 1/9.6, within six deviations
    assert abs(low.mean() - 0.5) < 6 / (12 * 3000) ** 0.5 and abs((low * (u >= 0.5)).mean() - 0.25) < 6 / (9.6 * 3000) ** 0.5


def test_a_first_token_next_to_impossible_is_not_taken(monkeypatch):
    """Token 0 has a share of 1e-11; a number whose first 24 bits are zero does not take it by that alone."""
    rand = torch.rand
    monkeypatch.setattr(module.torch, "rand", lambda *shape, **kw: torch.cat([torch.zeros(1, shape[-1]), rand(*shape, **kw)[-1:]]) if len(shape) > 1
                        else torch.zeros(*shape))
    logits = torch.tensor([[0.0, 25.0, 25.0]]).expand(50, 3)
    assert (_sampler(rows=50).next(logits) == 1).all()
