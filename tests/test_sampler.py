"""A Sampler's random numbers, masks and sequences without a next token, and the
generation calls that meet them, through the torch operations (no GPU compute)."""

import copy

import pytest
import torch

import cyclic_flow_attention.sampling as module
from cyclic_flow_attention import Sampler, Sampling, _native
from cyclic_flow_attention.generation import generate, generate_batch
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


class _Model(torch.nn.Module):
    """Answers with the logits 0, 1, ..., 8, or ``logits``, whatever it is asked."""

    def __init__(self, logits=None):
        super().__init__()
        self.embedding = torch.nn.Parameter(torch.zeros(1))
        self.logits = torch.arange(9.0) if logits is None else logits
        self.lm_head = lambda hidden: self._of(hidden.shape[:-1])
        self.model = lambda ids, **kw: (torch.zeros(*ids.shape, 1), None)

    def _of(self, shape):
        return self.logits.expand(*shape, 9).clone()

    def forward(self, ids, cache=None, use_cache=True):
        return dict(logits=self._of(ids.shape), cache=None)


@pytest.mark.parametrize("mask", [[False] * 8 + [True], (True,) * 9, torch.ones(9, dtype=torch.bool).numpy(), 5])
def test_masks_that_are_no_masks_are_refused(mask):
    """They were passed over."""
    with pytest.raises(ValueError, match="mask"):
        _sampler(allowed=mask)


def test_masks_that_follow_the_tokens_need_them():
    """choose, and next without the tokens, passed over the function."""
    sampler = _sampler(allowed=lambda rows: torch.arange(9) == len(rows[0]) + 3)
    with pytest.raises(ValueError, match="follows the tokens"):
        sampler.choose(torch.zeros(3, 9))
    with pytest.raises(ValueError, match="follows the tokens"):
        sampler.next(torch.zeros(3, 9))
    assert sampler.room == 4 and (sampler.lengths == 2).all()
    assert sampler.next(torch.zeros(3, 9), [[], [], []]).tolist() == [3] * 3
    assert sampler.choose(torch.zeros(3, 9), torch.arange(9) == 7).tolist() == [7] * 3
    free = _sampler(allowed=lambda rows: None)
    assert free.next(torch.arange(9.0).mul(99).expand(3, 9), [[], [], []]).tolist() == [8] * 3
    assert generate(_Model(), [1], 3, sampling=Sampling(allowed=lambda rows: torch.arange(9) == len(rows[0]) + 3)) == [3, 4, 5]


NONE, NAN_ROW = torch.full((9,), -float("inf")), torch.tensor([0.0] * 8 + [float("nan")])


def test_sequences_without_a_next_token_are_told():
    """A mask that leaves nothing, logits of NaN or nothing but -inf; told from then
    on. (A logit of +inf, as of a bias that forces a token, is taken.)"""
    sampler = _sampler(rows=5, room=3, temperature=torch.tensor([1.0, 1, 1, 1, 0]), top_k=3)
    assert sampler.stuck.dtype is torch.bool and not sampler.stuck.any()
    fine, inf = torch.arange(9.0), torch.tensor([float("inf")] + [0.0] * 8)
    trial = copy.deepcopy(sampler)
    trial.choose(torch.stack([fine, NAN_ROW, inf, NONE, fine]))
    assert trial.stuck.tolist() == [False, True, False, True, False] and not sampler.stuck.any()
    allowed = torch.ones(5, 9, dtype=torch.bool)
    allowed[4] = False
    ids = sampler.choose(torch.stack([99 * fine, 99 * fine, 99 * fine, NAN_ROW, fine]), allowed)
    assert sampler.stuck.tolist() == [False, False, False, True, True]
    assert sampler.to_list(ids, [False, False, False, True, True]) == [8, 8, 8, -1, -1]
    with pytest.raises(ValueError, match="sequence 3 has no next token"):
        sampler.to_list(ids)
    with pytest.raises(ValueError, match="sequence 4 has no next token"):
        sampler.to_list(ids, [False, False, False, True, False])
    sampler.choose(torch.stack([fine] * 5))
    assert sampler.stuck.tolist() == [False, False, False, True, True]


def _ends_after(n):
    def allowed(rows):
        return torch.tensor([[len(tokens) < n] * 9 for tokens in rows])
    return allowed


def test_generate_raises_where_a_sequence_has_no_next_token():
    """It answered token 0, which the mask forbids."""
    s = Sampling(allowed=_ends_after(2), top_k=1)
    assert generate(_Model(), [1, 2], 2, sampling=s) == [8, 8]
    with pytest.raises(ValueError, match="no next token"):
        generate(_Model(), [1, 2], 3, sampling=s)
    for logits in (NONE, NAN_ROW):
        with pytest.raises(ValueError, match="no next token"):
            generate(_Model(logits), [1, 2], 3, sampling=Sampling())
    assert generate(_Model(), [1, 2], 5, sampling=s, on_token=lambda tokens: len(tokens) == 2) == [8, 8]


def test_generate_batch_raises_where_a_row_that_goes_on_has_no_next_token():
    def allowed(rows):  # the first row ends after one token, the second by its mask after two
        return torch.tensor([[len(tokens) < n] * 9 for tokens, n in zip(rows, (1, 2))])

    prompts = [[1, 2], [3]]
    with pytest.raises(ValueError, match="sequence 0 has no next token"):
        generate_batch(_Model(), prompts, 2, sampling=Sampling(allowed=allowed, top_k=1))
    assert generate_batch(_Model(), prompts, 1, sampling=Sampling(allowed=allowed, top_k=1)) == [[8], [8]]
    # rows that have stopped have no mask to keep to
    first = Sampling(allowed=lambda rows: torch.tensor([[c == 8 and not rows[0] for c in range(9)], [c < 8 for c in range(9)]]), top_k=1)
    assert generate_batch(_Model(), prompts, 3, sampling=first, eos_token_id=8) == [[8], [7, 7, 7]]


def test_a_forced_token_goes_on():
    for temperature in (0.0, 1.0):
        s = Sampling(temperature=temperature, token_bias={5: float("inf")})
        assert generate(_Model(), [1], 3, sampling=s) == [5, 5, 5]
        assert generate_batch(_Model(), [[1], [2, 3]], 2, sampling=s) == [[5, 5], [5, 5]]


def test_a_refused_choice_takes_no_room():
    sampler = _sampler(room=1, allowed=lambda rows: torch.ones(8, dtype=torch.bool) if rows[0] else None)
    for logits, generated in ((torch.zeros(2, 9), [[], [], []]), (torch.zeros(3, 9), [[1], [1], [1]]), (torch.zeros(3, 9), None)):
        with pytest.raises(ValueError):
            sampler.next(logits, generated)
        assert sampler.room == 1 and (sampler.lengths == 2).all()
    sampler.next(torch.zeros(3, 9), [[], [], []])
    with pytest.raises(ValueError, match="room"):
        sampler.next(torch.zeros(3, 9), [[], [], []])
    assert sampler.room == 0 and (sampler.lengths == 3).all()


def test_generation_in_inference_mode():
    with torch.inference_mode():
        assert generate(_Model(), [1], 3, sampling=Sampling(top_k=1, frequency=0.5)) == [8, 8, 7]  # (8 - 2 x 0.5 is 7, and 7 the lower id)
        assert generate_batch(_Model(), [[1], [2, 3]], 2, sampling=Sampling(top_k=1)) == [[8, 8], [8, 8]]
