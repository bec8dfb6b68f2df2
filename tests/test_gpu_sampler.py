"""A Sampler's random numbers and sequences without a next token, on the GPU."""

import pytest
import torch

import cyclic_flow_attention.sampling as module
from cyclic_flow_attention import CyclicFlowAttentionConfig, CyclicFlowAttentionForCausalLM, Sampler, Sampling
from cyclic_flow_attention.generation import generate, generate_batch

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


V = 301


def _model():
    torch.manual_seed(3)
    config = CyclicFlowAttentionConfig(hidden_size=256, num_heads=1, head_dim=256, num_hidden_layers=1, vocab_size=V,
                                       intermediate_size=512, num_slots=128)
    return CyclicFlowAttentionForCausalLM(config).cuda().eval().to_bfloat16()


def test_generation_raises_where_a_sequence_has_no_next_token():
    """A mask that leaves nothing, from the first token on or after two of them; rows that have stopped do not count."""
    model, prompts = _model(), [[10, 20, 30], [7]]
    none = torch.zeros(2, V, dtype=torch.bool)
    none[0] = True

    def later(rows):
        return torch.tensor([[len(rows[0]) < 9] * V, [len(rows[1]) < 2] * V])

    for mask, n in ((none, 1), (later, 3)):
        s = Sampling(allowed=mask)
        with pytest.raises(ValueError, match="sequence 1 has no next token"):
            generate_batch(model, prompts, n, sampling=s)
        if n > 1:
            assert [len(r) for r in generate_batch(model, prompts, 9, sampling=s, on_token=lambda r: len(r) == 2)] == [2, 2]
    with pytest.raises(ValueError, match="sequence 0 has no next token"):
        generate(model, [7], 2, sampling=Sampling(allowed=none[1]))
    ids = torch.tensor([[10, 20, 30], [7, 8, 9]]).cuda()
    with pytest.raises(ValueError, match="sequence 1 has no next token"):
        model.generate(ids, 3, sampling=Sampling(allowed=none))
    with pytest.raises(ValueError, match="sequence 1 has no next token"):
        model.generate(ids, 3, eos_token_id=0, sampling=Sampling(allowed=none))
    forced = model.generate(ids, 3, sampling=Sampling(token_bias={5: float("inf")}))
    assert forced.shape == (2, 6) and (forced[:, 3:] == 5).all()


def test_graphed_decoding_tells_the_sequences_that_are_stuck():
    model = _model()
    ids = torch.randint(0, V, (3, 20), generator=torch.Generator().manual_seed(2)).cuda()
    allowed = torch.ones(3, V, dtype=torch.bool).cuda()
    with torch.no_grad():
        out = model(ids, use_cache=True)
        sampler = Sampler(Sampling(allowed=allowed, seed=4), ids, 9)
        first = sampler.next(out["logits"][:, -1])
        step = model.graphed_decoder(out["cache"], first[:, None], sampler=sampler)
        for n in range(8):
            if n == 4:  # the mask's own buffer, as a grammar between replays edits it
                allowed[1] = False
            if n == 6:
                allowed[1] = True
            tokens = step.step()
            assert sampler.stuck.tolist() == [False, n >= 4, False], n
        assert sampler.to_list(tokens[:, 0], [False, True, False]) == [tokens[0, 0], -1, tokens[2, 0]]
        with pytest.raises(ValueError, match="sequence 1 has no next token"):
            sampler.to_list(tokens[:, 0])
