"""Generation and distillation of the model through the operators on its logits."""

import pytest
import torch

import logits_bounds as lb
from cyclic_flow_attention import CyclicFlowAttentionConfig, CyclicFlowAttentionForCausalLM, Sampler, Sampling, ops
from cyclic_flow_attention.generation import generate, generate_batch

pytestmark = pytest.mark.gpu

V = 301


def _model(seed=3, dtype=torch.bfloat16, layers=2):
    torch.manual_seed(seed)
    config = CyclicFlowAttentionConfig(hidden_size=256, num_heads=1, head_dim=256, num_hidden_layers=layers, vocab_size=V,
                                       intermediate_size=512, num_slots=128)
    model = CyclicFlowAttentionForCausalLM(config).cuda().eval()
    return model.to_bfloat16() if dtype == torch.bfloat16 else model


def _replay(model, prompt, generated, s, uniforms):
    """The tokens that the definitions choose after the model's own logits of each prefix."""
    cache, current, tokens = None, list(prompt), list(prompt)
    for n, token in enumerate(generated):
        with torch.no_grad():
            out = model(torch.tensor([current]).cuda(), cache=cache, use_cache=True)
        cache, x = out["cache"], out["logits"][:, -1].cpu()
        y, _ = lb.adjust(x.double(), [tokens], [len(tokens)], [len(prompt)], [s.repetition], [s.presence], [s.frequency], None,
                         [list((s.token_bias or {}).items())], None if s.allowed is None else s.allowed[None].cpu(), x.dtype)
        want, _ = lb.choice(y[0].to(x.dtype).double().numpy(), float(uniforms[n]), s.temperature, s.top_k, s.top_p, s.min_p)
        assert token == want, n
        tokens.append(token)
        current = [token]


def _uniforms(seed, steps, rows):
    g = torch.Generator("cuda").manual_seed(seed)
    return [torch.rand(rows, device="cuda", generator=g).cpu() for _ in range(steps)]


def test_generate_with_sampling():
    model, prompt = _model(), [5, 9, 200, 9]
    allowed = torch.arange(V).cuda() % 7 != 3
    s = Sampling(temperature=0.8, top_k=60, top_p=0.95, min_p=0.001, repetition=1.3, presence=0.1, frequency=0.2, token_bias={17: 1.5},
                 allowed=allowed, seed=11)
    got = generate(model, prompt, 12, sampling=s)
    assert len(got) == 12 and all(t % 7 != 3 for t in got) and got == generate(model, prompt, 12, sampling=s)
    _replay(model, prompt, got, s, [u[0] for u in _uniforms(11, 12, 1)])
    out = model.generate(torch.tensor([prompt]).cuda(), 12, sampling=s)
    assert out[0].tolist() == prompt + got
    with pytest.raises(ValueError, match="generate_batch"):
        model.generate(torch.tensor([prompt]).cuda(), 2, sampling=Sampling(allowed=lambda rows: None))


def test_greedy_sampling_is_the_greedy_choice():
    model, prompts = _model(), [[10, 20, 30], list(range(4, 67))]
    want = generate_batch(model, prompts, max_new_tokens=8)
    assert generate_batch(model, prompts, max_new_tokens=8, sampling=Sampling(temperature=0.0)) == want
    assert generate(model, prompts[0], 8, sampling=Sampling(temperature=0.0)) == generate(model, prompts[0], 8)


def test_generate_batch_with_a_mask_that_follows_the_tokens():
    """Each row repeats what it has said less, and may only say tokens above its last one."""
    model, prompts = _model(), [[10, 20, 30], list(range(4, 67)), [7]]

    def above(rows):
        allowed = torch.zeros(3, V, dtype=torch.bool)
        for r, tokens in enumerate(rows):
            allowed[r, (tokens[-1] + 1 if tokens else 0):] = True
        allowed[:, V - 1] = True
        return allowed

    s = Sampling(temperature=torch.tensor([0.5, 1.0, 2.0]), top_p=0.9, frequency=torch.tensor([0.5, 0.0, 0.1]), allowed=above, seed=5)
    rows = generate_batch(model, prompts, 6, sampling=s)
    assert rows == generate_batch(model, prompts, 6, sampling=s)
    for tokens in rows:
        assert len(tokens) == 6 and all(b > a or b == V - 1 for a, b in zip(tokens, tokens[1:]))


def test_graphed_decoding_with_a_sampler():
    """Replays give the tokens of eager steps with the same seed, and stop where there is no room."""
    model = _model()
    ids = torch.randint(0, V, (3, 20), generator=torch.Generator().manual_seed(2)).cuda()
    s = Sampling(temperature=0.9, top_k=80, repetition=1.2, frequency=0.1, bias=torch.linspace(0, 1, V), seed=4)
    with torch.no_grad():
        out = model(ids, use_cache=True)
        eager, captured = Sampler(s, ids, 8), Sampler(s, ids, 8)
        first = eager.next(out["logits"][:, -1])
        assert torch.equal(first, captured.next(out["logits"][:, -1]))
        step = model.graphed_decoder(out["cache"], first[:, None], sampler=captured)
        cache, current = out["cache"], first[:, None]
        for n in range(7):
            r = model(current, cache=cache, use_cache=True)
            cache, current = r["cache"], eager.next(r["logits"][:, -1])[:, None]
            assert torch.equal(step.step(), current), n
        torch.cuda.synchronize()
        assert torch.equal(eager.history, captured.history) and torch.equal(eager.lengths, captured.lengths)
        assert (eager.lengths == 28).all() and (eager.history >= 0).all()
        with pytest.raises(ValueError, match="room"):
            step.step()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_of_sampled_sequences(dtype):
    """A student samples, the teacher scores, the student's loss and gradients are those of its logits."""
    student, teacher = _model(3, dtype), _model(4, dtype)
    prompts = torch.randint(0, V, (2, 10), generator=torch.Generator().manual_seed(1)).cuda()
    ids = student.generate(prompts, 54, sampling=Sampling(top_p=0.95, seed=9))
    assert ids.shape == (2, 64)
    mask = (torch.arange(64).cuda()[None] < torch.tensor([64, 41]).cuda()[:, None]).long()
    for m, T, tail in ((None, 2.0, False), (mask, 1.0, True)):
        score = teacher.score(ids, top_k=12, attention_mask=m)
        student.zero_grad(set_to_none=True)
        loss = student.distill(ids, score.top_ids, score.top_logprobs, temperature=T, tail=tail, attention_mask=m)
        loss.backward()
        got = {n: p.grad.clone() for n, p in student.named_parameters() if p.grad is not None}
        student.zero_grad(set_to_none=True)
        logits = student(ids, attention_mask=m)["logits"]
        top = score.top_ids if m is None else score.top_ids.masked_fill(m[:, 1:, None] == 0, -100)
        (ref, err), (dx, _) = lb.distill(logits[:, :-1].detach().cpu().reshape(-1, V).double(), top.cpu().reshape(-1, 12),
                                         score.top_logprobs.cpu().reshape(-1, 12).double(), T, tail, None, dtype)
        assert abs(loss.item() - ref) <= err
        logits.backward(torch.nn.functional.pad(dx.view(2, 63, V).to(dtype), (0, 0, 0, 1)).cuda())
        for n, p in student.named_parameters():
            if p.grad is not None and n.endswith(("lm_head.weight", "embeddings.weight", "down_proj.weight")):
                # fp32 sums in another order; bf16 gradients of the logits off by a rounding here and there
                bar = 1e-4 if dtype == torch.float32 else 2e-2
                assert (got[n].double() - p.grad.double()).norm() <= bar * p.grad.double().norm(), n
    with torch.no_grad():
        assert abs(student.distill(ids, score.top_ids, score.top_logprobs, tail=True, attention_mask=mask).item() - ref) <= 0.02 * ref
    with pytest.raises(ValueError, match="teacher's tokens"):
        student.distill(ids, score.top_ids[:, 1:], score.top_logprobs[:, 1:])
    assert ops.SampledTokens._fields == ("ids", "logprob")
