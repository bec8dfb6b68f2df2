"""The model's training step and scoring through the operators around its
blocks: losses and gradients against the same model in torch operations, what
runs where, and hooks that still see their modules."""

import pytest
import torch
import torch.nn.functional as F

import lm_bounds as lm
from cyclic_flow_attention import CyclicFlowAttentionConfig, CyclicFlowAttentionForCausalLM, _native
from cyclic_flow_attention.models.cyfa import modeling_cyfa

pytestmark = pytest.mark.gpu

V = 301


def _model(dtype, layers=2, tie=False):
    torch.manual_seed(3)
    config = CyclicFlowAttentionConfig(hidden_size=256, num_heads=1, head_dim=256, num_hidden_layers=layers, vocab_size=V,
                                       intermediate_size=512, num_slots=128, tie_word_embeddings=tie)
    model = CyclicFlowAttentionForCausalLM(config).cuda()
    return model.to_bfloat16() if dtype == torch.bfloat16 else model


def _batch(B=2, T=70):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (B, T), generator=g)
    labels = ids.clone()
    labels[1, 50:] = -100
    labels[0, 0] = -100
    return ids.cuda(), labels.cuda()


def _grads(model, ids, labels):
    model.zero_grad(set_to_none=True)
    out = model(ids, labels=labels)
    out["loss"].backward()
    return out, {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


_GATES = {"dt_bias": "a_proj.weight", "A_log": "a_proj.weight", "b_proj.bias": "b_proj.weight", "d_proj.bias": "d_proj.weight"}


class _Calls:
    def __init__(self, monkeypatch, *names):
        self.n = dict.fromkeys(names, 0)
        for name in names:
            monkeypatch.setattr(_native, name, self._count(name, getattr(_native, name)))

    def _count(self, name, fn):
        def call(*args, **kwargs):
            self.n[name] += 1
            return fn(*args, **kwargs)

        return call


@pytest.mark.parametrize("tie", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step_matches_torch_operations(monkeypatch, dtype, tie):
    model = _model(dtype, tie=tie)
    ids, labels = _batch()
    calls = _Calls(monkeypatch, "embed", "embed_grad", "token_loss", "token_loss_grad", "residual_norm", "residual_norm_grad")
    out, got = _grads(model, ids, labels)
    assert calls.n == dict(embed=1, embed_grad=1, token_loss=1, token_loss_grad=1, residual_norm=4, residual_norm_grad=4)
    loss = F.cross_entropy(out["logits"][:, :-1].double().reshape(-1, V), labels[:, 1:].reshape(-1), ignore_index=-100)
    assert abs(out["loss"].item() - loss.item()) <= 2.0**-18 * loss.item()
    monkeypatch.setattr(modeling_cyfa, "hip_autograd_ok", lambda *tensors: False)  # the same blocks, joined in torch operations
    plain, want = _grads(model, ids, labels)
    assert calls.n["token_loss"] == calls.n["embed"] == 1 and calls.n["residual_norm"] == 4
    assert got.keys() == want.keys()
    # Rounding differences through two layers: fp32 sums in another order; bf16 activations rounded at other places.
    bar = 2e-5 if dtype == torch.float32 else 4e-2
    for name, g in got.items():
        diff, size = (g.double() - want[name].double()).norm(), want[name].double().norm()
        gate = next((w for k, w in _GATES.items() if name.endswith(k)), None)
        if gate is not None:
            # One number: a sum of terms c_t over the tokens that cancel, off by bar of the sum of |c_t|. The gate's
            # weight has the gradient sum of c_t x_t with |x_t| = 16 (256 normalised columns), so that the sum of
            # |c_t| is at least its norm / 16. In bf16 the terms' own roundings leave nothing of the number.
            if dtype == torch.bfloat16:
                continue
            size = torch.maximum(size, want[name[:name.rindex("attn.") + 5] + gate].double().norm() / 16)
        assert diff <= bar * size + 1e-12, name
    assert abs(out["loss"].item() - plain["loss"].item()) <= (1e-5 if dtype == torch.float32 else 2e-2) * loss.item()


def test_training_gradients_are_the_same_bits_again():
    model = _model(torch.bfloat16)
    ids, labels = _batch()
    ids[:] = ids[0, :1]  # one token everywhere
    a, b = _grads(model, ids, labels)[1], _grads(model, ids, labels)[1]
    name = "model.embeddings.weight"
    assert torch.equal(a[name], b[name]) and a[name].abs().sum() > 0


def test_hooks_and_replaced_modules_run(monkeypatch):
    ids, labels = _batch()
    want = _grads(_model(torch.float32), ids, labels)[1]
    for pick in (lambda m: m.model.layers[0], lambda m: m.model.layers[1].mlp_norm, lambda m: m.model.norm,
                 lambda m: m.model.embeddings):
        model, seen = _model(torch.float32), []
        pick(model).register_forward_hook(lambda mod, args, out: seen.append(mod) and None)
        got = _grads(model, ids, labels)[1]
        assert len(seen) == 1
        for name, g in got.items():
            if not name.endswith(tuple(_GATES)):
                assert (g - want[name]).norm() <= 2e-5 * want[name].norm() + 1e-12, name
    model = _model(torch.float32)
    calls = _Calls(monkeypatch, "embed_grad", "residual_norm_grad")
    model.model.embeddings.weight.requires_grad_(False)
    _grads(model, ids, labels)
    assert calls.n == dict(embed_grad=0, residual_norm_grad=4)


def test_loss_without_gradients(monkeypatch):
    model = _model(torch.bfloat16)
    ids, labels = _batch()
    calls = _Calls(monkeypatch, "token_loss")
    with torch.no_grad():
        out = model(ids, labels=labels)
        loss = F.cross_entropy(out["logits"][:, :-1].double().reshape(-1, V), labels[:, 1:].reshape(-1), ignore_index=-100)
    assert calls.n["token_loss"] == 1 and abs(out["loss"].item() - loss.item()) <= 2.0**-18 * loss.item()
    with torch.no_grad():
        assert model(ids[:, :1], labels=labels[:, :1])["loss"].isnan()  # no label to predict


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_score(dtype):
    model = _model(dtype).eval()
    ids, _ = _batch(2, 64)
    lengths = torch.tensor([64, 41]).cuda()
    mask = (torch.arange(64, device="cuda")[None] < lengths[:, None]).long()
    for m in (None, mask):
        got = model.score(ids, top_k=4, attention_mask=m)
        with torch.no_grad():
            logits = model(ids, attention_mask=m)["logits"][:, :-1].cpu()
        tokens = ids[:, 1:].cpu()
        if m is not None:
            tokens = tokens.masked_fill(m[:, 1:].cpu() == 0, -100)
        ref = lm.logprobs(logits.reshape(-1, V).double(), tokens.reshape(-1), 4)
        assert got.logprob.shape == (2, 63) and got.top_ids.shape == (2, 63, 4) and not got.logprob.requires_grad
        lm.assert_within(got.logprob.reshape(-1), *ref["logprob"], "logprob")
        lm.assert_within(got.entropy.reshape(-1), *ref["entropy"], "entropy")
        lm.assert_within(got.top_logprobs.reshape(-1, 4), *ref["top"], "top")
        assert torch.equal(got.top_ids.reshape(-1, 4).cpu(), ref["ids"])
