"""The model's loss on the HIP path: every dtype with and without gradients, and
what may happen to the logits before the backward pass."""

import pytest
import torch
import torch.nn.functional as F

from cyclic_flow_attention import CyclicFlowAttentionConfig, CyclicFlowAttentionForCausalLM, _native

pytestmark = pytest.mark.gpu

V = 301


def _model(dtype):
    torch.manual_seed(3)
    config = CyclicFlowAttentionConfig(hidden_size=256, num_heads=1, head_dim=256, num_hidden_layers=1, vocab_size=V,
                                       intermediate_size=512, num_slots=128)
    model = CyclicFlowAttentionForCausalLM(config).cuda()
    return model if dtype == torch.float32 else model.to(dtype) if dtype == torch.float16 else model.to_bfloat16()


def _ids(B=2, T=40):
    return torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(1)).cuda()


@pytest.fixture
def launches(monkeypatch):
    n = []
    call = _native.token_loss
    monkeypatch.setattr(_native, "token_loss", lambda *args, **kwargs: n.append(1) or call(*args, **kwargs))
    return n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_loss_without_gradients_of_every_dtype(launches, dtype):
    model, ids = _model(dtype), _ids()
    labels = ids.clone()
    labels[1, 30:] = -100
    for context in (torch.no_grad(), torch.inference_mode()):
        with context:
            out = model(ids, labels=labels)
        want = F.cross_entropy(out["logits"][:, :-1].double().reshape(-1, V), labels[:, 1:].reshape(-1))
        assert abs(out["loss"].item() - want.item()) <= 2.0**-18 * want.item()
        with context:
            labels[0, 3] = V  # as in a training step
            assert model(ids, labels=labels)["loss"].isnan()
        labels[0, 3] = 5
    assert len(launches) == 4


def test_sizes_past_the_operators_keep_the_torch_operations(launches, monkeypatch):
    model, ids = _model(torch.float32), _ids()
    want = model(ids, labels=ids)["loss"]
    grads = torch.autograd.grad(want, [model.model.embeddings.weight])
    assert len(launches) == 1
    monkeypatch.setattr(_native, "LOGPROBS_MAX_V", V - 1)
    embeds = []
    for name, largest in (("EMBED_MAX_V", V - 1), ("EMBED_MAX_D", 255), ("EMBED_MAX_N", 79)):
        with monkeypatch.context() as m:
            m.setattr(_native, name, largest)
            m.setattr(_native, "embed", lambda *args: embeds.append(1))
            loss = model(ids, labels=ids)["loss"]
            (got,) = torch.autograd.grad(loss, [model.model.embeddings.weight])
        assert abs(loss.item() - want.item()) <= 2.0**-16 * want.item()
        assert (got - grads[0]).norm() <= 2e-5 * grads[0].norm()
    assert len(launches) == 1 and not embeds


def test_loss_of_no_tokens(launches):
    model = _model(torch.float32)
    logits = torch.zeros(2, 0, V, device="cuda", requires_grad=True)
    loss = model._loss(logits, torch.zeros(2, 0, dtype=torch.int64, device="cuda"))
    assert loss.isnan() and torch.autograd.grad(loss, [logits])[0].shape == logits.shape and not launches
