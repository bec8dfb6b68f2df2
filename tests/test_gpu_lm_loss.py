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
    loss = model._loss(torch.zeros(2, 0, 256, device="cuda"), logits, torch.zeros(2, 0, dtype=torch.int64, device="cuda"))
    assert loss.isnan() and torch.autograd.grad(loss, [logits])[0].shape == logits.shape and not launches


EDITS = {"no_grad": lambda x: x.detach().mul_(0.5), "recorded": lambda x: x.div_(3.0), "masked": lambda x: x[0].fill_(float("-inf"))}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("edit", EDITS)
def test_logits_edited_before_the_backward_pass(launches, dtype, edit):
    """The gradients are those of the logits that the loss saw."""
    model, ids = _model(dtype), _ids()
    params = list(model.parameters())

    def grads(change, **kwargs):
        out = model(ids, labels=ids)
        if change:
            change(out["logits"])
        return torch.autograd.grad(out["loss"], params, **kwargs)

    want = grads(None)
    for kwargs in ({}, {"retain_graph": True}, {"create_graph": True}):
        for name, a, b in zip(dict(model.named_parameters()), grads(EDITS[edit], **kwargs), grads(None, **kwargs)):
            if kwargs.get("create_graph"):
                # the recorded lookup's gradient adds up to 80 rows by fp32 atomics, in no fixed order, before it rounds to the dtype
                assert (a.double() - b.double()).norm() <= (2.0**-16 if dtype == torch.float32 else 2.0**-7) * b.double().norm(), name
            else:
                assert torch.equal(a, b), name
    assert len(launches) == 7 and all(torch.equal(a, b) for a, b in zip(want, grads(None)))


def test_edited_logits_whose_source_was_edited_too():
    model, ids = _model(torch.float32), _ids()
    model.lm_head.weight.requires_grad_(False)
    out = model(ids, labels=ids)
    out["logits"].detach().zero_()
    model.lm_head.weight.mul_(2)
    with pytest.raises(RuntimeError, match="edited in place|modified by an inplace"):
        out["loss"].backward()


def test_saved_tensor_hooks_of_the_caller_stay_in_charge(launches):
    model, ids = _model(torch.float32), _ids()
    want = torch.autograd.grad(model(ids, labels=ids)["loss"], [model.lm_head.weight])[0]
    with torch.autograd.graph.save_on_cpu():
        loss = model(ids, labels=ids)["loss"]
    assert torch.equal(torch.autograd.grad(loss, [model.lm_head.weight])[0], want)
    with torch.autograd.graph.disable_saved_tensors_hooks("not here"):
        loss = model(ids, labels=ids)["loss"]
    assert torch.equal(torch.autograd.grad(loss, [model.lm_head.weight])[0], want)
    assert len(launches) == 3


def test_replaced_heads_keep_the_torch_operations(launches):
    model, ids = _model(torch.float32), _ids()
    want = torch.autograd.grad(model(ids, labels=ids)["loss"], [model.lm_head.weight])[0]
    seen = []
    model.lm_head.register_forward_hook(lambda mod, args, out: seen.append(out) and None)
    out = model(ids, labels=ids)
    out["logits"].detach().zero_()
    got = torch.autograd.grad(out["loss"], [model.lm_head.weight])[0]
    assert len(seen) == 1 and len(launches) == 1 and (got - want).norm() <= 2e-5 * want.norm()
    with torch.no_grad():
        model(ids, labels=ids)
    assert len(launches) == 2
