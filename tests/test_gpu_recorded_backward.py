"""Recorded and batched backward passes of the joins between a model's blocks,
where one input was computed from another, and forward-mode derivatives and
traces of the operators around the blocks."""

import pytest
import torch

from cyclic_flow_attention import CyclicFlowAttentionConfig, CyclicFlowAttentionForCausalLM, ops
from cyclic_flow_attention.models.cyfa import modeling_cyfa

pytestmark = pytest.mark.gpu


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("make_y", [torch.tanh, lambda x: x])
def test_join_of_a_block_computed_from_its_residual(make_y):
    cots = _randn(3, 3, 5, 24)
    x = _randn(1, 5, 24).cuda().requires_grad_(True)
    w = (1 + 0.1 * _randn(2, 24)).cuda().requires_grad_(True)
    s, h = ops.residual_norm(x, make_y(x), w, gate=2 * x, scale=0.5, eps=1e-3)
    plain = torch.autograd.grad([s, h], [x, w], [cots[0].cuda(), cots[1].cuda()], retain_graph=True)
    recorded = torch.autograd.grad([s, h], [x, w], [cots[0].cuda(), cots[1].cuda()], create_graph=True)
    batched = torch.autograd.grad(h, [x], cots.cuda(), is_grads_batched=True, retain_graph=True)[0]
    again = torch.autograd.grad(h, [x], cots[2].cuda(), retain_graph=True)[0]
    z, v = x.detach().double().cpu().requires_grad_(True), w.detach().double().cpu().requires_grad_(True)
    rs = z + 0.5 * make_y(z) * torch.sigmoid(2 * z)
    rh = rs * (rs.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * v
    want = torch.autograd.grad([rs, rh], [z, v], [cots[0].double(), cots[1].double()], retain_graph=True)
    for got in (plain, recorded):
        for a, b in zip(got, want):  # fp32 through two reductions of 24 terms
            assert (a.double().cpu() - b).abs().max() <= 2.0**-18 * b.abs().max()
    for i in range(3):
        (b,) = torch.autograd.grad(rh, [z], cots[i].double(), retain_graph=True)
        for a in (batched[i],) + ((again,) if i == 2 else ()):
            assert (a.double().cpu() - b).abs().max() <= 2.0**-18 * b.abs().max()


def test_model_gradients_of_a_recorded_pass(monkeypatch):
    """The first-order gradients of a pass with create_graph, against one without
    and against the joins in torch operations."""
    torch.manual_seed(3)
    config = CyclicFlowAttentionConfig(hidden_size=256, num_heads=1, head_dim=256, num_hidden_layers=2, vocab_size=301,
                                       intermediate_size=512, num_slots=128)
    model = CyclicFlowAttentionForCausalLM(config).cuda()
    ids = torch.randint(0, 301, (2, 70), generator=torch.Generator().manual_seed(1)).cuda()
    # (the gates' parameters are sums that cancel over the tokens; the other gradients would show a path counted twice)
    params = {n: p for n, p in model.named_parameters() if not n.endswith(("dt_bias", "A_log", "b_proj.bias", "d_proj.bias"))}

    def grads(recorded):
        loss = model(ids, labels=ids)["loss"]
        return [g.detach() for g in torch.autograd.grad(loss, list(params.values()), create_graph=recorded)]

    want = grads(False)
    got = grads(True)
    monkeypatch.setattr(modeling_cyfa, "hip_autograd_ok", lambda *tensors: False)
    plain = grads(True)
    for name, a, b, c in zip(params, got, want, plain):
        for other in (b, c):  # fp32 sums in another order through two layers
            assert (a.double() - other.double()).norm() <= 2e-5 * other.double().norm() + 1e-12, name


def test_forward_mode_derivatives_and_traces():
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x, d = _randn(1, 5, 40).cuda(), _randn(2, 5, 40).cuda()
    t, w = torch.tensor([1, 39, 0, 7, 7]).cuda(), torch.ones(40, device="cuda")

    def calls(x):
        r = ops.token_logprobs(x, t, top_k=3)
        return (r.logprob, r.entropy, r.top_logprobs, ops.token_loss(x, t), ops.embed_tokens(t % 5, x),
                *ops.residual_norm(x, 2 * x, w))

    h = 2.0**-7
    with torch.no_grad():
        high, low, at = calls(x + h * d), calls(x - h * d), calls(x)  # the kernels
        with forward_ad.dual_level():
            outs = [forward_ad.unpack_dual(o) for o in calls(forward_ad.make_dual(x, d))]
        traced = make_fx(calls)(_randn(3, 5, 40).cuda())(x)
        ids = [ops.token_logprobs(x + e * d, t, top_k=3).top_ids for e in (h, -h)]
    for i, (a, b, c, o, g) in enumerate(zip(high, low, at, outs, traced)):
        off = (o.tangent - (a - b) / (2 * h)).abs()
        if i == 2:  # (alternatives that change places between the two points: their quotient is no derivative)
            assert (ids[0] != ids[1]).sum() == 2
            off = off[ids[0] == ids[1]]
        # third derivatives of order ten times h^2, fp32 values of order ten over h
        assert off.max() <= 20 * h * h + 60 * 2.0**-24 / h
        assert (o.primal - c).abs().max() <= 2.0**-18 * (1 + c.abs().max())
        assert (g - c).abs().max() <= 2.0**-18 * (1 + c.abs().max())
