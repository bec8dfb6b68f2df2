"""The operators on a model's logits (ops.adjust_logits, sample_tokens,
distill_loss) against float64 on the CPU, at sizes, masks and values where they
can go wrong; the bounds are derived in logits_bounds."""

import math

import numpy as np
import pytest
import torch

import lm_bounds as lm
import logits_bounds as lb

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def _ops():
    from cyclic_flow_attention import ops

    return ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(shape, generator=_gen(seed))


def _rand(seed, *shape):
    return torch.rand(shape, generator=_gen(seed))


def _randint(seed, n, *shape):
    return torch.randint(0, n, shape, generator=_gen(seed))


def _bits(allowed):
    """bool [rows, V] as int32 words, token j at bit j % 32 of word j // 32."""
    rows, V = allowed.shape
    full = torch.zeros(rows, (V + 31) // 32 * 32, dtype=torch.int64)
    full[:, :V] = allowed
    words = (full.view(rows, -1, 32) << torch.arange(32)).sum(-1)
    return (words - ((words >> 31) << 32)).int()


def _cuda(t):
    return tuple(map(_cuda, t)) if isinstance(t, tuple) else t.cuda() if isinstance(t, torch.Tensor) else t


# ---------------------------------------------------------------- adjust_logits


def _adjust_case(seed, rows, V, L, dtype, wide=True, bias=True, tokens=5, mask="bool", train=True):
    x = (_randn(seed, rows, V) * 4).to(dtype)
    x[0, ::3] = 0.0
    history = (_rand(seed + 1, rows, L) ** 3 * (V + 2)).long() - 1  # some outside [0, V)
    kw = dict(history=history if wide else history.int(), lengths=_randint(seed + 2, L + 3, rows) - 1,
              prompt_lengths=_randint(seed + 3, L + 2, rows), repetition=0.8 + _rand(seed + 4, rows),
              presence=_randn(seed + 5, rows), frequency=_randn(seed + 6, rows))
    kw["lengths"][0] = 0
    kw["prompt_lengths"][-1] = 0
    kw["lengths"][-1] = L
    if bias:
        kw["bias"] = _randn(seed + 7, V)
    if tokens:
        ids = _randint(seed + 8, V + 1, rows, tokens)
        ids[:, -1] = ids[:, 0]  # the same token twice
        kw["token_bias"] = (ids, _randn(seed + 9, rows, tokens))
    allowed = None
    if mask:
        allowed = _rand(seed + 10, rows, V) < 0.7
        if rows > 1:
            allowed[1] = False  # nothing left
        kw["allowed"] = allowed if mask == "bool" else _bits(allowed)
    return x, kw, allowed


def _adjust_ref(x, kw, allowed, dy=None):
    rows, V = x.shape
    tokens = None
    if "token_bias" in kw:
        tokens = [list(zip(i.tolist(), v.tolist())) for i, v in zip(*kw["token_bias"])]
    bias = kw["bias"].double().expand(rows, V) if "bias" in kw else None
    L = kw["history"].shape[1]
    lists = [kw[n].double().tolist() for n in ("repetition", "presence", "frequency")]
    return lb.adjust(x.double(), kw["history"].tolist(), [min(n, L) for n in kw["lengths"].tolist()], kw["prompt_lengths"].tolist(), *lists,
                     bias, tokens, allowed, x.dtype, None if dy is None else dy.double())


@pytest.mark.parametrize("rows,V,L,dtype,wide,bias,tokens,mask", [
    (1, 1, 1, F32, True, False, 0, ""), (2, 7, 9, BF, True, True, 3, "bool"), (3, 33, 2, F16, False, False, 2, "bits"),
    (9, 257, 100, F32, False, True, 0, "bits"), (5, 1023, 700, BF, True, False, 9, "bool"), (20, 2051, 33, F16, True, True, 0, ""),
    (1, 32000, 513, BF, True, False, 17, "bits"), (3, 50001, 4097, F32, True, True, 300, "bool"), (9, 8193, 1, BF, False, True, 1, "bits"),
    (70, 40000, 65, BF, True, True, 1024, "bits"), (3, 9001, 20000, BF, True, False, 40, "bool"), (260, 33000, 40, F16, True, False, 2, ""),
    (4, 300, 17000, F32, False, True, 0, "bits"), (129, 66001, 4100, BF, False, False, 3, "bits")])
def test_adjust(rows, V, L, dtype, wide, bias, tokens, mask):
    x, kw, allowed = _adjust_case(V + L, rows, V, L, dtype, wide, bias, tokens, mask)
    dy = (_randn(V, rows, V)).to(dtype)
    xg = x.cuda().requires_grad_(True)
    y = _ops().adjust_logits(xg, **{n: _cuda(t) for n, t in kw.items()})
    (dx,) = torch.autograd.grad(y, [xg], dy.cuda())
    want, grad = _adjust_ref(x, kw, allowed, dy)
    assert y.dtype == dx.dtype == dtype
    lm.assert_within(y, *want, "y")
    lm.assert_within(dx, *grad, "dx")
    with torch.no_grad():
        args = {n: _cuda(t) for n, t in kw.items()}
        assert torch.equal(_ops().adjust_logits(x.cuda(), **args).view(torch.uint8), y.detach().view(torch.uint8))
        own = x.cuda()
        assert _ops().adjust_logits(own, **args, out=own) is own and torch.equal(own.view(torch.uint8), y.detach().view(torch.uint8))


def test_adjust_of_nothing_and_of_single_rows():
    ops, x = _ops(), _randn(1, 3, 50).cuda()
    assert torch.equal(ops.adjust_logits(x), x)
    assert torch.equal(ops.adjust_logits(x, torch.zeros(3, 0, dtype=torch.int64).cuda(), repetition=2.0), x)
    assert ops.adjust_logits(x[:0], torch.zeros(0, 4, dtype=torch.int64).cuda()).shape == (0, 50)
    one = ops.adjust_logits(x[0], torch.tensor([4, 4, 60, -1]).cuda(), frequency=1.0, repetition=2.0,
                            allowed=torch.arange(50).cuda() != 7)
    want = x[0].clone()
    want[4] = (want[4] / 2 if want[4] > 0 else want[4] * 2) - 2
    want[7] = -INF
    assert torch.equal(one, want)
    assert x._version == 0 and ops.adjust_logits(x, bias=torch.ones(50).cuda(), out=x)._version == 1


def test_adjust_of_values_past_the_finite():
    """Infinities and NaN in masked places, beside them, and in places that nothing touches."""
    x = _randn(1, 4, 64)
    x[0, 3], x[0, 4], x[0, 5] = NAN, INF, -INF
    x[1] = torch.finfo(F32).min
    x[2, 9] = NAN
    allowed = torch.ones(4, 64, dtype=torch.bool)
    allowed[0, 3:5] = False
    history = torch.tensor([[3, 4, 5], [0, 1, 2], [1, 1, 1], [0, 0, 0]])
    xg = x.cuda().requires_grad_(True)
    y = _ops().adjust_logits(xg, history.cuda(), repetition=2.0, presence=1.0, allowed=allowed.cuda())
    out = y.detach().cpu()
    assert out[0, 3] == out[0, 4] == out[0, 5] == -INF and (out[1, :3] == -INF).all() and (out[1, 3:] == x[1, 3:]).all()
    assert out[2, 9].isnan() and torch.equal(out[3, 1:], x[3, 1:])
    dy = torch.full((4, 64), 3.0)
    dy[0, 3] = NAN  # of a token that is not allowed
    (dx,) = torch.autograd.grad(y, [xg], dy.cuda())
    assert dx[0, 3] == dx[0, 4] == 0 and dx[0, 5] == 6 and (dx[1, :3] == 6).all() and (dx[1, 3:] == 3).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_adjust_of_views_and_broadcast_options(dtype):
    ops, B, T, V, L = _ops(), 3, 6, 1003, 40
    base = (_randn(5, B, T + 1, V + 5) * 3).to(dtype)
    ids = _randint(6, V, B, L)
    lengths = torch.arange(T) + L - T
    repetition, bias = 1 + _rand(7, B, 1), _randn(8, T, V)
    mask = _rand(9, B, 1, V) < 0.5
    for make in (lambda t: t[:, :-1, 3:V + 3], lambda t: t[:, 1:, :V], lambda t: t.transpose(0, 1)[1:].transpose(0, 1)[..., 5:],
                 lambda t: t[..., :V].permute(2, 0, 1).contiguous().permute(1, 2, 0)[:, :-1]):
        x = make(base)
        xg = make(base.cuda()).detach().requires_grad_(True)
        y = ops.adjust_logits(xg, ids[:, None].cuda(), lengths.cuda(), torch.tensor(5).cuda(), repetition=repetition.cuda(), frequency=0.5,
                              bias=bias.cuda(), token_bias=(torch.tensor([1, 3]).cuda(), torch.tensor([0.5, -1.0]).cuda()),
                              allowed=mask.cuda())
        dy = _randn(3, B, T, V).to(dtype)
        (dx,) = torch.autograd.grad(y, [xg], dy.cuda().transpose(0, 1).contiguous().transpose(0, 1))
        flat = lambda t: t.expand(B, T, *t.shape[2:]).reshape(B * T, *t.shape[2:])  # noqa: E731
        want, grad = lb.adjust(flat(x).double(), flat(ids[:, None]).tolist(), lengths.repeat(B).tolist(), [5] * (B * T),
                               flat(repetition).tolist(), [0.0] * (B * T), [0.5] * (B * T), bias.repeat(B, 1).double(),
                               [[(1, 0.5), (3, -1.0)]] * (B * T), flat(mask), dtype, flat(dy).double())
        lm.assert_within(y.reshape(-1, V), *want, "y")
        lm.assert_within(dx.reshape(-1, V), *grad, "dx")
        own = base.cuda()
        if make(own).stride(-1) == 1:  # in place in a strided view: its surroundings stay
            rest = torch.ones_like(base)
            make(rest).zero_()
            ops.adjust_logits(make(own), bias=bias.cuda(), out=make(own))
            assert torch.equal(own.cpu() * rest, base * rest)
            lm.assert_within(make(own).reshape(-1, V), *lb.adjust(flat(x).double(), None, [0] * 18, [0] * 18, [1.0] * 18, [0.0] * 18,
                                                                  [0.0] * 18, bias.repeat(B, 1).double(), None, None, dtype), "in place")


def test_adjust_gradient_is_the_difference_quotient():
    x, h = _randn(1, 3, 40).double(), 2.0**-4
    history = torch.tensor([[1, 2], [5, 5], [0, 39]]).cuda()

    def value(z):
        y = _ops().adjust_logits(z.float().cuda(), history, repetition=1.25, presence=0.5, frequency=0.25)
        return (y.double().cpu() * _randn(2, 3, 40).double()).sum()

    xg = x.float().cuda().requires_grad_(True)
    y = _ops().adjust_logits(xg, history, repetition=1.25, presence=0.5, frequency=0.25)
    (dx,) = torch.autograd.grad(y, [xg], _randn(2, 3, 40).cuda())
    x = x.float().double()
    for r, c in ((0, 1), (0, 7), (1, 5), (2, 39), (2, 0)):
        assert abs(x[r, c]) > h  # on one side of zero
        d = torch.zeros_like(x)
        d[r, c] = h
        assert abs((value(x + d) - value(x - d)) / (2 * h) - dx[r, c].item()) < 200 * 2.0**-24 * 4 / h


def test_adjust_recorded_backward_and_edited_logits():
    x, history = _randn(3, 2, 30), torch.tensor([[1, 1, 4], [0, 29, 3]])
    xg, dy = x.cuda().requires_grad_(True), _randn(4, 2, 30).cuda().requires_grad_(True)
    allowed = (torch.arange(30) % 4 != 1).cuda()
    y = _ops().adjust_logits(xg, history.cuda(), repetition=1.5, frequency=0.5, allowed=allowed)
    (dx,) = torch.autograd.grad(y, [xg], dy, create_graph=True)
    (plain,) = torch.autograd.grad(y, [xg], dy.detach(), retain_graph=True)
    assert torch.equal(dx, plain)
    (ddy,) = torch.autograd.grad(dx.sum(), [dy])
    _, (slope, bound) = lb.adjust(x.double(), history.tolist(), [3, 3], [0, 0], [1.5] * 2, [0.0] * 2, [0.5] * 2, None, None,
                                  allowed.cpu().expand(2, 30), F32, torch.ones(2, 30).double())
    lm.assert_within(ddy, slope, bound, "ddy")
    with torch.no_grad():
        xg.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, [xg], dy.detach())


# ---------------------------------------------------------------- sample_tokens


def _check_choice(x, u, got, T=1.0, k=0, p=1.0, least=0.0, what=""):
    at = lambda v, r: float(v[r]) if isinstance(v, torch.Tensor) else v  # noqa: E731
    rows = x.double().numpy()
    for r in range(x.shape[0]):
        want = lb.choice(rows[r], float(u[r]), at(T, r), int(at(k, r)), at(p, r), at(least, r))
        assert got.ids[r].item() == want[0], (what, r, got.ids[r].item(), want)
        assert abs(got.logprob[r].item() - want[1]) <= 2.0**-23 * (1 + abs(want[1])), (what, r, got.logprob[r].item(), want)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows,V,T,k,p,least", [
    (1, 1, 1.0, 0, 1.0, 0.0), (5, 2, 0.5, 1, 1.0, 0.0), (9, 7, 1.0, 3, 0.9, 0.0), (12, 64, 0.01, 0, 1.0, 0.0), (40, 255, 3.0, 0, 0.5, 0.0),
    (6, 1000, 1.0, 999, 1.0, 0.1), (7, 2051, 0.8, 50, 0.95, 0.0), (30, 4096, 100.0, 2000, 0.99, 0.0), (5, 32000, 0.8, 0, 0.95, 0.0),
    (4, 32000, 1.0, 0, 1.0, 0.05), (3, 32003, 1.3, 20000, 0.7, 0.0), (3, 50001, 1.0, 40, 1.0, 0.02), (300, 513, 1.0, 20, 0.8, 0.01),
    (2, 70001, 1.0, 0, 0.9, 0.0), (2, 131072, 1.0, 0, 1.0, 0.0), (2, 150000, 0.7, 5000, 0.99, 0.0)])
def test_sample(rows, V, T, k, p, least, dtype):
    x = (_randn(rows + V, rows, V) * 3).to(dtype)  # 16-bit logits of a large vocabulary hold many equal ones
    u = _rand(V, rows)
    got = _ops().sample_tokens(x.cuda(), u.cuda(), temperature=T, top_k=k, top_p=p, min_p=least)
    assert got.ids.dtype == torch.int64 and got.logprob.dtype == F32
    _check_choice(x, u, got, T, k, p, least)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_sample_with_settings_of_each_row(dtype):
    rows, V = 64, 3001
    x = (_randn(1, rows, V) * 3).to(dtype)
    x[10:20] = x[10:20].clamp(max=2.0)  # many equal largest
    u = _rand(2, rows).double()
    T, k, p, least = 2 * _rand(3, rows), _randint(4, 60, rows), 0.3 + 0.8 * _rand(5, rows), 0.2 * _rand(6, rows) - 0.1
    T[3], T[4], k[5], p[6] = 0.0, -1.0, V + 5, 2.0
    got = _ops().sample_tokens(x.cuda(), u.cuda(), temperature=T.cuda(), top_k=k.cuda().int(), top_p=p.cuda(), min_p=least.cuda())
    _check_choice(x, u, got, T, k, p, least)


@pytest.mark.parametrize("V,dtype", [(50001, BF), (50001, F32), (40000, F16), (131073, BF)])
def test_sample_of_few_wide_rows_with_settings_of_each(V, dtype):
    """Rows that are shared out, of which some have a top_k that one wave handles:
    thousands of equal elements behind a few larger ones, rows of one value, rows
    without probabilities, a vocabulary that ends inside a vector."""
    rows = 12
    x = (_randn(V, rows, V) * 2).clamp(max=9.0).to(dtype)
    x[0:6] = torch.where(torch.arange(V) % 3 == 0, 1.0, -2.0 - torch.arange(V) % 2).to(dtype)
    x[0:6, 17:20] = torch.tensor([3.0, 2.0, 2.5]).to(dtype)
    x[6, V // 2:] = -INF
    x[7] = 0.5
    x[8, 4000] = NAN
    x[9] = -INF
    x[10, 39999], x[10, 4] = INF, INF
    u = _rand(V + 1, rows)
    k = torch.tensor([50, 128, 129, 0, 1, 20000, 64, 100, 5, 5, 5, 0])
    p = torch.tensor([1.0, 0.9, 0.8, 0.5, 1.0, 0.99, 1.0, 0.7, 0.9, 0.9, 0.9, 0.9])
    least = torch.tensor([0.0, 0.0, 0.05, 0.2, 0.0, 0.0, 0.1, 0.0, 0.0, 0.0, 0.0, 0.0])
    T = torch.tensor([1.0, 2.0, 0.7, 1.0, 1.0, 1.5, 1.0, 1.0, 1.0, 1.0, 1.0, 0.8])
    got = _ops().sample_tokens(x.cuda(), u.cuda(), temperature=T.cuda(), top_k=k.cuda(), top_p=p.cuda(), min_p=least.cuda())
    fine = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 11])
    _check_choice(x[fine], u[fine], type(got)(got.ids.cpu()[fine], got.logprob.cpu()[fine]), T[fine], k[fine], p[fine], least[fine])
    assert got.ids[8:11].tolist() == [4000, 0, 4] and got.logprob[8:11].isnan().all()


@pytest.mark.parametrize("rows,V,dtype", [(2100, 3, F32), (4111, 37, BF), (2309, 1022, F16), (1031, 8205, BF), (1030, 8194, F32), (5, 8191, BF)])
def test_sample_of_whole_rows_in_turn(rows, V, dtype):
    """More rows than workgroups, which take them one after another: ordinary rows
    beside those without probabilities, greedy ones, rows of one value."""
    x = (_randn(V, rows, V) * 3).to(dtype)
    kind = _randint(rows, 8, rows)
    kind[-3:] = torch.tensor([0, 1, 7])
    x[kind == 0, V // 2] = NAN
    x[kind == 1] = -INF
    x[kind == 2, V - 1] = INF
    x[kind == 3] = 0.25
    x[kind == 4, : V - 1] = -INF
    u, T = _rand(1, rows), 0.2 + 2 * _rand(2, rows)
    T[kind == 5] = 0.0
    for least in (0.0, 0.3 * _rand(3, rows) - 0.05):
        got = _ops().sample_tokens(x.cuda(), u.cuda(), temperature=T.cuda(), min_p=least.cuda() if isinstance(least, torch.Tensor) else least)
        fine = (kind > 2).nonzero()[:, 0]
        own = least[fine] if isinstance(least, torch.Tensor) else least
        _check_choice(x[fine], u[fine], type(got)(got.ids.cpu()[fine], got.logprob.cpu()[fine]), T[fine], 0, 1.0, own, (rows, V))
        for k, at in ((0, V // 2), (1, 0), (2, V - 1)):
            assert (got.ids.cpu()[kind == k] == at).all() and got.logprob.cpu()[kind == k].isnan().all()
    again = _ops().sample_tokens(x[7:].cuda(), u[7:].cuda(), temperature=T[7:].cuda(), min_p=least[7:].cuda())  # others' turns
    assert torch.equal(again.ids, got.ids[7:]) and torch.equal(again.logprob.nan_to_num(9.0), got.logprob[7:].nan_to_num(9.0))


def test_sample_at_the_borders():
    """Weights whose sums are exact: which token a number on a border takes, ties
    by the lower id, the first kept and the last number below one."""
    x = torch.zeros(8, 1000)
    x[:, 500:] = -INF
    u = torch.tensor([0.0, 0.25, 0.5, 0.998, 1 - 2.0**-24, 0.002, 0.5, 0.5])
    got = _ops().sample_tokens(x.cuda(), u.cuda())
    assert got.ids.tolist() == [0, 125, 250, 499, 499, 1, 250, 250] or got.ids.tolist()[3] in (498, 499)
    _check_choice(x, u, got)
    got = _ops().sample_tokens(x.cuda(), u.cuda(), top_p=0.5)  # exactly half of the mass: 250 tokens
    assert got.ids.tolist()[:3] == [0, 62, 125] and got.ids[4] == 249
    got = _ops().sample_tokens(x.cuda(), u.cuda(), top_k=4, top_p=0.75)
    assert got.ids[:3].tolist() == [0, 0, 1] and got.ids[4] == 2
    got = _ops().sample_tokens(x.cuda(), u.cuda(), top_k=4, min_p=1.0)
    assert got.ids[4] == 3 and abs(got.logprob[4].item() + math.log(4)) < 1e-6
    out = torch.tensor([-0.5, 1.0, 7.0, NAN, INF, -INF, 0.0, 0.5])  # numbers outside [0, 1) take the ends
    got = _ops().sample_tokens(x.cuda(), out.cuda())
    assert got.ids.tolist() == [0, 499, 499, 0, 499, 0, 0, 250]
    wide = torch.tensor([0.3, 1 - 2.0**-53], dtype=torch.float64)
    got = _ops().sample_tokens(x[:2].cuda(), wide.cuda())
    assert got.ids.tolist() == [150, 499]


def test_sample_of_rows_all_alike():
    """Rows of one value, of two, of the type's lowest: ties by the thousand."""
    for dtype in (BF, F32):
        for V in (1, 9, 1024, 5000, 32000, 100003):
            x = torch.full((6, V), 1.5).to(dtype)
            x[1] = torch.finfo(dtype).min
            x[2, V // 2:] = -2.0
            x[3, ::2] = torch.finfo(dtype).min
            x[4] = 0.0
            x[4, ::2] = -0.0
            x[5, V // 3:] = -INF if V // 3 else 1.5
            u = _rand(V, 6)
            for T, k, p in ((1.0, 0, 1.0), (1.0, 0, 0.6), (0.7, max(1, V // 3), 1.0), (2.0, 700, 0.9), (1e30, 0, 0.5)):
                got = _ops().sample_tokens(x.cuda(), u.cuda(), temperature=T, top_k=k, top_p=p)
                _check_choice(x, u, got, T, k, p, 0.0, (dtype, V, T, k, p))


def test_sample_of_rows_without_probabilities():
    x = _randn(2, 7, 3000)
    x[0] = -INF
    x[1, 70], x[1, 2999] = NAN, NAN
    x[2, 9], x[2, 5] = INF, INF
    x[3, 2500], x[3, 200] = NAN, INF
    x[4, 1:] = -INF
    x[5] = -INF
    x[5, 2998] = -3e38
    u = _rand(1, 7)
    for kw in ({}, dict(top_k=5, top_p=0.5, min_p=0.1), dict(temperature=0.0)):
        got = _ops().sample_tokens(x.cuda(), u.cuda(), **kw)
        assert got.ids[:6].tolist() == [0, 70, 5, 2500, 0, 2998]
        assert got.logprob[:4].isnan().all() and (got.logprob[4:6] == 0).all()
    assert got.ids[6].item() == int(x[6].argmax()) and got.logprob[6] == 0


def test_sample_of_few_values_far_apart():
    """A spread that overflows, outliers that leave every other element in one
    bin, clusters of thousands within a few steps of each other."""
    V = 40000
    x = _randn(3, 6, V)
    x[0, 7] = 3e38
    x[0, 8] = -3e38
    x[1] = 100 + x[1] * 1e-5
    x[1, 5] = -1e30
    x[2] = 20.0 + (torch.arange(V) % 3).float() * 2.0**-19
    x[3] = -20.0 - (torch.arange(V) // 100).float() * 1e-30
    x[4] = torch.where(torch.arange(V) % 5 == 0, 1e-40, -1e-40)
    x[5, :] = 1.0
    x[5, 1::2] = 1.0 + 2.0**-23
    u = _rand(4, 6)
    for T, k, p in ((1.0, 0, 0.7), (1e-3, 0, 0.9), (1e5, 12345, 0.9), (1.0, 1, 1.0), (1.0, 39999, 1.0), (1e-30, 0, 1.0)):
        got = _ops().sample_tokens(x.cuda(), u.cuda(), temperature=T, top_k=k, top_p=p)
        _check_choice(x, u, got, T, k, p, 0.0, (T, k, p))


@pytest.mark.parametrize("make", [
    lambda x: x[:, :-1], lambda x: x[:, 1::2], lambda x: x[..., 3:-2], lambda x: x.transpose(0, 1),
    lambda x: x[:1].expand(4, -1, -1), lambda x: x[0, 0], lambda x: x[:, :0], lambda x: x[None, :, None], lambda x: x.permute(2, 0, 1)])
def test_sample_of_views(make):
    base = (_randn(5, 3, 6, 1003) * 2).to(BF)
    x, xg = make(base), make(base.cuda())
    u = _rand(1, *x.shape[:-1])
    got = _ops().sample_tokens(xg, u.cuda(), top_k=30, top_p=0.9)
    assert got.ids.shape == got.logprob.shape == u.shape
    flat = type(got)(*(t.reshape(-1).cpu() for t in got))
    _check_choice(x.reshape(-1, x.shape[-1]), u.reshape(-1), flat, 1.0, 30, 0.9)


def test_sample_follows_the_probabilities():
    """Many numbers evenly spaced give each token its share."""
    x = torch.log(torch.tensor([0.1, 0.4, 0.2, 0.3])).double()
    n = 4000
    u = (torch.arange(n).double() + 0.5) / n
    got = _ops().sample_tokens(x.float().expand(n, 4).cuda(), u.cuda())
    assert (torch.bincount(got.ids.cpu(), minlength=4) - torch.tensor([400, 1600, 800, 1200])).abs().max() <= 1
    assert (got.ids.cpu()[1:] >= got.ids.cpu()[:-1]).all()
    again = _ops().sample_tokens(x.float().expand(n, 4).cuda().requires_grad_(True), u.cuda())
    assert torch.equal(again.ids, got.ids) and not again.logprob.requires_grad


# ---------------------------------------------------------------- distill_loss


def _teacher(seed, x, k):
    t = x.double() + _randn(seed, *x.shape)
    top = torch.log_softmax(t, -1).topk(k, -1)
    return top.indices, top.values.float()


def _check_distill(x, ids, values, T, tail, weights, d_loss=1.0, what=""):
    xg = x.cuda().requires_grad_(True)
    w = None if weights is None else weights.cuda()
    loss = _ops().distill_loss(xg, ids.cuda(), values.cuda(), temperature=T, tail=tail, weights=w)
    (dx,) = torch.autograd.grad(loss, [xg], torch.tensor(d_loss).cuda())
    assert loss.dtype == F32 and loss.shape == () and dx.dtype == x.dtype and dx.shape == x.shape
    V, k = x.shape[-1], ids.shape[-1]
    want, grad = lb.distill(x.reshape(-1, V).double(), ids.reshape(-1, k), values.reshape(-1, k).double(), T, tail,
                            None if weights is None else weights.reshape(-1), x.dtype, d_loss)
    lm.assert_within(loss, *want, f"{what} loss")
    lm.assert_within(dx.reshape(-1, V), *grad, f"{what} dx")
    with torch.no_grad():
        again = _ops().distill_loss(x.cuda(), ids.cuda(), values.cuda(), temperature=T, tail=tail, weights=w)
    assert torch.equal(again, loss.detach()) or again.isnan() and loss.isnan()
    return dx


@pytest.mark.parametrize("rows,V,k,dtype,T,tail", [
    (3, 1, 1, F32, 1.0, False), (4, 9, 9, BF, 2.0, False), (5, 9, 8, F32, 1.0, True), (6, 255, 3, F16, 0.5, False), (7, 255, 65, F32, 1.0, True),
    (300, 257, 8, BF, 1.0, False), (6, 1001, 20, BF, 1.0, True), (3, 2048, 256, F32, 4.0, False), (3, 2051, 130, F16, 1.0, True),
    (2, 32000, 20, BF, 2.0, False), (2, 32000, 64, F32, 1.0, True), (3, 50001, 5, BF, 1.0, True), (2, 40003, 100, F32, 1.5, False),
    (1, 131072, 20, F16, 1.0, True)])
def test_distill(rows, V, k, dtype, T, tail):
    x = (_randn(V, rows, V) * 3).to(dtype)
    ids, values = _teacher(rows, x, k)
    weights = None
    if rows > 2:
        ids[1, k // 2:] = -100   # fewer tokens
        ids[2] = V               # none
        weights = _rand(k, rows) + 0.1
        weights[0] = 0.0
    dx = _check_distill(x, ids, values, T, tail, weights, 1024.0 if dtype == F16 else 1.0)
    if rows > 2:
        assert not dx[0].any() and not dx[2].any()


@pytest.mark.parametrize("tail,T", [(False, 1.0), (False, 3.0), (True, 1.0)])
@pytest.mark.parametrize("V", [40, 3000])
def test_distill_of_special_rows(V, tail, T):
    x = _randn(1, 10, V) * 2
    ids, values = _teacher(2, x, 6)
    x[0, 5:] = -INF                                # five logits left
    x[1] = torch.finfo(F32).min                    # a mask of the lowest value: uniform
    x[2, ids[2]] = 90.0                            # the rest is far below fp32's smallest weight
    values[3, 2] = -INF                            # an entry that is left out
    ids[4] = ids[4, 0]                             # the same token six times
    values[4] = math.log(0.1)
    ids[5, 3:] = torch.tensor([V, -1, -100])
    values[6] = torch.log_softmax(torch.arange(6.0), 0)  # no mass in the rest, but for rounding
    x[7] = 500.0
    x[8, ids[8, :2]] = -60.0                       # the teacher's tokens are the student's last
    values[9] = -0.0 if not tail else -30.0        # next to all of the mass in the rest
    ids[0] = torch.arange(6)                       # one of them impossible for the student
    values[0, 5] = -INF
    _check_distill(x, ids, values, T, tail, None)


@pytest.mark.parametrize("T", [0.25, 1.0, 3.0])
def test_distill_of_a_teachers_logits_of_any_size(T):
    """The loss and the gradient know the teacher's logits by their differences:
    a row of the type's lowest value is one of zeros, and large logits cost no digits."""
    x = _randn(1, 5, 90).cuda().requires_grad_(True)
    ids, near = _randint(2, 90, 5, 7).cuda(), (_randint(3, 64, 5, 7) / 8.0).cuda()
    near[0] = near[1] = 0.0
    far = near + 2.0**16  # exact: 19 bits
    far[0], far[1] = torch.finfo(F32).min, torch.finfo(F32).max
    results = []
    for values in (near, far):
        loss = _ops().distill_loss(x, ids, values, temperature=T)
        results.append((loss, *torch.autograd.grad(loss, [x])))
    (a, da), (b, db) = results
    # the same numbers are formed of the same differences
    assert torch.equal(a, b) and torch.equal(da, db)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_of_rows_without_probabilities(tail):
    x = _randn(3, 5, 200)
    ids, values = _teacher(4, x, 3)
    x[0], x[1, 3], x[2, 3] = -INF, NAN, INF
    weights = torch.tensor([0.0, 0.0, 0.0, 1.0, 2.0])
    dx = _check_distill(x, ids, values, 1.0, tail, weights)
    assert not dx[:3].any()
    for r in range(3):
        xg = x[r:r + 1].cuda().requires_grad_(True)
        loss = _ops().distill_loss(xg, ids[r:r + 1].cuda(), values[r:r + 1].cuda(), tail=tail)
        (dx,) = torch.autograd.grad(loss, [xg])
        assert loss.isnan() and dx.isnan().any()
        assert tail or dx.isnan().all()
    none = _ops().distill_loss(x.cuda(), torch.full_like(ids, -100).cuda(), values.cuda(), tail=tail)
    assert none.isnan()
    assert _ops().distill_loss(x[:0].cuda(), ids[:0].cuda(), values[:0].cuda(), tail=tail).isnan()
    xg = x.cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(_ops().distill_loss(xg, ids.cuda(), values.cuda(), tail=tail), [xg], torch.tensor(0.0).cuda())
    assert not dx.any()  # no cotangent reaches the rows


@pytest.mark.parametrize("make", [
    lambda x: x[:, :-1], lambda x: x[:, 1::2], lambda x: x[..., 3:-2], lambda x: x.transpose(0, 1),
    lambda x: x[:1].expand(4, -1, -1), lambda x: x[0, 0], lambda x: x[None, :, None], lambda x: x.permute(2, 0, 1)])
def test_distill_of_views(make):
    x = make((_randn(5, 3, 6, 1003) * 2).to(BF))
    ids, values = _teacher(1, x, 2)
    xg = make((_randn(5, 3, 6, 1003) * 2).to(BF).cuda()).detach().requires_grad_(True)
    loss = _ops().distill_loss(xg, ids.cuda().int(), values.cuda().double(), tail=True)
    (dx,) = torch.autograd.grad(loss, [xg])
    V = x.shape[-1]
    want, grad = lb.distill(x.reshape(-1, V).double(), ids.reshape(-1, 2), values.reshape(-1, 2).double(), 1.0, True, None, BF)
    lm.assert_within(loss, *want, "loss")
    lm.assert_within(dx.reshape(-1, V), *grad, "dx")


def test_distill_gradient_is_the_difference_quotient():
    x, h = _randn(11, 3, 37).double(), 2.0**-6
    ids, values = _teacher(12, x, 4)
    for kw in (dict(temperature=2.0), dict(tail=True)):
        def value(z):
            return _ops().distill_loss(z.float().cuda(), ids.cuda(), values.cuda(), **kw).item()

        xg = x.float().cuda().requires_grad_(True)
        (dx,) = torch.autograd.grad(_ops().distill_loss(xg, ids.cuda(), values.cuda(), **kw), [xg])
        at = x.float().double()
        for r, c in ((0, 0), (0, 7), (1, 36), (2, int(ids[2, 0])), (1, int(ids[1, 3]))):
            d = torch.zeros_like(at)
            d[r, c] = h
            # third derivatives of order one times h^2, fp32 values of order ten over h
            assert abs((value(at + d) - value(at - d)) / (2 * h) - dx[r, c].item()) < 8 * h * h + 60 * 2.0**-24 / h, (kw, r, c)


def test_distill_recorded_backward():
    x = _randn(12, 4, 50)
    ids, values = _teacher(13, x, 5)
    for kw in (dict(temperature=2.0), dict(tail=True)):
        xg = x.cuda().requires_grad_(True)
        loss = _ops().distill_loss(xg, ids.cuda(), values.cuda(), **kw)
        (plain,) = torch.autograd.grad(loss, [xg], retain_graph=True)
        (dx,) = torch.autograd.grad(loss, [xg], create_graph=True)
        (ddx,) = torch.autograd.grad(dx.square().sum(), [xg])
        T, tail, h, d = kw.get("temperature", 1.0), kw.get("tail", False), 1e-4, _randn(14, 4, 50).double()
        ref = lb.distill(x.double(), ids, values.double(), T, tail, None, F32)[1][0]
        assert (dx.double().cpu() - ref).abs().max() < 1e-5 and (plain.double().cpu() - ref).abs().max() < 1e-5
        quotient = sum(s * lb.distill(x.double() + s * h * d, ids, values.double(), T, tail, None, F32)[1][0].square().sum()
                       for s in (1, -1)) / (2 * h)
        assert abs(quotient - (ddx.double().cpu() * d).sum()) < 1e-4


# ---------------------------------------------------------------- together


def _step(logits, history, lengths, prompts, uniform, allowed, ops):
    """A decode step's choice, the tokens kept; then the loss of the choice's logits against those before."""
    y = ops.adjust_logits(logits, history, lengths, prompts, repetition=1.2, presence=0.1, frequency=0.2, allowed=allowed)
    r = ops.sample_tokens(y.detach(), uniform, temperature=0.9, top_k=40, top_p=0.95)
    top = ops.token_logprobs(logits.detach(), r.ids, top_k=8)
    loss = ops.distill_loss(y, top.top_ids, top.top_logprobs, tail=True, weights=uniform)
    (dx,) = torch.autograd.grad(loss, [logits])
    return y.detach(), r.ids, r.logprob, loss.detach(), dx


def _step_inputs(seed, rows=12, V=5003, L=70):
    return ((_randn(seed, rows, V) * 3).to(BF).cuda().requires_grad_(True), _randint(seed + 1, V, rows, L).cuda(),
            _randint(seed + 2, L, rows).cuda(), _randint(seed + 3, 20, rows).cuda(), _rand(seed + 4, rows).cuda(),
            (_rand(seed + 5, rows, V) < 0.9).cuda())


def test_a_run_of_them_together():
    x, history, lengths, prompts, u, allowed = inputs = _step_inputs(1)
    y, ids, logprob, loss, dx = _step(*inputs, ops=_ops())
    xc = x.detach().cpu()
    rows, V = xc.shape
    want, bound = lb.adjust(xc.double(), history.tolist(), lengths.tolist(), prompts.tolist(), [1.2] * rows, [0.1] * rows, [0.2] * rows,
                            None, None, allowed.cpu(), BF)
    lm.assert_within(y, want, bound, "y")
    yc = y.cpu()
    _check_choice(yc, u.cpu(), type("r", (), dict(ids=ids.cpu(), logprob=logprob.cpu())), 0.9, 40, 0.95)
    assert allowed.cpu().gather(1, ids.cpu()[:, None]).all()
    top = lm.order(xc.double(), 8)
    values = torch.log_softmax(xc.double(), -1).gather(1, top)
    teacher = _ops().token_logprobs(x.detach(), ids, top_k=8).top_logprobs.cpu().double()
    assert (teacher - values).abs().max() < 1e-4
    # (the student's row is y; the slope of y by x scales the gradient, which is rounded twice)
    (ref, err), (dy, e_dy) = lb.distill(yc.double(), top, teacher, 1.0, True, u.cpu(), BF)
    lm.assert_within(loss, ref, err, "loss")
    _, (gx, e_gx) = lb.adjust(xc.double(), history.tolist(), lengths.tolist(), prompts.tolist(), [1.2] * rows, [0.1] * rows,
                              [0.2] * rows, None, None, allowed.cpu(), BF, dy)
    lm.assert_within(dx, gx, e_gx + 1.3 * e_dy, "dx")


def test_together_captured_and_replayed():
    """Graphs of two batches, replayed in turn with eager work between: every replay's results are the eager ones."""
    graphs = []
    for seed in (1, 2):
        inputs = _step_inputs(seed, rows=9 + seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(*inputs, ops=_ops())
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*inputs, ops=_ops())
        graphs.append((g, inputs, out))
    for n in range(4):
        for g, inputs, _ in graphs:
            inputs[4].copy_(_rand(n, inputs[4].shape[0]))
            inputs[1].copy_(_randint(n, 5003, *inputs[1].shape))
            g.replay()
        torch.cuda.synchronize()
        for g, inputs, out in graphs:
            fresh = (inputs[0].detach().clone().requires_grad_(True),) + inputs[1:]
            for a, b in zip(out, _step(*fresh, ops=_ops())):
                assert torch.equal(a, b)
            with torch.no_grad():
                inputs[0].mul_(1.01)


def test_wide_and_whole_rows_captured_and_replayed():
    """The paths of few wide rows, of whole rows in turn and of long histories in two graphs, replayed in turn."""
    ops, graphs = _ops(), []
    for seed in (3, 4):
        wide, many = (_randn(seed, 5, 50001) * 3).to(BF).cuda(), (_randn(seed + 1, 2500, 300) * 3).cuda()
        history, u, v = _randint(seed, 300, 2500, 600).cuda(), _rand(seed, 5).cuda(), _rand(seed, 2500).cuda()

        def run(wide=wide, many=many, history=history, u=u, v=v):
            y = ops.adjust_logits(many, history, repetition=1.2, frequency=0.1)
            return (*ops.sample_tokens(wide, u, top_p=0.9), *ops.sample_tokens(wide, u, temperature=2.0), y, *ops.sample_tokens(y, v, min_p=0.01))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, run, out, (u, v, history)))
    for n in range(4):
        for g, _, _, (u, v, history) in graphs:
            u.copy_(_rand(n, 5))
            v.copy_(_rand(n + 9, 2500))
            history.copy_(_randint(n, 300, 2500, 600))
            g.replay()
        torch.cuda.synchronize()
        for _, run, out, _ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, run()))


def test_together_on_other_streams_and_threads():
    from concurrent.futures import ThreadPoolExecutor

    ops = _ops()

    def run(stream):
        with torch.cuda.stream(stream):
            out = _step(*_step_inputs(5), ops=ops)
            wide = ops.sample_tokens((_randn(1, 3, 140000) * 2).cuda(), _rand(2, 3).cuda(), top_p=0.9)
            stream.synchronize()
        return [*out, *wide]

    want = run(torch.cuda.current_stream())
    with ThreadPoolExecutor(2) as pool:
        for _ in range(3):
            for got in pool.map(run, [torch.cuda.Stream() for _ in range(2)]):
                assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Logits of more than 2^31 elements: the last rows as in calls of their own."""
    ops, rows, V = _ops(), 70001, 32001
    assert rows * V > 2**31
    x = torch.zeros(rows, V, dtype=BF, device="cuda")
    last = (_randn(1, 3, V) * 3).to(BF).cuda()
    x[-3:] = last
    u = torch.full((rows,), 0.5, device="cuda")
    got = ops.sample_tokens(x, u, top_k=100, top_p=0.9)
    own = ops.sample_tokens(last, u[:3], top_k=100, top_p=0.9)
    assert torch.equal(got.ids[-3:], own.ids) and torch.equal(got.logprob[-3:], own.logprob) and got.ids[7] == 45
    history = torch.arange(50, device="cuda").expand(rows, 50)
    y = ops.adjust_logits(x.requires_grad_(True), history, frequency=0.5)
    assert torch.equal(y[-3:], ops.adjust_logits(last, history[:3], frequency=0.5)) and y[9, 0] == -0.5 and y[9, 50] == 0
    ids = torch.full((rows, 4), -100, device="cuda")
    ids[-3:] = torch.tensor([0, 5, 77, V - 1])
    values = torch.full((rows, 4), -1.5, device="cuda")
    loss = ops.distill_loss(x, ids, values, tail=True)
    (dx,) = torch.autograd.grad(loss, [x])
    lastg = last.clone().requires_grad_(True)
    want = ops.distill_loss(lastg, ids[-3:], values[-3:], tail=True)
    assert torch.equal(loss, want) and torch.equal(dx[-3:], torch.autograd.grad(want, [lastg])[0]) and not dx[:-3].any()


def test_more_rows_than_a_launch_takes():
    """2^20 and more workgroups: the last rows as in calls of their own."""
    ops, rows = _ops(), (1 << 22) + 9
    x = (_randn(1, rows, 5) * 2).to(BF).cuda()
    history = _randint(2, 5, rows, 3).cuda()
    y = ops.adjust_logits(x, history, repetition=1.5, frequency=0.25)
    allowed = torch.ones(5, dtype=torch.bool, device="cuda")
    plain = x.float()
    n = torch.zeros(rows, 5, device="cuda").scatter_add_(1, history, torch.ones(rows, 3, device="cuda"))
    plain = torch.where(n > 0, torch.where(plain > 0, plain / 1.5, plain * 1.5) - 0.25 * n, plain).to(BF)
    assert torch.equal(y, plain) and torch.equal(ops.adjust_logits(x, history, repetition=1.5, frequency=0.25, allowed=allowed), plain)
    u = _rand(3, rows).cuda()
    got = ops.sample_tokens(x, u, top_k=3, top_p=0.9)
    ids, values = _randint(4, 6, rows, 2).cuda(), -_rand(5, rows, 2).cuda() - 1
    weights = torch.zeros(rows, device="cuda")
    weights[-9:] = 1.0
    xg = x.clone().requires_grad_(True)
    loss = ops.distill_loss(xg, ids, values, tail=True, weights=weights)
    (dx,) = torch.autograd.grad(loss, [xg])
    assert not dx[:-9].any()
    for part in (slice(0, 7), slice((1 << 20) - 3, (1 << 20) + 3), slice((1 << 22) - 3, rows)):
        own = ops.sample_tokens(x[part], u[part], top_k=3, top_p=0.9)
        assert torch.equal(got.ids[part], own.ids) and torch.equal(got.logprob[part], own.logprob)
    xg = x[-9:].clone().requires_grad_(True)
    last = ops.distill_loss(xg, ids[-9:], values[-9:], tail=True)
    assert torch.equal(last, loss) and torch.equal(torch.autograd.grad(last, [xg])[0], dx[-9:])


def test_the_most_shared_memory():
    """The largest slices, histories and token biases, and the largest vocabulary beside a tail, of one workgroup."""
    rows, V, L = 136, 65536, 16383
    x, kw, allowed = _adjust_case(5, 3, V, L, BF, False, False, 1024, "bits")
    kw["lengths"][:] = L
    args = {n: _cuda(t) for n, t in kw.items()}
    args["token_bias"] = tuple(t.repeat(46, 1)[:rows] for t in args["token_bias"])
    y = _ops().adjust_logits(x.cuda().repeat(46, 1)[:rows], **{n: t if isinstance(t, tuple) else t.repeat(46, *[1] * (t.dim() - 1))[:rows]
                                                              for n, t in args.items()})
    lm.assert_within(y[:3], *_adjust_ref(x, kw, allowed), "y")
    assert all(torch.equal(y[r].view(torch.uint8), y[r % 3].view(torch.uint8)) for r in (3, 70, 135))
    V = 1 << 19
    x = (_randn(6, 2, V) * 3).to(BF)
    ids, values = _teacher(7, x, 256)
    _check_distill(x, ids, values, 1.0, True, None)


def test_inference_tensors():
    ops = _ops()
    with torch.inference_mode():
        x = _randn(1, 4, 33).cuda()
        y = ops.adjust_logits(x, torch.tensor([1, 1]).cuda(), presence=1.0)
        assert ops.adjust_logits(x, torch.tensor([1, 1]).cuda(), presence=1.0, out=x) is x and torch.equal(x, y)
        r = ops.sample_tokens(x, torch.full((4,), 0.5).cuda())
        loss = ops.distill_loss(x, r.ids[:, None], torch.zeros(4, 1).cuda())
    assert abs(loss.item() + torch.log_softmax(x, -1).gather(1, r.ids[:, None]).mean().item()) < 1e-5
