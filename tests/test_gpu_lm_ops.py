"""The operators around a model's blocks (ops.token_logprobs, token_loss,
embed_tokens, residual_norm) against float64 on the CPU, at sizes and values
where they can go wrong; the bounds are derived in lm_bounds."""

import math

import pytest
import torch

import lm_bounds as lm

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def _ops():
    from cyclic_flow_attention import ops

    return ops


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def _randint(seed, n, *shape):
    return torch.randint(0, n, shape, generator=torch.Generator().manual_seed(seed))


def _check_logprobs(got, x, tokens, k, what=""):
    ref = lm.logprobs(x.double(), tokens, k)
    for name, value in (("logprob", got.logprob), ("entropy", got.entropy), ("top", got.top_logprobs)):
        if name in ref:
            lm.assert_within(value, *ref[name], f"{what} {name}")
    if k:
        assert torch.equal(got.top_ids.cpu(), ref["ids"]), what
    else:
        assert got.top_logprobs is None and got.top_ids is None


# ---------------------------------------------------------------- token_logprobs


@pytest.mark.parametrize("rows,V,dtype,k", [
    (1, 1, F32, 1), (3, 7, BF, 7), (2, 8, F16, 3), (5, 255, BF, 32), (4, 257, F32, 20), (7, 1000, F16, 5), (66, 2051, BF, 1),
    (2, 8192, F32, 0), (3, 32000, BF, 20), (2, 32768, BF, 32), (3, 50001, BF, 5), (2, 70003, F32, 9), (300, 513, BF, 0),
    (1, 131072, F16, 31), (1, 300000, BF, 32), (40, 40000, F32, 7), (100, 33001, BF, 2), (250, 16385, F32, 0), (6, 98305, F16, 0),
    (520, 40001, BF, 3)])
def test_logprobs(rows, V, dtype, k):
    x = (_randn(rows + V, rows, V) * 3).to(dtype)  # 16-bit logits of a large vocabulary hold many equal ones
    tokens = _randint(V, V, rows)
    got = _ops().token_logprobs(x.cuda(), tokens.cuda(), top_k=k)
    assert got.logprob.dtype == got.entropy.dtype == F32
    _check_logprobs(got, x, tokens, k)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_logprobs_of_masked_rows(dtype):
    V, low = 1500, torch.finfo(dtype).min
    x = (_randn(1, 9, V) * 2).to(dtype)
    x[0, 5:] = -INF                      # five tokens left
    x[1] = -INF
    x[1, 1499] = 3.0                     # one, in the last column
    x[2] = low                           # nothing left under a mask of the lowest value: uniform
    x[3, 3:] = low
    x[4, :] = 7.5                        # all equal
    x[5, 10] = torch.finfo(dtype).max    # a spread that overflows a difference
    x[5, 11:] = low
    x[6, ::2] = -INF
    x[7] = -x[7].abs() - 60              # far below zero
    x[8] = 0.0
    x[8, 1::2] = -0.0                    # equal zeros: the lower id first
    tokens = torch.tensor([3, 1499, 77, 1, 1400, 10, 1, 20, 6])
    got = _ops().token_logprobs(x.cuda(), tokens.cuda(), top_k=12)
    _check_logprobs(got, x, tokens, 12)
    assert got.logprob[1].item() == 0.0 and got.entropy[1].item() == 0.0
    assert abs(got.logprob[2].item() + math.log(V)) < 1e-5


def test_logprobs_of_masked_rows_in_parts():
    """Rows shared out to several workgroups: parts of nothing but -inf, of the
    lowest value, with a NaN, with all of the alternatives."""
    V = 100003
    x = (_randn(1, 6, V) * 2).to(BF)
    x[0, 40000:] = -INF
    x[1] = -INF
    x[1, V - 1] = 2.0
    x[2, 70000] = NAN
    x[3] = torch.finfo(BF).min
    x[4, 33000:33020] = 30.0
    x[5] = -INF
    tokens = torch.tensor([5, V - 1, 3, 99999, 33001, 0])
    got = _ops().token_logprobs(x.cuda(), tokens.cuda(), top_k=20)
    keep = torch.tensor([0, 1, 3, 4])
    _check_logprobs(type(got)(*(t.cpu()[keep] for t in got)), x[keep], tokens[keep], 20)
    assert torch.equal(got.top_ids.cpu(), lm.order(x.double(), 20))
    for row in (2, 5):
        assert got.logprob[row].isnan() and got.entropy[row].isnan()
    labels = tokens.cuda()
    labels[2] = labels[5] = -100
    loss = _ops().token_loss(x.cuda(), labels)
    ref, err = lm.logprobs(x[keep].double(), tokens[keep])["logprob"]
    lm.assert_within(loss, -ref.mean(), lm.rounded(ref.mean(), err.mean(), F32), "loss")


def test_logprobs_of_rows_without_probabilities():
    x = _randn(2, 5, 300)
    x[0] = -INF
    x[1, 7] = NAN
    x[2, 9] = INF
    x[3, 5], x[3, 200] = NAN, INF
    tokens = torch.zeros(5, dtype=torch.int64)
    got = _ops().token_logprobs(x.cuda(), tokens.cuda(), top_k=3)
    assert got.logprob[:4].isnan().all() and got.entropy[:4].isnan().all() and got.top_logprobs[:4].isnan().all()
    assert torch.equal(got.top_ids.cpu(), lm.order(x.double(), 3))
    _check_logprobs(_ops().token_logprobs(x[4:].cuda(), tokens[4:].cuda(), top_k=3), x[4:], tokens[4:], 3)


@pytest.mark.parametrize("V,k,dtype", [(70000, 32, BF), (66000, 32, F32), (4000, 32, F16)])
def test_alternatives_gathered_in_few_columns(V, k, dtype):
    """More elements reach the threshold than are held at once: the largest all
    lie in the columns of few threads, or all but a few are equal."""
    x = torch.full((3, V), -5.0)
    x[0] = -INF
    x[0, 17] = 1.0
    cols = torch.arange(V)
    few = (cols // 8) % 64 < k - 1
    x[1, few] = (_randn(3, int(few.sum())) + 4)
    x[2, few] = 2.0 + torch.arange(int(few.sum())) * 2.0**-6
    x = x.to(dtype)
    tokens = torch.tensor([17, 3, 5])
    got = _ops().token_logprobs(x.cuda(), tokens.cuda(), top_k=k)
    assert torch.equal(got.top_ids.cpu(), lm.order(x.double(), k))


@pytest.mark.parametrize("make", [
    lambda x: x[:, :-1], lambda x: x[:, 1::2], lambda x: x[..., 3:-2], lambda x: x.transpose(0, 1),
    lambda x: x[:1].expand(4, -1, -1), lambda x: x[0, 0], lambda x: x[:, :0], lambda x: x[None, :, None],
    lambda x: x.permute(2, 0, 1), lambda x: x[:, 2:3]])
def test_logprobs_of_views(make):
    base = (_randn(5, 3, 6, 1003) * 2).to(BF)
    x, xg = make(base), make(base.cuda())
    tokens = _randint(1, x.shape[-1], *x.shape[:-1])
    xg = xg.detach().requires_grad_(True)
    got = _ops().token_logprobs(xg, tokens.cuda(), top_k=2)
    assert got.logprob.shape == tokens.shape and got.top_ids.shape == tokens.shape + (2,)
    V = x.shape[-1]
    flat = type(got)(*(t.reshape(-1, *t.shape[tokens.dim():]) for t in got))
    _check_logprobs(flat, x.reshape(-1, V), tokens.reshape(-1), 2)
    d = _randn(9, *tokens.shape)
    (dx,) = torch.autograd.grad(got.logprob, [xg], d.cuda())
    ref = lm.logprobs_grad(x.reshape(-1, V).double(), tokens.reshape(-1), None, d.reshape(-1).double(), None, None, BF)
    lm.assert_within(dx.reshape(-1, V), *ref, "dx")


def test_logprobs_of_ignored_and_impossible_tokens():
    x = _randn(6, 5, 40)
    tokens = torch.tensor([4, -100, 40, -1, 39], dtype=torch.int32)
    xg = x.cuda().requires_grad_(True)
    got = _ops().token_logprobs(xg, tokens.cuda())
    _check_logprobs(got, x, tokens.long(), 0)
    assert got.logprob[1].item() == 0.0 and got.logprob[2:4].isnan().all()
    (dx,) = torch.autograd.grad(got.logprob[[0, 1, 4]].sum(), [xg])
    ref = lm.logprobs_grad(x.double(), tokens.long(), None, torch.tensor([1.0, 1, 0, 0, 1]).double(), None, None, F32)
    lm.assert_within(dx, *ref, "dx")
    assert not dx[1:4].any()
    zero = _ops().token_logprobs(x.cuda(), torch.zeros(5, dtype=torch.int64, device="cuda"), ignore_index=0)
    assert not zero.logprob.any()


@pytest.mark.parametrize("rows,V,dtype,k,parts", [
    (3, 1, F32, 1, "let"), (4, 9, BF, 9, "let"), (5, 255, F16, 3, "t"), (6, 1001, BF, 20, "let"), (2, 32000, BF, 0, "le"),
    (3, 50001, BF, 5, "e"), (9, 2048, F32, 32, "let"), (300, 257, BF, 0, "l"), (2, 40000, F32, 0, "le")])
def test_logprobs_gradient(rows, V, dtype, k, parts):
    x = (_randn(V, rows, V) * 3).to(dtype)
    if V > 100:
        x[0, 50:] = -INF
    tokens = _randint(rows, V, rows)
    tokens[-1] = int(x[-1].double().argmax())  # a token that is an alternative too
    xg = x.cuda().requires_grad_(True)
    got = _ops().token_logprobs(xg, tokens.cuda(), top_k=k)
    assert not (k and got.top_ids.requires_grad)
    cots = {"l": _randn(1, rows), "e": _randn(2, rows), "t": _randn(3, rows, max(k, 1))}
    if rows > 2:
        for c in cots.values():
            c[1] = 0
    outs = {"l": got.logprob, "e": got.entropy, "t": got.top_logprobs}
    (dx,) = torch.autograd.grad([outs[c] for c in parts], [xg], [cots[c].cuda() for c in parts])
    assert dx.dtype == dtype
    given = [cots[c].double() if c in parts else None for c in "let"]
    ids = got.top_ids.cpu() if k else None
    lm.assert_within(dx, *lm.logprobs_grad(x.double(), tokens, ids, *given, dtype), "dx")
    if rows > 2:
        assert not dx[1].any()


def test_logprobs_gradient_of_rows_without_probabilities():
    x = _randn(3, 4, 200)
    x[0], x[1, 3], x[2, 3] = -INF, NAN, INF
    xg = x.cuda().requires_grad_(True)
    got = _ops().token_logprobs(xg, torch.zeros(4, dtype=torch.int64).cuda(), top_k=2)
    outs = [got.logprob, got.entropy, got.top_logprobs]
    ones = [torch.ones_like(t) for t in outs]
    for part in range(3):
        (dx,) = torch.autograd.grad(outs[part], [xg], ones[part], retain_graph=True)
        assert dx[:3].isnan().all(-1).all() and dx[3].isfinite().all()
    none = [torch.cat([torch.zeros_like(o[:3]), o[3:]]) for o in ones]  # rows that no cotangent reaches
    (dx,) = torch.autograd.grad(outs, [xg], none)
    assert not dx[:3].any() and dx[3].isfinite().all()


def test_logprobs_gradient_is_the_difference_quotient():
    x = _randn(11, 3, 37).double()
    tokens, h = torch.tensor([0, 36, 5]), 2.0**-6
    w = [_randn(s, *shape) for s, shape in ((1, (3,)), (2, (3,)), (3, (3, 4)))]
    xg = x.float().cuda().requires_grad_(True)
    got = _ops().token_logprobs(xg, tokens.cuda(), top_k=4)
    outs = [got.logprob, got.entropy, got.top_logprobs]
    (dx,) = torch.autograd.grad(outs, [xg], [t.cuda() for t in w])

    def value(z):
        r = _ops().token_logprobs(z.float().cuda(), tokens.cuda())
        top = z.float() - torch.logsumexp(z, -1, keepdim=True)
        return ((r.logprob.cpu().double() * w[0]).sum() + (r.entropy.cpu().double() * w[1]).sum()
                + (top.double().gather(1, got.top_ids.cpu()) * w[2]).sum())

    x = x.float().double()
    for r, c in ((0, 0), (0, 7), (1, 36), (2, 1), (2, int(got.top_ids[2, 0]))):
        d = torch.zeros_like(x)
        d[r, c] = h
        quotient = (value(x + d) - value(x - d)) / (2 * h)
        # third derivatives of order one times h^2, fp32 values of order ten over h
        assert abs(quotient.item() - dx[r, c].item()) < 8 * h * h + 60 * 2.0**-24 / h, (r, c)


def test_logprobs_recorded_backward():
    x = _randn(12, 4, 50)
    tokens = torch.tensor([3, -100, 49, 0])
    xg = x.cuda().requires_grad_(True)
    got = _ops().token_logprobs(xg, tokens.cuda(), top_k=2)
    (dx,) = torch.autograd.grad(got.logprob.sum() + 2 * got.entropy.sum(), [xg], create_graph=True)
    (ddx,) = torch.autograd.grad(dx.square().sum(), [xg])
    xd = x.double().requires_grad_(True)
    lp = torch.log_softmax(xd, -1)
    total = lp[0, 3] + lp[2, 49] + lp[3, 0] - 2 * (lp.exp() * lp).sum()
    (rx,) = torch.autograd.grad(total, [xd], create_graph=True)
    (rrx,) = torch.autograd.grad(rx.square().sum(), [xd])
    assert (dx.double().cpu() - rx).abs().max() < 1e-5 and (ddx.double().cpu() - rrx).abs().max() < 1e-4


# ---------------------------------------------------------------- token_loss


@pytest.mark.parametrize("B,T,V,dtype", [(1, 1, 1, F32), (2, 5, 13, F16), (3, 37, 256, F32), (2, 33, 1001, BF), (4, 300, 64, BF),
                                         (2, 2, 32000, BF)])
def test_loss(B, T, V, dtype):
    x = (_randn(T, B, T, V) * 3).to(dtype)
    labels = _randint(V, V, B, T)
    if T > 1:
        labels[:, -2:] = -100
        labels[0, 0] = 0
    xg = x.cuda().requires_grad_(True)
    loss = _ops().token_loss(xg, labels.cuda())
    (dx,) = torch.autograd.grad(loss, [xg], torch.tensor(0.75).cuda())
    kept = (labels != -100).reshape(-1)
    ref, err = lm.logprobs(x.reshape(-1, V).double(), labels.reshape(-1))["logprob"]
    mean, bound = -ref[kept].mean(), err[kept].mean()
    lm.assert_within(loss, mean, lm.rounded(mean, bound, F32), "loss")
    d = torch.where(kept, -0.75 / kept.sum().double(), 0.0)
    lm.assert_within(dx.reshape(-1, V), *lm.logprobs_grad(x.reshape(-1, V).double(), labels.reshape(-1), None, d, None, None, dtype),
                     "dx")
    assert torch.equal(_ops().token_loss(xg.detach(), labels.cuda()), loss.detach())


def test_loss_without_labels_and_with_impossible_ones():
    x = _randn(1, 6, 20).cuda().requires_grad_(True)
    labels = torch.full((6,), -100, device="cuda")
    loss = _ops().token_loss(x, labels)
    assert loss.isnan() and not torch.autograd.grad(loss, [x])[0].any()
    labels[2] = 20
    loss = _ops().token_loss(x, labels)
    (dx,) = torch.autograd.grad(loss, [x])
    assert loss.isnan() and dx[2].isnan().all() and not dx[3].any()
    assert _ops().token_loss(x[:0], labels[:0]).isnan()
    assert torch.autograd.grad(_ops().token_loss(x[:0], labels[:0]), [x])[0].shape == x.shape
    with torch.no_grad():
        row = x[:1].clone()
        row[:] = -INF
    row.requires_grad_(True)  # a masked row whose label is ignored
    two = torch.cat([row, x[:1]])
    loss = _ops().token_loss(two, torch.tensor([-100, 3]).cuda())
    assert loss.isfinite() and torch.autograd.grad(loss, [row])[0].abs().max().item() == 0


def test_loss_recorded_backward():
    x = _randn(2, 5, 30)
    labels = torch.tensor([1, -100, 29, 0, 7])
    xg, xd = x.cuda().requires_grad_(True), x.double().requires_grad_(True)
    out = []
    for t, loss in ((xg, _ops().token_loss(xg, labels.cuda())), (xd, torch.nn.functional.cross_entropy(xd, labels))):
        (dx,) = torch.autograd.grad(loss, [t], create_graph=True)
        out.append((dx, torch.autograd.grad((dx * dx).sum(), [t])[0]))
    for a, b in zip(*out):
        assert (a.double().cpu() - b).abs().max() < 1e-6


# ---------------------------------------------------------------- embed_tokens


@pytest.mark.parametrize("n,V,D,dtype,scale", [
    (1, 1, 1, F32, 1.0), (3, 5, 3, BF, 2.0), (64, 32, 7, F16, 1.0), (65, 300, 8, BF, 0.5), (129, 3, 33, F32, 1.0),
    (1000, 1000, 100, BF, 32.0), (700, 2, 513, F16, 1.0), (4097, 513, 64, F32, 1.0), (200, 1500, 1024, BF, 1.0),
    (1025, 140000, 16, BF, 1.0), (37, 64, 2050, F32, 3.0), (64, 90, 1000, BF, 1.0), (65, 90, 1000, BF, 1.0), (64, 3, 5, F16, 2.0),
    (65, 7, 3, F32, 1.0), (9, 70000, 1024, BF, 1.0)])
def test_embed(n, V, D, dtype, scale):
    w = _randn(n, V, D).to(dtype)
    ids = (_randint(V, V, n).double() ** 2 / V).long()  # low ids come up more often
    dy = _randn(D, n, D).to(dtype)
    wg = w.cuda().requires_grad_(True)
    out = _ops().embed_tokens(ids.cuda(), wg, scale=scale)
    ref = w[ids].double() * scale
    lm.assert_within(out, ref, lm.rounded(ref, 0 * ref, dtype), "out")
    (dw,) = torch.autograd.grad(out, [wg], dy.cuda(), retain_graph=True)
    lm.assert_within(dw, *lm.embed_grad(ids, dy.double(), V, scale, -1, dtype), "dw")
    assert torch.equal(dw, torch.autograd.grad(out, [wg], dy.cuda())[0])  # the same bits again
    assert not dw.cpu()[torch.bincount(ids, minlength=V) == 0].any()


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 127, 128, 1000, 20000])
def test_embed_gradient_of_one_id(n):
    """Every position holds the same id, the last of the vocabulary or the first."""
    V, D = 777, 40
    for at in (0, V - 1, 400):
        ids = torch.full((n,), at)
        wg = _randn(1, V, D).cuda().requires_grad_(True)
        dy = _randn(n, n, D)
        (dw,) = torch.autograd.grad(_ops().embed_tokens(ids.cuda(), wg), [wg], dy.cuda())
        lm.assert_within(dw, *lm.embed_grad(ids, dy.double(), V, 1.0, -1, F32), "dw")


def test_embed_ids_of_any_shape_padding_and_impossible_ids():
    V, D = 50, 24
    w = _randn(1, V, D).to(BF)
    ids = _randint(3, V, 4, 30)
    ids[0, :5] = torch.tensor([-1, V, 2**40, -(2**40), -100])
    ids[1] = 7
    ids[2, ::2] = V - 1
    dy = _randn(2, 4, 30, D).to(BF)
    for view in (lambda t: t, lambda t: t[:, ::3], lambda t: t.transpose(0, 1), lambda t: t[0, 5]):
        for pad, row in ((None, -1), (7, 7), (-1, V - 1)):
            x, d = view(ids), view(dy)
            wg = w.cuda().requires_grad_(True)
            out = _ops().embed_tokens(view(ids.cuda()), wg, padding_idx=pad)
            assert out.shape == x.shape + (D,)
            inside = ((x >= 0) & (x < V))[..., None]
            assert torch.equal(out.cpu().masked_fill(~inside, 0.0), w[x.clamp(0, V - 1)].masked_fill(~inside, 0.0))
            assert out.cpu().isnan().eq(~inside).all()
            (dw,) = torch.autograd.grad(out, [wg], view(dy.cuda()))
            lm.assert_within(dw, *lm.embed_grad(x.reshape(-1), d.reshape(-1, D).double(), V, 1.0, row, BF), "dw")
    small = _ops().embed_tokens(torch.tensor([1, 3], dtype=torch.int32, device="cuda"), w.cuda().t().contiguous().t())
    assert torch.equal(small.cpu(), w[[1, 3]])


def test_embed_gradient_past_the_caches():
    """A gradient of 135 MB in rows of whole lines, and in rows that are not."""
    for V, D, dtype in ((66000, 1024, BF), (66001, 1023, BF), (33000, 1024, F32)):
        ids = _randint(V, 200, 300)
        ids[::2] = V - 1 - ids[::2]
        dy = _randn(1, 300, D).to(dtype)
        w = torch.empty(V, D, dtype=dtype, device="cuda").requires_grad_(True)
        (dw,) = torch.autograd.grad(_ops().embed_tokens(ids.cuda(), w, padding_idx=5), [w], dy.cuda())
        rows = torch.unique(ids)
        at = torch.searchsorted(rows, ids)
        pad = int(torch.searchsorted(rows, 5)) if 5 in rows else -1
        lm.assert_within(dw.cpu()[rows], *lm.embed_grad(at, dy.double(), len(rows), 1.0, pad, dtype), "dw")
        dw[rows.cuda()] = 0
        assert not dw.any()


def test_embed_recorded_backward():
    ids = torch.tensor([2, 0, 2, 1, -5]).cuda()
    w = _randn(1, 4, 6).cuda().requires_grad_(True)
    d = _randn(2, 5, 6).cuda().requires_grad_(True)
    (dw,) = torch.autograd.grad(_ops().embed_tokens(ids, w, scale=2.0, padding_idx=1), [w], d, create_graph=True)
    v = _randn(3, 4, 6).cuda()
    (dd,) = torch.autograd.grad((dw * v).sum(), [d])
    want = torch.stack([2 * v[2], 2 * v[0], 2 * v[2], 0 * v[1], 0 * v[1]])
    assert torch.equal(dd, want)


# ---------------------------------------------------------------- residual_norm


def _join_inputs(rows, D, dtype, post, gate, seed=0):
    def make(i):
        return _randn(seed + i, rows, D).to(dtype)

    return dict(x=make(1) * 2, y=make(2), weight=1 + 0.2 * _randn(seed + 3, D), post=1 + 0.2 * _randn(seed + 4, D) if post else None,
                gate=make(5) if gate else None), make(6), make(7)


def _check_join(t, d_s, d_h, scale, eps, dtype, call=None):
    leaves = {n: v.cuda().requires_grad_(True) for n, v in t.items() if v is not None}
    s, h = (call or _ops().residual_norm)(leaves["x"], leaves["y"], leaves["weight"], post_weight=leaves.get("post"),
                                          gate=leaves.get("gate"), scale=scale, eps=eps)
    grads = dict(zip(leaves, torch.autograd.grad([s, h], list(leaves.values()), [d_s.cuda(), d_h.cuda()])))
    ref = lm.residual(*(None if v is None else v.double() for v in t.values()), scale, eps, d_s.double(), d_h.double())
    for name, (value, err) in ref.items():
        got = {"s": s, "h": h, **grads}[name]
        assert got.dtype == (F32 if name in ("weight", "post") else dtype)
        lm.assert_within(got, value, lm.rounded(value, err, got.dtype), name)
    with torch.no_grad():
        again = _ops().residual_norm(*(None if v is None else v.cuda() for v in t.values()), scale=scale, eps=eps)
    assert torch.equal(again[0], s) and torch.equal(again[1], h)


@pytest.mark.parametrize("post,gate", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("rows,D,dtype,scale", [
    (1, 1, F32, 1.0), (3, 3, F32, 0.5), (2, 7, BF, 1.0), (5, 8, BF, 1.0), (4, 9, F16, -0.5), (3, 64, F32, 1.0), (65, 100, BF, 1.0),
    (2, 257, F32, 2.0), (9, 512, F16, 1.0), (5, 513, BF, 0.5), (1, 1024, BF, 1.0), (3, 1001, F32, 1.0), (2, 1536, BF, 1.0),
    (600, 40, BF, 1.0), (3, 2048, F32, 1.0), (4, 2049, BF, 1.0), (2, 5000, F16, 1.0), (2, 8192, F32, 1.0), (3, 8191, BF, 0.25),
    (2100, 36, F32, 1.0), (16, 520, BF, 1.0), (17, 520, BF, 1.0), (4, 3000, F32, 0.5), (5, 3000, F32, 0.5)])
def test_residual_norm(rows, D, dtype, scale, post, gate):
    t, d_s, d_h = _join_inputs(rows, D, dtype, post, gate, seed=D)
    _check_join(t, d_s, d_h, scale, 1e-6, dtype)


def test_residual_norm_of_zero_rows_and_no_rows():
    t, d_s, d_h = _join_inputs(4, 96, BF, True, True)
    t["y"][1] = 0
    t["x"][2], t["y"][2] = 0, 0
    t["gate"][3] = -300.0
    _check_join(t, d_s, d_h, 1.0, 1e-2, BF)
    t, d_s, d_h = _join_inputs(0, 96, BF, True, True)
    _check_join(t, d_s, d_h, 1.0, 1e-6, BF)
    t, d_s, d_h = _join_inputs(3, 96, F32, True, True)
    t["x"][1, 5] = NAN
    s, h = _ops().residual_norm(*(v.cuda() for v in t.values()))
    assert h[1].isnan().all() and h[[0, 2]].isfinite().all() and s[1].isnan().sum() == 1


def test_residual_norm_of_views_and_other_weights():
    """Strided and misaligned operands, weights of another dtype, one cotangent only."""
    t, d_s, d_h = _join_inputs(12, 40, BF, True, True)

    def strided(x, y, weight, post_weight, gate, scale, eps):
        wide = torch.cat([x, y, gate], 1)
        shape = (3, 4, 40)
        parts = [wide[:, i * 40:(i + 1) * 40].unflatten(0, (3, 4)) for i in range(3)]
        out = _ops().residual_norm(parts[0], parts[1], weight.double(), post_weight=post_weight.double(), gate=parts[2],
                                   scale=scale, eps=eps)
        assert out[0].shape == shape
        return tuple(o.flatten(0, 1) for o in out)

    _check_join(t, d_s, d_h, 1.0, 1e-6, BF, strided)

    def misaligned(x, y, weight, post_weight, gate, scale, eps):
        def off(v):
            base = torch.cat([v.new_zeros(1), v.reshape(-1)])
            return base[1:].view(v.shape)

        return _ops().residual_norm(off(x), off(y), off(weight), post_weight=off(post_weight), gate=off(gate), scale=scale, eps=eps)

    _check_join(t, d_s, d_h, 1.0, 1e-6, BF, misaligned)
    zero = torch.zeros_like(d_s)
    leaves = {n: v.cuda().requires_grad_(True) for n, v in t.items()}
    s, h = _ops().residual_norm(leaves["x"], leaves["y"], leaves["weight"], leaves["post"], leaves["gate"])
    for out, given in ((s, (d_s, zero)), (h, (zero, d_h))):
        ref = lm.residual(*(v.double() for v in t.values()), 1.0, 1e-6, given[0].double(), given[1].double())
        grads = torch.autograd.grad(out, list(leaves.values()), given[0 if out is s else 1].cuda(), retain_graph=True,
                                    allow_unused=True)
        for name, g in zip(leaves, grads):
            lm.assert_within(g, ref[name][0], lm.rounded(*ref[name], g.dtype), name)


def test_residual_norm_gradient_of_some_inputs():
    t, d_s, d_h = _join_inputs(6, 64, F32, True, True)
    full = None
    names = list(t)
    for wanted in (names, ["x"], ["y"], ["gate"], ["weight"], ["post"], ["y", "weight"]):
        leaves = {n: v.cuda().requires_grad_(n in wanted) for n, v in t.items()}
        out = _ops().residual_norm(leaves["x"], leaves["y"], leaves["weight"], leaves["post"], leaves["gate"])
        grads = dict(zip(wanted, torch.autograd.grad(out, [leaves[n] for n in wanted], [d_s.cuda(), d_h.cuda()])))
        full = full or grads
        for n in wanted:
            assert torch.equal(grads[n], full[n]), n
    for wanted in (["x"], ["y"], ["x", "y"]):  # the plain join: dy is dx
        leaves = {n: v.cuda().requires_grad_(n in wanted) for n, v in t.items()}
        out = _ops().residual_norm(leaves["x"], leaves["y"], leaves["weight"])
        grads = torch.autograd.grad(out, [leaves[n] for n in wanted], [d_s.cuda(), d_h.cuda()])
        ref = lm.residual(t["x"].double(), t["y"].double(), t["weight"].double(), None, None, 1.0, 1e-6, d_s.double(), d_h.double())
        for g in grads:
            lm.assert_within(g, ref["x"][0], lm.rounded(*ref["x"], F32), "plain")


def test_residual_norm_gradients_of_one_tensor_and_of_leaves():
    """x and y one tensor; the plain join's gradients of two leaves are tensors of their own."""
    t, d_s, d_h = _join_inputs(5, 72, F32, False, False)
    x, w = t["x"].cuda().requires_grad_(True), t["weight"].cuda()
    for scale in (1.0, 0.5):
        (dx,) = torch.autograd.grad(_ops().residual_norm(x, x, w, scale=scale), [x], [d_s.cuda(), d_h.cuda()])
        ref = lm.residual(t["x"].double(), t["x"].double(), t["weight"].double(), None, None, scale, 1e-6, d_s.double(), d_h.double())
        total = ref["x"][0] + ref["y"][0]
        err = sum(lm.rounded(*ref[n], F32) for n in ("x", "y"))
        lm.assert_within(dx, total, lm.rounded(total, err, F32), "x twice")
    y = t["y"].cuda().requires_grad_(True)
    s, h = _ops().residual_norm(x, y, w)
    (s.sum() + h.sum()).backward()
    kept = y.grad.clone()
    x.grad.zero_()
    assert torch.equal(y.grad, kept) and kept.abs().sum() > 0


def test_residual_norm_recorded_backward():
    t, d_s, d_h = _join_inputs(3, 20, F32, True, True)
    out = []
    for dt, dev in ((F32, "cuda"), (torch.float64, "cpu")):
        leaves = [v.to(dev, dt).requires_grad_(True) for v in t.values()]
        x, y, w, p, g = leaves
        if dev == "cuda":
            s, h = _ops().residual_norm(x, y, w, p, g, scale=0.5, eps=1e-3)
        else:
            s = x + 0.5 * y * (y.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * p * g.sigmoid()
            h = s * (s.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * w
        grads = torch.autograd.grad([s, h], leaves, [d_s.to(dev, dt), d_h.to(dev, dt)], create_graph=True)
        out.append(list(grads) + list(torch.autograd.grad(sum(q.square().sum() for q in grads), leaves)))
    for a, b in zip(*out):
        assert (a.double().cpu() - b).abs().max() <= 1e-4 * (1 + b.abs().max())


# ---------------------------------------------------------------- together


def _tiny_lm(ids, labels, embedding, joins, head, ops=None):
    """Tokens in, loss out: lookup, two joins around elementwise blocks, head."""
    if ops is None:
        def norm(t, w):
            return t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w

        x = embedding[ids] * 4.0
        h = x
        for w, p in joins:
            x = x + 0.5 * norm(torch.tanh(h), p) * torch.sigmoid(h)
            h = norm(x, w)
        return torch.nn.functional.cross_entropy((h @ head.t()).reshape(-1, head.shape[0]), labels.reshape(-1))
    x = ops.embed_tokens(ids, embedding, scale=4.0)
    h = x
    for w, p in joins:
        x, h = ops.residual_norm(x, torch.tanh(h), w, post_weight=p, gate=h, scale=0.5)
    return ops.token_loss(h @ head.t(), labels)


def _tiny_inputs():
    V, D = 211, 48
    params = [_randn(1, V, D) * 0.3] + [1 + 0.1 * _randn(i, D) for i in range(2, 6)] + [_randn(6, V, D) * 0.2]
    ids = _randint(7, V, 3, 50)
    labels = torch.cat([ids[:, 1:], torch.full((3, 1), -100)], 1)
    labels[2, 20:] = -100
    return ids, labels, params


def _unpack(params):
    return params[0], [(params[1], params[2]), (params[3], params[4])], params[5]


def test_together_trains_with_the_gradients_of_the_formulas():
    ids, labels, params = _tiny_inputs()
    ref = [p.double().requires_grad_(True) for p in params]
    loss = _tiny_lm(ids, labels, *_unpack(ref))
    want = torch.autograd.grad(loss, ref)
    got_p = [p.cuda().requires_grad_(True) for p in params]
    got_loss = _tiny_lm(ids.cuda(), labels.cuda(), *_unpack(got_p), ops=_ops())
    got = torch.autograd.grad(got_loss, got_p)
    assert abs(got_loss.item() - loss.item()) < 1e-5
    # fp32 through two joins and two products of 48 terms: 2^-18 of each gradient's largest value
    for g, r in zip(got, want):
        assert (g.double().cpu() - r).abs().max() <= 2.0**-18 * r.abs().max()


def test_together_captured_and_replayed():
    """A captured training step on changing inputs, replayed with eager work
    between; two graphs that interleave."""
    ids, labels, params = _tiny_inputs()
    ops = _ops()

    def step(ids, labels, params):
        loss = _tiny_lm(ids, labels, *_unpack(params), ops=ops)
        lp = ops.token_logprobs(params[5][:40], torch.arange(40, device="cuda"), top_k=3)
        return [loss.detach(), *torch.autograd.grad(loss, params), *(t.detach() for t in lp)]

    graphs = []
    side = torch.cuda.Stream()
    for seed in range(2):
        p = [t.cuda().requires_grad_(True) for t in params]
        i, lab = ids.cuda(), labels.cuda()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(i, lab, p)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(i, lab, p)
        graphs.append((g, i, lab, p, out))
    for n in range(4):
        for g, i, lab, p, out in graphs:
            i.copy_(_randint(n, 211, 3, 50))
            g.replay()
        torch.cuda.synchronize()
        for g, i, lab, p, out in graphs:
            fresh = [t.detach().clone().requires_grad_(True) for t in p]
            for a, b in zip(out, step(i, lab, fresh)):
                assert torch.equal(a, b)
            with torch.no_grad():
                p[0].mul_(1.01)


def test_together_on_another_stream():
    ids, labels, params = _tiny_inputs()
    p = [t.cuda().requires_grad_(True) for t in params]
    want = torch.autograd.grad(_tiny_lm(ids.cuda(), labels.cuda(), *_unpack(p), ops=_ops()), p)
    side = torch.cuda.Stream()
    i, lab = ids.cuda(), labels.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = [t.detach().clone().requires_grad_(True) for t in p]
        got = torch.autograd.grad(_tiny_lm(i, lab, *_unpack(q), ops=_ops()), q)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- sizes and uses past the ordinary


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: their last rows as in calls of their own."""
    ops = _ops()
    rows, V = 70001, 32001
    assert rows * V > 2**31
    x = torch.zeros(rows, V, dtype=BF, device="cuda")
    last = (_randn(1, 3, V) * 3).to(BF).cuda()
    x[-3:] = last
    tokens = torch.full((rows,), 5, device="cuda")
    tokens[-3:] = torch.tensor([0, V - 1, 77])
    x.requires_grad_(True)
    got = ops.token_logprobs(x, tokens, top_k=3)
    ends = last.cpu().double()
    ref = lm.logprobs(ends, tokens[-3:].cpu(), 3)
    for name, value in (("logprob", got.logprob), ("entropy", got.entropy), ("top", got.top_logprobs)):
        lm.assert_within(value[-3:], *ref[name], name)
    assert torch.equal(got.top_ids[-3:].cpu(), ref["ids"]) and got.top_ids[5].tolist() == [0, 1, 2]
    d = torch.zeros(rows)
    d[-3:] = torch.tensor([1.0, -2.0, 0.5])
    (dx,) = torch.autograd.grad(got.logprob, [x], d.cuda())
    lm.assert_within(dx[-3:], *lm.logprobs_grad(ends, tokens[-3:].cpu(), None, d[-3:].double(), None, None, BF), "dx")
    assert not dx[:-3].any()
    del x, dx, got

    n, D = 70001, 32001
    w = _randn(2, 3, D).to(BF).cuda().requires_grad_(True)
    ids = torch.zeros(n, dtype=torch.int64, device="cuda")
    ids[-2:] = torch.tensor([1, 2])
    out = ops.embed_tokens(ids, w, padding_idx=0)
    assert torch.equal(out[-2:], w[1:]) and torch.equal(out[-3], w[0])
    dy = torch.zeros(n, D, dtype=BF, device="cuda")
    dy[-2:] = _randn(3, 2, D).to(BF).cuda()
    (dw,) = torch.autograd.grad(out, [w], dy)
    assert torch.equal(dw[1:], dy[-2:]) and not dw[0].any()
    del out, dy, dw

    rows, D = 270001, 8001
    assert rows * D > 2**31
    t, d_s, d_h = _join_inputs(3, D, BF, False, False, seed=4)
    x, y = (torch.zeros(rows, D, dtype=BF, device="cuda") for _ in range(2))
    x[-3:], y[-3:] = t["x"], t["y"]
    weight = t["weight"].cuda()
    s, h = ops.residual_norm(x.requires_grad_(True), y, weight)
    ref = lm.residual(*(v.double() for v in (t["x"], t["y"], t["weight"])), None, None, 1.0, 1e-6, d_s.double(), d_h.double())
    lm.assert_within(s[-3:], ref["s"][0], lm.rounded(*ref["s"], BF), "s")
    lm.assert_within(h[-3:], ref["h"][0], lm.rounded(*ref["h"], BF), "h")
    dh = torch.zeros_like(y)
    dh[-3:] = d_h
    (dx,) = torch.autograd.grad(h, [x], dh)
    ref = lm.residual(*(v.double() for v in (t["x"], t["y"], t["weight"])), None, None, 1.0, 1e-6, 0 * d_s.double(), d_h.double())
    lm.assert_within(dx[-3:], ref["x"][0], lm.rounded(*ref["x"], BF), "dx")
    assert not dx[:-3].any()


@pytest.mark.parametrize("rows,V,dtype", [(2100, 32000, BF), (1100, 32000, F32), (40000, 2048, F16), (2100, 32004, BF)])
def test_rows_past_the_caches(rows, V, dtype):
    """Logits and gradients of 128 MiB or more, in whole lines and not: the same
    bits as in calls of fewer rows, and the formulas' on some."""
    ops = _ops()
    x = (torch.randn(rows, V, device="cuda", generator=torch.Generator("cuda").manual_seed(V)) * 3).to(dtype)
    assert x.numel() * x.element_size() >= 128 << 20
    tokens = _randint(rows, V, rows).cuda()
    with torch.no_grad():
        plain = ops.token_logprobs(x, tokens)
        plain_loss = ops.token_loss(x, tokens)
    x.requires_grad_(True)
    got = ops.token_logprobs(x, tokens)
    loss = ops.token_loss(x, tokens)
    assert torch.equal(plain.logprob, got.logprob) and torch.equal(plain.entropy, got.entropy) and torch.equal(plain_loss, loss)
    d, e = _randn(1, rows), _randn(2, rows)
    (dx,) = torch.autograd.grad([got.logprob, got.entropy], [x], [d.cuda(), e.cuda()])
    (dl,) = torch.autograd.grad(loss, [x])
    some = torch.tensor([0, 1, rows // 2, rows - 1])
    xd, td = x.detach()[some.cuda()].cpu().double(), tokens.cpu()[some]
    lm.assert_within(got.logprob[some.cuda()], *lm.logprobs(xd, td)["logprob"], "logprob")
    lm.assert_within(dx[some.cuda()], *lm.logprobs_grad(xd, td, None, d[some].double(), e[some].double(), None, dtype), "dx")
    lm.assert_within(dl[some.cuda()], *lm.logprobs_grad(xd, td, None, torch.full((4,), -1.0 / rows).double(), None, None, dtype), "dl")
    for part in (slice(0, rows // 3), slice(rows // 3, rows // 2 + 7)):
        own = x.detach()[part].clone().requires_grad_(True)
        r = ops.token_logprobs(own, tokens[part])
        (own_dx,) = torch.autograd.grad([r.logprob, r.entropy], [own], [d.cuda()[part], e.cuda()[part]])
        assert torch.equal(own_dx, dx[part]) and torch.equal(r.logprob, got.logprob[part])


def test_two_backward_passes_and_calls_of_two_threads():
    """A retained graph gives the same gradients again, and calls of two threads on streams of their own do not meet."""
    from concurrent.futures import ThreadPoolExecutor

    ids, labels, params = _tiny_inputs()
    ops = _ops()

    def gradients(stream):
        with torch.cuda.stream(stream):
            p = [t.cuda().requires_grad_(True) for t in params]
            lab = labels.cuda()
            loss = _tiny_lm(ids.cuda(), lab, *_unpack(p), ops=ops)
            first = torch.autograd.grad(loss, p, retain_graph=True)
            second = torch.autograd.grad(loss, p)
            big = ops.token_logprobs(_randn(3, 2, 140000).cuda(), torch.tensor([5, 139999]).cuda(), top_k=5)
            stream.synchronize()
        return [loss.detach(), *first, *second, big.logprob, big.entropy, big.top_logprobs, big.top_ids]

    want = gradients(torch.cuda.Stream())
    k = len(params)
    for a, b in zip(want[1:1 + k], want[1 + k:1 + 2 * k]):
        assert torch.equal(a, b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    with ThreadPoolExecutor(2) as pool:
        for _ in range(3):
            for got in pool.map(gradients, streams):
                assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_inference_tensors_and_frozen_inputs():
    ops = _ops()
    with torch.inference_mode():
        x = _randn(1, 4, 33).cuda()
        t = torch.tensor([0, 1, 2, 32]).cuda()
        lp = ops.token_logprobs(x, t, top_k=1)
        loss = ops.token_loss(x, t)
        e = ops.embed_tokens(t, x)
        s, h = ops.residual_norm(x, x, torch.ones(33, device="cuda"))
    assert abs(loss.item() + lp.logprob.mean().item()) < 1e-5
    assert not (lp.logprob.requires_grad or e.requires_grad or s.requires_grad)
    assert torch.equal(s, x + x) and h.shape == x.shape
    frozen = ops.token_logprobs(x.clone(), t)  # grad mode, nothing to record
    assert not frozen.logprob.requires_grad and torch.equal(frozen.logprob, lp.logprob)


def test_embed_gradient_of_ids_that_share_a_remainder():
    """Ids whose positions one workgroup of the sort places, few and many of them at a time."""
    V, D, n = 60000, 8, 5000
    for ids in (_randint(1, 200, n) * 256 + 3, _randint(2, 3, n) * 256, (torch.arange(n) % 230) * 256 + 255,
                torch.where(_randint(3, 2, n) == 0, _randint(4, 230, n) * 256 + 7, torch.full((n,), 7))):
        w = torch.zeros(V, D, device="cuda", requires_grad=True)
        dy = _randn(5, n, D)
        (dw,) = torch.autograd.grad(_ops().embed_tokens(ids.cuda(), w), [w], dy.cuda())
        lm.assert_within(dw, *lm.embed_grad(ids, dy.double(), V, 1.0, -1, F32), "dw")


@pytest.mark.parametrize("n", [16384, 16385, 20011, 33000])
def test_embed_gradient_of_many_mixed_ids(n):
    """More positions than the sort keeps between counting and placing, with
    several ids to a workgroup: of a whole vocabulary, of few ids, and of ids
    that share a remainder, few and many of them at a time."""
    V, D = 5000, 24
    same = torch.where(_randint(5, 2, n) == 0, _randint(6, 19, n) * 256 + 7, torch.full((n,), 7))
    impossible = torch.where(_randint(7, 3, n) == 0, torch.tensor(V), _randint(8, V, n))
    for ids in (_randint(1, V, n), (_randint(2, V, n).double() ** 3 / V**2).long(), _randint(3, 19, n) * 256 + 3, same, impossible):
        w = torch.zeros(V, D, device="cuda", requires_grad=True)
        dy = _randn(9, n, D)
        out = _ops().embed_tokens(ids.cuda(), w, padding_idx=11)
        (dw,) = torch.autograd.grad(out, [w], dy.cuda(), retain_graph=True)
        lm.assert_within(dw, *lm.embed_grad(ids, dy.double(), V, 1.0, 11, F32), "dw")
        assert torch.equal(dw, torch.autograd.grad(out, [w], dy.cuda())[0])
