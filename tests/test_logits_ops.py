"""Host-side checks of the operators on a model's logits: struct layouts against
the header, argument errors raised before any launch, refusals of the Python
entry points, calls that torch has to see, and the torch operations behind them
against the definitions (no GPU compute)."""

import ctypes

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import lm_bounds as lm
import logits_bounds as lb
from cyclic_flow_attention import Sampler, Sampling, _native, ops
from test_abi import _c_layout

VALUE, UNSUPPORTED, ALIGN = _native.CYFA_ERR_VALUE, _native.CYFA_ERR_UNSUPPORTED, _native.CYFA_ERR_ALIGN
INF, NAN = float("inf"), float("nan")


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("name", ["CyfaAdjustArgs", "CyfaSampleArgs", "CyfaDistillArgs"])
def test_struct_layout_matches_header(tmp_path, name):
    cls = getattr(_native, name)
    fields = [f for f, _ in cls._fields_]
    got = [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]
    assert got == _c_layout(tmp_path, name, fields)


def _caller(fn, cls, good):
    def call(grad, dtype=0, **change):
        a = cls(**{**good, **change})
        return getattr(_native.load_library(), fn)(ctypes.byref(a), dtype, grad, None)

    return call


def test_adjust_validates_before_launch():
    call = _caller("cyfa_adjust_logits", _native.CyfaAdjustArgs, dict(
        rows=4, inner=4, V=100, x=0x10000, x_row=100, y=0x20000, y_row=100, dy=0x30000, repetition=1.0))
    for grad in (0, 1):
        assert call(grad, dtype=3) == call(grad, V=0) == call(grad, rows=-1) == call(grad, inner=0) == call(grad, L=-1) == VALUE
        assert call(grad, x=None) == call(grad, y=None) == call(grad, L=3) == call(grad, n_tokens=-1) == VALUE
        assert call(grad, n_tokens=2) == call(grad, n_tokens=2, token_ids=0x40000) == VALUE
        assert call(grad, V=(1 << 28) + 1) == call(grad, L=1 << 31, history=0x40000) == UNSUPPORTED
        assert call(grad, n_tokens=_native.ADJUST_MAX_TOKENS + 1) == UNSUPPORTED
        assert call(grad, x=0x10001) == call(grad, dtype=1, y=0x20002) == call(grad, lengths=0x40004) == ALIGN
        assert call(grad, history=0x40004, wide=1) == call(grad, history=0x40002) == call(grad, bias=0x40002) == ALIGN
        assert call(grad, rows=0) == _native.CYFA_OK
    assert call(1, dy=None) == call(1, y=0x10000) == call(1, y=0x30000) == VALUE
    assert _native.load_library().cyfa_adjust_logits(None, 0, 0, None) == VALUE


def test_sample_validates_before_launch():
    call = _caller("cyfa_sample_tokens", _native.CyfaSampleArgs, dict(
        rows=4, inner=4, row_stride=100, V=100, x=0x10000, uniform=0x20000, ids=0x30000, logprob=0x40000, temperature=1.0))
    assert call(1) == call(0, dtype=-1) == call(0, V=0) == call(0, rows=-1) == call(0, inner=0) == VALUE
    assert call(0, x=None) == call(0, uniform=None) == call(0, ids=None) == call(0, logprob=None) == VALUE
    assert call(0, V=(1 << 28) + 1) == UNSUPPORTED
    assert call(0, x=0x10001) == call(0, uniform64=0x20004) == call(0, top_ks=0x20004) == call(0, top_ps=0x20002) == ALIGN
    assert call(0, rows=0) == _native.CYFA_OK
    assert _native.load_library().cyfa_sample_tokens(None, 0, 0, None) == VALUE
    size = _native._sample_bytes(4, 50000)  # few rows of many columns are shared out
    assert size > 0 and _native._sample_bytes(4, 100) == _native._sample_bytes(4096, 50000) == _native._sample_bytes(0, 50000) == 0
    wide = dict(V=50000, row_stride=50000)
    assert call(0, **wide) == call(0, workspace=0x50000, workspace_bytes=size - 1, **wide) == _native.CYFA_ERR_WORKSPACE
    assert call(0, workspace=0x50008, workspace_bytes=size, **wide) == ALIGN


def test_distill_validates_before_launch():
    call = _caller("cyfa_distill_loss", _native.CyfaDistillArgs, dict(
        rows=4, inner=4, row_stride=100, V=100, x=0x10000, k=5, ids=0x20000, values=0x30000, temperature=1.0, kept=0x40000,
        loss=0x50000, total=0x60000, parts=0x90000, d_loss=0x70000, dx=0x80000))
    for grad in (0, 1):
        assert call(grad, dtype=3) == call(grad, V=0) == call(grad, rows=-1) == call(grad, inner=0) == call(grad, k=0) == VALUE
        assert call(grad, temperature=0.0) == call(grad, temperature=NAN) == call(grad, temperature=INF) == VALUE
        assert call(grad, temperature=2.0, tail=1) == call(grad, x=None) == call(grad, ids=None) == call(grad, total=None) == VALUE
        assert call(grad, k=_native.DISTILL_MAX_K + 1) == call(grad, V=(1 << 28) + 1) == UNSUPPORTED
        assert call(grad, tail=1, V=_native.DISTILL_MAX_TAIL_V + 1) == UNSUPPORTED
        assert call(grad, x=0x10001) == call(grad, ids=0x20004) == call(grad, values=0x30002) == ALIGN
    assert call(0, parts=0x90004) == ALIGN and call(0, parts=None) == VALUE
    assert call(0, loss=None) == call(1, d_loss=None) == call(1, dx=None) == call(0, kept=None) == VALUE
    assert call(1, rows=0) == _native.CYFA_OK
    assert _native.load_library().cyfa_distill_loss(None, 0, 0, None) == VALUE


def test_adjust_refuses():
    x, h = torch.zeros(3, 40), torch.zeros(3, 5, dtype=torch.int64)
    n = torch.zeros(3, dtype=torch.int64)
    adjust = ops.adjust_logits
    with pytest.raises(ValueError, match="GPU"):
        adjust(x, h)
    for bad, match in ((dict(lengths=n), "lengths"), (dict(history=h.float()), "int64 or int32"), (dict(history=h[:2]), "broadcast"),
                       (dict(history=h, lengths=n[:2]), "broadcast"), (dict(history=h, lengths=n.float()), "int64 or int32"),
                       (dict(history=h, repetition=0.0), "positive"), (dict(repetition=n), "float"),
                       (dict(presence=torch.zeros(2)), "broadcast"), (dict(bias=torch.zeros(39)), "broadcast"),
                       (dict(bias=torch.zeros(40, dtype=torch.int64)), "float"),
                       (dict(token_bias=(n[:, None], torch.zeros(3, 2))), "token_bias"),
                       (dict(token_bias=(torch.zeros(3, 1), torch.zeros(3, 1))), "int64 or int32"),
                       (dict(allowed=torch.ones(3, 39, dtype=torch.bool)), "allowed"), (dict(allowed=torch.ones(3, 40)), "bool"),
                       (dict(allowed=torch.ones(3, 1, dtype=torch.int32)), "allowed"),
                       (dict(allowed=torch.ones(2, 40, dtype=torch.bool)), "broadcast"), (dict(out=x[:2]), "out must"),
                       (dict(out=x.half()), "out must"), (dict(out=torch.zeros(40, 3).t()), "contiguous rows"),
                       (dict(out=torch.zeros(1, 40).expand(3, 40)), "one element"), (dict(history=torch.tensor(3)), "scalar")):
        with pytest.raises(ValueError, match=match):
            adjust(x, **bad)
    with pytest.raises(ValueError, match="vocabulary"):
        adjust(x[:, :0])
    with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
        adjust(x.double())
    with pytest.raises(NotImplementedError, match="token biases"):
        adjust(x, token_bias=(torch.zeros(1025, dtype=torch.int64), torch.zeros(1025)))
    with pytest.raises(NotImplementedError, match="no gradient"):
        adjust(x, bias=torch.zeros(40, requires_grad=True))
    with pytest.raises(NotImplementedError, match="no out"):
        adjust(x.clone().requires_grad_(True), out=x)
    buffer = torch.zeros(4, 40)
    with pytest.raises(ValueError, match="themselves"):
        adjust(buffer[:3], out=buffer[1:])


def test_sample_refuses():
    x, u = torch.zeros(3, 40), torch.zeros(3)
    sample = ops.sample_tokens
    with pytest.raises(ValueError, match="GPU"):
        sample(x, u)
    for bad, match in ((dict(temperature=-1.0), "temperature"), (dict(temperature=NAN), "temperature"), (dict(top_k=-1), "top_k"),
                       (dict(top_p=0.0), "top_p"), (dict(top_p=1.5), "top_p"), (dict(min_p=-0.1), "min_p"), (dict(min_p=2.0), "min_p"),
                       (dict(top_k=u), "int64 or int32"), (dict(top_p=torch.ones(3, dtype=torch.int64)), "float"),
                       (dict(temperature=torch.ones(2)), "broadcast")):
        with pytest.raises(ValueError, match=match):
            sample(x, u, **bad)
    with pytest.raises(ValueError, match="uniform"):
        sample(x, u[:2])
    with pytest.raises(ValueError, match="fp32 or fp64"):
        sample(x, u.half())
    with pytest.raises(ValueError, match="vocabulary"):
        sample(x[:, :0], u)
    with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
        sample(x.double(), u)


def test_distill_refuses():
    x, ids, v = torch.zeros(3, 40), torch.zeros(3, 5, dtype=torch.int64), torch.zeros(3, 5)
    distill = ops.distill_loss
    with pytest.raises(ValueError, match="GPU"):
        distill(x, ids, v)
    for args, kw, match in (((x, ids[:2], v[:2]), {}, "top_ids"), ((x, ids[:, :0], v[:, :0]), {}, "top_ids"), ((x, ids[0], v[0]), {}, "top_ids"),
                            ((x, v, v), {}, "int64 or int32"), ((x, ids, v[:, :4]), {}, "top_logprobs"), ((x, ids, ids), {}, "float"),
                            ((x, ids, v), dict(temperature=0.0), "positive"), ((x, ids, v), dict(temperature=NAN), "positive"),
                            ((x, ids, v), dict(temperature=2.0, tail=True), "tail"), ((x, ids, v), dict(weights=v), "weights"),
                            ((x, ids, v), dict(temperature=torch.tensor(1.0)), "number"), ((x[:, :0], ids, v), {}, "vocabulary")):
        with pytest.raises(ValueError, match=match):
            distill(*args, **kw)
    with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
        distill(x.double(), ids, v)
    with pytest.raises(NotImplementedError, match="at most 256"):
        distill(x, ids[:, :1].expand(3, 257), v[:, :1].expand(3, 257))
    with pytest.raises(NotImplementedError, match="columns"):
        distill(torch.zeros(1, (1 << 19) + 1), ids[:1], v[:1], tail=True)
    for bad in (dict(top_logprobs=v.clone().requires_grad_(True)), dict(top_logprobs=v, weights=torch.ones(3, requires_grad=True))):
        with pytest.raises(NotImplementedError, match="no gradient"):
            distill(x, ids, **bad)


def test_sampler_refuses():
    with pytest.raises(ValueError, match="prompts"):
        Sampler(Sampling(), torch.zeros(3, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="room"):
        Sampler(Sampling(), torch.zeros(3, 2, dtype=torch.int64), -1)
    sampler = Sampler(Sampling(), torch.zeros(3, 2, dtype=torch.int64), 1)
    sampler.take()
    with pytest.raises(ValueError, match="room"):
        sampler.next(torch.zeros(3, 9))


    sampler = Sampler(Sampling(), torch.zeros(1, 2, dtype=torch.int64), 4)
    for shape in ((3, 9), (9,), (1, 1, 9)):
        with pytest.raises(ValueError, match="sequences"):
            sampler.next(torch.zeros(shape))
    for lengths in (torch.tensor([1, 2]), torch.tensor([1, 2, 3]), torch.tensor([0, -1, 2]), torch.tensor([1.0, 1.0, 1.0])):
        with pytest.raises(ValueError, match="lengths"):
            Sampler(Sampling(), torch.zeros(3, 2, dtype=torch.int64), 1, lengths)


def test_out_apart_from_what_is_read():
    """out may lie beside the logits and the options in one allocation, not among them."""
    whole = torch.zeros(4, 3, 8)
    with pytest.raises(ValueError, match="GPU device"):  # (no other objection)
        ops.adjust_logits(whole[0], bias=whole[1], out=whole[2])
    for out, kw in ((whole.view(-1)[4:28].view(3, 8), {}), (whole[:, 0, :][:3], {}), (whole[2], dict(bias=whole[2, 1])),
                    (whole[0], dict(bias=whole[0])), (whole[3], dict(presence=whole[3, 0, 4:7])),
                    (whole[1], dict(token_bias=(torch.zeros(2, dtype=torch.int64), whole[1, 2, 3:5])))):
        with pytest.raises(ValueError, match="apart"):
            ops.adjust_logits(whole[0], out=out, **kw)


def test_generate_refuses_two_settings():
    from cyclic_flow_attention.generation import generate

    for kw in (dict(temperature=0.5), dict(top_p=0.5), dict(seed=1)):
        with pytest.raises(ValueError, match="Sampling"):
            generate(None, [1], sampling=Sampling(), **kw)


# ---------------------------------------------------------------- torch operations in place of the kernels


@pytest.fixture
def no_launch(monkeypatch):
    def launch(*args, **kwargs):
        raise AssertionError("a kernel was launched")

    monkeypatch.setattr(_native, "require_device", lambda *tensors: tensors[0].device)
    for name in ("adjust", "sample", "distill_loss", "distill_loss_grad"):
        monkeypatch.setattr(_native, name, launch)


HISTORY = torch.tensor([[1, 4, 4, 2, -1], [0, 10, 11, 0, 3], [5, 5, 5, 5, 5], [9, 8, 7, 6, 5], [-100] * 5])
LENGTHS, PROMPTS = torch.tensor([5, 4, 5, 0, 5]), torch.tensor([1, 0, 5, 0, 2])
IDS = torch.tensor([[3, 1, 7], [0, -100, 4], [2, 2, 5], [-100, -100, 11], [10, 9, 8]])
VALUES = torch.tensor([[-0.5, -1.5, -2.5]]).expand(5, 3)
ALLOWED = _randn(9, 5, 11) > -0.5
BIAS = _randn(8, 11)


def _adjust(x):
    return (ops.adjust_logits(x, HISTORY, LENGTHS, PROMPTS, repetition=1.5, presence=0.25, frequency=0.5, bias=BIAS,
                              token_bias=(torch.tensor([2, 2, 12]), torch.tensor([1.0, 2.0, 3.0])), allowed=ALLOWED),)


def _adjust64(x):
    n, m = torch.zeros(5, 11), torch.zeros(5, 11)
    for r in range(5):
        for i, t in enumerate(HISTORY[r, :LENGTHS[r]].tolist()):
            if 0 <= t < 11:
                n[r, t] += 1
                m[r, t] += i >= PROMPTS[r]
    y = torch.where(n > 0, torch.where(x > 0, x / 1.5, x * 1.5), x) - m * 0.5 - (m > 0) * 0.25 + BIAS
    y = y + torch.zeros(11, dtype=torch.float64).index_fill(0, torch.tensor([2]), 3.0)
    return (torch.where(ALLOWED, y, -INF),)


def _distill(x, **kw):
    return (ops.distill_loss(x, IDS, VALUES, **kw),)


def _distill64(x, T=1.0, tail=False):
    lq, total = torch.log_softmax(x / T, -1), 0.0
    for r in (0, 1, 2, 4):
        at = IDS[r][(IDS[r] >= 0) & (IDS[r] < 11)]
        t = VALUES[r][(IDS[r] >= 0) & (IDS[r] < 11)].double()
        p = t.exp() if tail else torch.softmax(t / T, 0)
        total = total + (p * (p.log() - lq[r, at])).sum()
        if tail:
            others = torch.tensor([c for c in range(11) if c not in at.tolist()])
            rest = 1 - p.sum()
            if rest > 0:
                total = total + rest * (rest.log() - torch.logsumexp(lq[r, others], 0))
    return (total / 4,)


# name: (call, the same in 64 bits)
CALLS = {
    "adjust_logits": (lambda x: tuple(y.masked_fill(~ALLOWED, 0.0) for y in _adjust(x)), lambda x: tuple(y.masked_fill(~ALLOWED, 0.0) for y in _adjust64(x))),
    "distill_loss": (lambda x: _distill(x, temperature=2.0), lambda x: _distill64(x, T=2.0)),
    "distill_tail": (lambda x: _distill(x, tail=True), lambda x: _distill64(x, tail=True)),
}


def _close(got, want, what):
    assert len(got) == len(want)
    for a, b in zip(got, want):  # fp32 through reductions of at most 11 terms
        assert (a.double() - b).abs().max() <= 2.0**-18 * (1 + b.abs().max()), what


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_derivatives(no_launch, name):
    fn, fn64 = CALLS[name]
    x, dx = _randn(1, 5, 11), _randn(2, 5, 11)
    want = torch.func.jvp(fn64, (x.double(),), (dx.double(),))[1]
    _close(torch.func.jvp(fn, (x,), (dx,))[1], want, name)


@pytest.mark.parametrize("name", CALLS)
def test_transforms(no_launch, name):
    fn, fn64 = CALLS[name]
    x = torch.stack([_randn(1, 5, 11), 2 * _randn(2, 5, 11)])
    got = torch.vmap(fn)(x)
    for i in range(2):
        _close([o[i] for o in got], fn64(x[i].double()), name)
    got = torch.func.grad(lambda t: fn(t)[0].sum())(x[0])
    _close([got], [torch.func.grad(lambda t: fn64(t)[0].sum())(x[0].double())], name)


@pytest.mark.filterwarnings("ignore")  # (tracing warns of the checks of arguments)
@pytest.mark.parametrize("name", CALLS)
def test_traced_and_compiled_calls_compute(no_launch, name):
    fn, fn64 = CALLS[name]
    x, other = _randn(1, 5, 11), _randn(3, 5, 11)
    want = fn64(other.double())
    with torch.no_grad():
        _close(make_fx(fn)(x)(other), want, name)
        _close(torch.jit.trace(fn, (x,), check_trace=False)(other), want, name)
        graph = torch.compile(fn, backend="eager", fullgraph=True)
        graph(x)
        _close(graph(other), want, name)


def test_subclasses_and_modes(no_launch):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.n += 1
            return func(*args, **(kwargs or {}))

    class Own(torch.Tensor):
        pass

    x, u = _randn(1, 5, 11), torch.rand(5, generator=torch.Generator().manual_seed(1))
    for fn, fn64 in CALLS.values():
        with Count() as mode:
            _close(fn(x), fn64(x.double()), "mode")
        assert mode.n > 2
        got = fn(x.as_subclass(Own))
        assert all(type(o) is Own for o in got)
    with Count():
        ids, logprob = ops.sample_tokens(x, u, temperature=0.7, top_k=5, top_p=0.8)
        out = torch.empty_like(x)
        assert ops.adjust_logits(x, bias=BIAS, out=out) is out and torch.equal(out, x + BIAS)
    for r in range(5):
        want = lb.choice(x[r].double().numpy(), float(u[r]), 0.7, 5, 0.8, 0.0)
        assert ids[r] == want[0] and abs(logprob[r] - want[1]) < 1e-6


def test_the_torch_operations_keep_the_definitions(no_launch):
    """Rows without probabilities, greedy rows, settings of each row's own."""
    x = torch.stack([torch.tensor([1.0, 3.0, 3.0, -0.0, 0.0, 2.0])] * 8)
    x[1, 4] = NAN
    x[2, 0] = INF
    x[3] = -INF
    x[4, :] = -INF
    x[4, 2] = -3.0
    u = torch.tensor([0.4, 0.1, 0.2, 0.3, 0.9, 0.0, 1.0, NAN])
    T = torch.tensor([0.0, 1, 1, 1, 1, 1, 1, 1])
    with forward_ad.dual_level():
        r = ops.sample_tokens(x, u, temperature=T, top_k=torch.tensor([0, 0, 0, 0, 0, 1, 2, 1], dtype=torch.int32))
    assert r.ids[:6].tolist() == [1, 4, 0, 0, 2, 1] and r.ids[6] == 2 and r.logprob[0] == 0 and r.logprob[1:4].isnan().all()
    assert r.logprob[4] == 0 and abs(r.logprob[6] - np.log(0.5)) < 1e-6


def test_recorded_backward_passes(no_launch):
    """The torch operations behind a recorded backward pass against the formulas' second derivatives."""
    from cyclic_flow_attention.ops import distill, sampling

    x = _randn(4, 5, 11).requires_grad_(True)
    weights = torch.tensor([1.0, 2.0, 0.0, 1.0, 0.5])
    loss = distill._plain(x, IDS, VALUES, weights, 1.0, True)
    (dx,) = torch.autograd.grad(loss, [x], create_graph=True)
    (ddx,) = torch.autograd.grad(dx.square().sum(), [x])
    (ref, _), (rdx, _) = lb.distill(x.detach().double(), IDS, VALUES.double(), 1.0, True, weights, torch.float32)
    assert abs(loss.item() - ref) < 1e-5 and (dx.double() - rdx).abs().max() < 1e-5
    h = 1e-4
    d = _randn(5, 5, 11).double()
    quotient = sum(s * lb.distill(x.detach().double() + s * h * d, IDS, VALUES.double(), 1.0, True, weights, torch.float32)[1][0].square().sum()
                   for s in (1, -1)) / (2 * h)
    assert abs(quotient - (ddx.double() * d).sum()) < 1e-4
    n, _, allowed = sampling._tables(x.detach(), HISTORY, LENGTHS, PROMPTS, ALLOWED)
    assert n[0].tolist() == [0, 1, 1, 0, 2, 0, 0, 0, 0, 0, 0] and n[1].tolist() == [2, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1] and not n[3:].any()
    bits = torch.tensor([[0b101, 1 << 3], [-1, 0b1]], dtype=torch.int32)
    words = sampling._tables(torch.zeros(2, 36), None, None, None, bits)[2]
    assert words[0].nonzero()[:, 0].tolist() == [0, 2, 35] and words[1].nonzero()[:, 0].tolist() == list(range(33))


@pytest.mark.parametrize("T", [0.25, 1.0])
def test_a_teachers_logits_of_any_size(no_launch, T):
    from cyclic_flow_attention.ops import distill

    x, ids = _randn(1, 3, 20), torch.arange(12).view(3, 4)
    values = torch.zeros(3, 4)
    values[2] = torch.arange(4.0)
    far = values + 2.0**16
    far[0], far[1] = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    near, much = (distill._plain(x, ids, v, None, T, False) for v in (values, far))
    assert torch.equal(near, much) and near.isfinite()


@pytest.mark.parametrize("tail,T", [(False, 1.0), (False, 3.0), (True, 1.0)])
def test_distillation_without_a_rest_or_rows(no_launch, tail, T):
    """Teachers that know every token, rows that do not count, values of -inf."""
    from cyclic_flow_attention.ops import distill

    x = _randn(6, 3, 4)
    x[2, 1] = -INF
    ids = torch.tensor([[0, 1, 2, 3], [1, 1, 7, -1], [0, 1, 2, 3]])
    values = torch.log_softmax(_randn(7, 3, 4), -1)
    values[2, 1] = -INF
    (ref, _), (rdx, _) = lb.distill(x.double(), ids, values.double(), T, tail, None, torch.float32)
    xg = x.clone().requires_grad_(True)
    loss = distill._plain(xg, ids, values, None, T, tail)
    (dx,) = torch.autograd.grad(loss, [xg])
    assert abs(loss.item() - ref) < 1e-5 and (dx.double() - rdx).abs().max() < 1e-5
    none = distill._plain(x, torch.full_like(ids, -100), values, None, T, tail)
    assert none.isnan()
    some = distill._plain(torch.cat([x[:1], torch.full((1, 4), NAN)]), ids[:2], values[:2], torch.tensor([1.0, 0.0]), T, tail)
    (ref, _), _ = lb.distill(x[:1].double(), ids[:1], values[:1].double(), T, tail, None, torch.float32)
    assert abs(some.item() - ref) < 1e-5
