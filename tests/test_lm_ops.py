"""Host-side checks of the operators around a model's blocks: struct layouts
against the header, argument errors raised before any launch, and refusals of
the Python entry points (no GPU compute)."""

import ctypes

import pytest
import torch

from cyclic_flow_attention import _native, ops
from test_abi import _c_layout

VALUE, UNSUPPORTED, ALIGN, WORKSPACE = (_native.CYFA_ERR_VALUE, _native.CYFA_ERR_UNSUPPORTED, _native.CYFA_ERR_ALIGN,
                                        _native.CYFA_ERR_WORKSPACE)


@pytest.mark.parametrize("name", ["CyfaLogprobArgs", "CyfaEmbedArgs", "CyfaResidualArgs"])
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


def test_logprobs_validates_before_launch():
    call = _caller("cyfa_logprobs", _native.CyfaLogprobArgs, dict(
        rows=4, inner=4, row_stride=100, V=100, x=0x10000, tokens=0x20000, logprob=0x30000, stats=0x40000, dx=0x50000))
    for grad in (0, 1):
        assert call(grad, dtype=3) == call(grad, V=0) == call(grad, rows=-1) == call(grad, inner=0) == VALUE
        assert call(grad, k=101) == call(grad, k=-1) == call(grad, x=None) == call(grad, tokens=None) == VALUE
        assert call(grad, k=33) == call(grad, V=(1 << 28) + 1) == UNSUPPORTED
        assert call(grad, x=0x10001) == call(grad, tokens=0x20004) == call(grad, stats=0x40002) == ALIGN
        assert call(grad, dtype=1, x=0x10002) == ALIGN
    assert call(0, logprob=None) == call(0, k=2) == call(0, k=2, top_ids=0x60000) == call(0, loss=0x60000) == VALUE
    assert call(1, dx=None) == call(1, stats=None) == call(1, d_entropy=0x60000) == call(1, d_top=0x60000, k=2) == VALUE
    assert call(1, d_loss=0x60000) == call(1, d_loss=0x60000, count=0x70000, d_logprob=0x70000) == VALUE
    assert call(0, rows=0) == call(1, rows=0) == _native.CYFA_OK
    lib = _native.load_library()
    size = lib.cyfa_logprobs_workspace_bytes
    assert size(4, 100, 0, 0) == size(512, 1 << 20, 5, 0) == size(-1, 8, 0, 0) == size(4, 0, 0, 0) == 0
    n = size(4, 1 << 20, 5, 0)
    assert n >= 4 * 16 * (12 + 5 * 8)
    assert call(0, V=1 << 20) == WORKSPACE
    assert call(0, V=1 << 20, workspace=0x90000, workspace_bytes=size(4, 1 << 20, 0, 0) - 1) == WORKSPACE
    assert call(0, V=1 << 20, workspace=0x90004, workspace_bytes=n) == ALIGN
    assert lib.cyfa_logprobs(None, 0, 0, None) == lib.cyfa_embed(None, 0, 0, None) == VALUE
    assert lib.cyfa_residual_norm(None, 0, 0, None) == VALUE


def test_embed_validates_before_launch():
    size = _native.load_library().cyfa_embed_grad_workspace_bytes
    n = size(100, 50, 64)
    assert n >= (100 + 51 + 64) * 4 and size(64, 50, 64) == 0  # few positions are not sorted
    assert size(-1, 50, 64) == size(1, 0, 64) == size(1, 50, 0) == size(1 << 31, 50, 64) == size(1, (1 << 26) + 1, 64) == 0
    call = _caller("cyfa_embed", _native.CyfaEmbedArgs, dict(
        n=100, V=50, D=64, ids=0x10000, weight=0x20000, out=0x30000, dy=0x40000, dweight=0x50000, padding=-1,
        workspace=0x60000, workspace_bytes=n))
    for grad in (0, 1):
        assert call(grad, dtype=-1) == call(grad, V=0) == call(grad, D=0) == call(grad, n=-1) == call(grad, ids=None) == VALUE
        assert call(grad, n=1 << 31) == call(grad, V=(1 << 26) + 1) == UNSUPPORTED
        assert call(grad, ids=0x10004) == call(grad, dy=0x40001) == call(grad, dtype=1, out=0x30002) == ALIGN
    assert call(0, out=None) == call(0, weight=None) == call(1, dy=None) == call(1, dweight=None) == VALUE
    assert call(1, workspace=None) == call(1, workspace_bytes=n - 1) == WORKSPACE
    assert call(1, workspace=0x60010) == ALIGN
    assert call(0, n=0) == _native.CYFA_OK


def test_residual_norm_validates_before_launch():
    size = _native.load_library().cyfa_residual_grad_workspace_bytes
    n = size(100, 64)
    assert n >= 2 * 64 * 4 and size(0, 64) > 0 and size(-1, 64) == size(1, 0) == 0
    call = _caller("cyfa_residual_norm", _native.CyfaResidualArgs, dict(
        rows=100, D=64, x=0x10000, y=0x20000, weight=0x30000, s=0x40000, h=0x50000, stats=0x60000, workspace=0x70000,
        workspace_bytes=n))
    for grad in (0, 1):
        assert call(grad, dtype=5) == call(grad, D=0) == call(grad, rows=-1) == call(grad, weight=None) == call(grad, x=None) == VALUE
        assert call(grad, D=8193) == UNSUPPORTED
        assert call(grad, y=0x20001) == call(grad, weight=0x30002) == call(grad, dtype=1, gate=0x80002) == ALIGN
    assert call(0, s=None) == call(0, h=None) == call(1, stats=None) == call(1, dgate=0x80000) == call(1, dpost=0x80000) == VALUE
    assert call(1, workspace=None) == call(1, workspace_bytes=n - 1) == WORKSPACE
    assert call(1, workspace=0x70008) == ALIGN
    assert call(0, rows=0) == _native.CYFA_OK


def test_token_ops_refuse():
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    for fn in (ops.token_logprobs, ops.token_loss):
        with pytest.raises(ValueError, match="GPU"):
            fn(x, t)
        with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
            fn(x.double(), t)
        with pytest.raises(ValueError, match="shape"):
            fn(x, t[:2])
        with pytest.raises(ValueError, match="vocabulary"):
            fn(x[:, :0], t)
        with pytest.raises(ValueError, match="vocabulary"):
            fn(torch.tensor(1.0), t)
        with pytest.raises(ValueError, match="int64 or int32"):
            fn(x, t.float())
    for k in (9, -1):
        with pytest.raises(ValueError, match="top_k"):
            ops.token_logprobs(x, t, top_k=k)
    with pytest.raises(NotImplementedError, match="at most 32"):
        ops.token_logprobs(torch.zeros(3, 64), t, top_k=33)


def test_embed_refuses():
    w, ids = torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        ops.embed_tokens(ids, w)
    with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
        ops.embed_tokens(ids, w.double())
    for bad in (w[0], w[:, :0], w[:0]):
        with pytest.raises(ValueError, match="vocabulary, width"):
            ops.embed_tokens(ids, bad)
    with pytest.raises(ValueError, match="int64 or int32"):
        ops.embed_tokens(ids.float(), w)
    with pytest.raises(ValueError, match="scale"):
        ops.embed_tokens(ids, w, scale=torch.tensor(2.0, requires_grad=True))
    for pad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            ops.embed_tokens(ids, w, padding_idx=pad)


def test_residual_norm_refuses():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    with pytest.raises(ValueError, match="GPU"):
        ops.residual_norm(x, x, w)
    with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
        ops.residual_norm(x.double(), x.double(), w)
    with pytest.raises(NotImplementedError, match="8192"):
        ops.residual_norm(torch.zeros(1, 8193), torch.zeros(1, 8193), torch.zeros(8193))
    for bad in (torch.tensor(1.0), x[:, :0]):
        with pytest.raises(ValueError, match="width"):
            ops.residual_norm(bad, bad, w)
    with pytest.raises(ValueError, match="scale"):
        ops.residual_norm(x, x, w, scale=torch.tensor(0.5, requires_grad=True))
    for y in (x[:2], x.half()):
        with pytest.raises(ValueError, match="y must be"):
            ops.residual_norm(x, y, w)
        with pytest.raises(ValueError, match="gate must be"):
            ops.residual_norm(x, x, w, gate=y)
    for bad in (w[:7], w.long(), w[None]):
        with pytest.raises(ValueError, match="weight must be"):
            ops.residual_norm(x, x, bad)
        with pytest.raises(ValueError, match="post_weight must be"):
            ops.residual_norm(x, x, w, post_weight=bad)


def test_recorded_backward_of_impossible_tokens_stays_off_the_table():
    """The torch operations behind a recorded backward pass never index with a
    token outside the vocabulary."""
    from cyclic_flow_attention.ops.vocab import _plain_logprobs, _plain_loss

    x = torch.randn(4, 6, requires_grad=True)
    tokens = torch.tensor([2, 6, -1, -100])
    logprob, entropy = _plain_logprobs(x, tokens, None, -100)
    want = torch.log_softmax(x.double(), -1)
    assert abs(logprob[0].item() - want[0, 2].item()) < 1e-6 and logprob[1:3].isnan().all() and logprob[3] == 0
    assert (entropy.double() + (want.exp() * want).sum(-1)).abs().max() < 1e-6
    assert _plain_loss(x, tokens, -100)[0].isnan()
    kept = torch.tensor([2, -100, 0, -100])
    loss = _plain_loss(x, kept, -100)[0]
    assert abs(loss.item() + (want[0, 2] + want[2, 0]).item() / 2) < 1e-6
    assert _plain_loss(x, torch.full((4,), -100), -100)[0].isnan()


def test_largest_sizes_are_the_librarys():
    lib = _native.load_library()
    size = lib.cyfa_embed_grad_workspace_bytes
    N, V, D = _native.EMBED_MAX_N, _native.EMBED_MAX_V, _native.EMBED_MAX_D
    assert min(size(N, 5, 1), size(65, V, 1), size(65, 5, D)) > 0
    assert size(N + 1, 5, 1) == size(65, V + 1, 1) == size(65, 5, D + 1) == 0
    size = lib.cyfa_logprobs_workspace_bytes
    V, k = _native.LOGPROBS_MAX_V, _native.LOGPROBS_MAX_TOP
    assert size(1, V, k, 0) > 0 and size(1, V + 1, k, 0) == size(1, V, k + 1, 0) == 0
    call = _caller("cyfa_residual_norm", _native.CyfaResidualArgs, dict(
        rows=0, D=1, x=0x10000, y=0x20000, weight=0x30000, s=0x40000, h=0x50000))
    assert call(0, D=_native.RESIDUAL_MAX_D) == _native.CYFA_OK and call(0, D=_native.RESIDUAL_MAX_D + 1) == UNSUPPORTED


@pytest.mark.parametrize("rows,V,k", [(1, 100, 3), (65, 1 << 20, 0), (64, 32768, 5), (3, 1 << 20, 7)])
def test_workspaces_are_what_the_library_asks_for(monkeypatch, rows, V, k):
    """Whatever the rule by which it shares rows out."""
    class Library:
        @staticmethod
        def cyfa_logprobs_workspace_bytes(*asked):
            assert asked == (rows, V, k, 1)
            return 768

    _native._logprobs_bytes.cache_clear()
    monkeypatch.setattr(_native, "load_library", Library)
    args = _native.CyfaLogprobArgs(rows=rows, V=V, k=k)
    workspace = _native._logprobs_workspace(args, torch.float32, torch.device("cpu"))
    _native._logprobs_bytes.cache_clear()
    assert workspace.numel() == args.workspace_bytes == 768 and args.workspace == workspace.data_ptr()
