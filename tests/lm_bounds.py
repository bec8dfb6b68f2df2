"""Float64 results of the operators around a model's blocks, from their
definitions, each with a bound on what fp32 computation and one rounding to the
result's dtype may be off by.

u is half a step of the dtype relative to the value. The fp32 bounds count: a
product, sum or conversion 2^-24 of its value, the hardware exponential,
reciprocal and root 2^-23, the exponential's argument t a further |t| 2^-22
(difference, product with log2 e, that constant), and a sum of n terms n 2^-24
of the sum of their magnitudes, n the longest chain of additions."""

import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
SMALLEST = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24, torch.float32: 2.0**-149}


def rounded(ref, err, dtype):
    """err with the rounding of ref to dtype on top (subnormals flush at worst)."""
    flush = 2.0**-126 if dtype != torch.float16 else SMALLEST[dtype]
    return err + HALF_STEP[dtype] * (ref.abs() + err) + flush


def assert_within(got, ref, err, what):
    got = got.detach().double().cpu()
    ref, err = ref.detach().cpu(), err.detach().cpu()
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} {tuple(ref.shape)}"
    # (a value past fp32's range rounds to infinity)
    same = (got == ref) | (got.isnan() & ref.isnan()) | (got.isinf() & (got == ref.float().double()))
    bad = ~(same | (ref.isfinite() & ((got - ref).abs() <= err)))
    if bad.any():
        i = tuple(int(j) for j in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {i}: "
                             f"{got[i].item()} for {ref[i].item()} +- {err[i].item()}")


def order(x, k):
    """The k largest of each row of x by (value, lower index first), NaN largest."""
    key = torch.where(x.isnan(), torch.full_like(x, float("inf")), x)
    nan = x.isnan().double()
    idx = torch.sort(key, dim=-1, descending=True, stable=True).indices
    idx = idx.gather(-1, torch.sort(nan.gather(-1, idx), dim=-1, descending=True, stable=True).indices)
    return idx[..., :k]


def log_softmax(x):
    """log softmax; the maximum goes first, as rows of the lowest value lose log V beside it."""
    x = x - x.amax(-1, keepdim=True)
    return x - x.exp().sum(-1, keepdim=True).log()


def logprobs(x, tokens, k=0, ignore=-100):
    """dict of (value, bound): logprob, entropy, top; and ids. x float64 [rows, V]."""
    V = x.shape[-1]
    lp = log_softmax(x)
    p = lp.exp()
    zero = torch.zeros((), dtype=x.dtype)
    plogp = torch.where(p == 0, zero, p * lp)
    entropy = -plogp.sum(-1)
    chain = (V / 256 + 64) * 2.0**-24
    d_sum = chain + 2.0**-22 + 2.0**-21 * (entropy + 1)  # of log S: the terms' errors weighted by p
    inside = (tokens >= 0) & (tokens < V)
    at = lp.gather(-1, tokens.clamp(0, V - 1)[:, None])[:, 0]
    logprob = torch.where(inside, at, torch.full_like(at, float("nan")))
    logprob = torch.where(tokens == ignore, zero, logprob)
    out = {"logprob": (logprob, d_sum + 2.0**-22 * at.abs()),
           "entropy": (entropy, (chain + 2.0**-21) * (2 + 2 * plogp.abs().sum(-1) + (p * lp.masked_fill(p == 0, 0.0).square()).sum(-1)))}
    if k:
        ids = order(x, k)
        top = lp.gather(-1, ids)
        out["top"] = (top, d_sum[:, None] + 2.0**-22 * top.abs())
        out["ids"] = ids
    return out


def logprobs_grad(x, tokens, ids, d_lp, d_ent, d_top, dtype, ignore=-100):
    """(dx, bound) of x float64 [rows, V]; cotangents float64 or None."""
    rows, V = x.shape
    zeros = torch.zeros(rows, dtype=x.dtype)
    d_lp = zeros if d_lp is None else d_lp.masked_fill(tokens == ignore, 0.0)
    d_ent = zeros if d_ent is None else d_ent
    lp = log_softmax(x)
    p = lp.exp()
    surprise = torch.where(p == 0, torch.zeros((), dtype=x.dtype), -lp)
    entropy = (p * surprise).sum(-1)
    own = torch.zeros_like(x)
    own.scatter_add_(1, tokens.clamp(0, V - 1)[:, None], d_lp[:, None])
    size = d_lp.abs()
    if d_top is not None:
        own.scatter_add_(1, ids, d_top)
        size = size + d_top.abs().sum(-1)
    dx = own - p * own.sum(-1, keepdim=True) + p * (surprise - entropy[:, None]) * d_ent[:, None]
    chain = (V / 256 + 64) * 2.0**-24
    terms = size[:, None] + d_ent.abs()[:, None] * (surprise + entropy[:, None] + 1)
    rel = 2.0**-20 + 2 * chain + 2.0**-21 * surprise
    err = p * terms * rel + 40 * 2.0**-24 * (own.abs() + dx.abs())
    dx = torch.where((size + d_ent.abs() == 0)[:, None], torch.zeros((), dtype=x.dtype), dx)
    return dx, rounded(dx, err, dtype)


def embed_grad(ids, dy, V, scale, padding, dtype):
    """(dweight, bound) from dy float64 [n, D]."""
    kept = (ids >= 0) & (ids < V) & (ids != padding)
    ids, dy = ids[kept], dy[kept]
    shape = (V, dy.shape[-1])
    total = torch.zeros(shape, dtype=dy.dtype).index_add_(0, ids, dy)
    size = torch.zeros(shape, dtype=dy.dtype).index_add_(0, ids, dy.abs())
    count = torch.bincount(ids, minlength=V).double()[:, None]
    ref = total * scale
    return ref, rounded(ref, (count + 2) * 2.0**-24 * size * abs(scale), dtype)


def residual(x, y, weight, post, gate, scale, eps, d_s=None, d_h=None):
    """dict of (value, fp32 bound before rounding) of float64 inputs [rows, D]:
    s, h, and with cotangents x, y, gate, weight, post (their gradients)."""
    D = x.shape[-1]
    chain = (D / 64 + 12) * 2.0**-24
    r1 = (y.square().mean(-1, keepdim=True) + eps).rsqrt() if post is not None else 1.0
    n = y * r1
    u = n if post is None else n * post
    sig = 1.0 if gate is None else torch.sigmoid(gate)
    b = u * sig
    s = x + scale * b
    r2 = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    m = s * r2
    e_b = chain + 2.0**-20
    e_s = 2.0**-23 * s.abs() + e_b * (scale * b).abs()          # absolute
    s_err = (s * e_s).abs().mean(-1, keepdim=True) * r2 * r2    # relative error of r2 from that of s
    e_r2 = chain + 2.0**-22 + s_err
    e_m = e_s * r2 + m.abs() * e_r2
    out = {"s": (s, e_s), "h": (m * weight, (e_m + 2.0**-23 * m.abs()) * weight.abs())}
    if d_s is None:
        return out
    e = d_h * weight
    a = (e * m).mean(-1, keepdim=True)
    e_a = (e.abs() * e_m).mean(-1, keepdim=True) + (chain + 2.0**-22) * (e * m).abs().mean(-1, keepdim=True)
    dx = d_s + r2 * (e - m * a)
    size = d_s.abs() + r2 * (e.abs() + m.abs() * a.abs())
    e_dx = 2.0**-21 * size + e_r2 * r2 * (e.abs() + m.abs() * a.abs()) + r2 * (e_m * a.abs() + m.abs() * e_a)
    out["x"] = dx, e_dx
    db = scale * dx
    e_db = abs(scale) * e_dx + 2.0**-23 * db.abs()
    if gate is not None:
        f = u * sig * (1 - sig)
        out["gate"] = db * f, e_db * f.abs() + db.abs() * (f.abs() * (e_b + 2.0**-21) + u.abs() * sig * 2.0**-21)
    du = db * sig
    e_du = e_db * sig + du.abs() * 2.0**-21
    rows = x.shape[0]
    tall = (rows / 4 + 600) * 2.0**-24  # a workgroup's rows, its waves, the workgroups

    def columns(f, g, e_f, e_g):
        return (f * g).sum(0), (tall * (f * g).abs() + e_f * g.abs() + f.abs() * e_g).sum(0)

    out["weight"] = columns(d_h, m, 0 * m, e_m)
    if post is None:
        out["y"] = du, e_du
        return out
    e_n = (chain + 2.0**-22) * n.abs()
    out["post"] = columns(du, n, e_du, e_n)
    q = du * post
    e_q = e_du * post.abs() + 2.0**-23 * q.abs()
    c = (q * n).mean(-1, keepdim=True)
    # the kernel forms c from sums over d_s + r2 e and m, each larger than what they leave
    w = (scale * sig * post * n).abs()
    e_c = ((chain + 2.0**-20) * (w * (size + r2 * a.abs() * m.abs()))).mean(-1, keepdim=True)
    e_c = e_c + (w * e_dx).mean(-1, keepdim=True) + (e_q * n.abs() + q.abs() * e_n).mean(-1, keepdim=True)
    out["y"] = r1 * (q - n * c), r1 * (e_q + n.abs() * e_c + e_n * c.abs() + (chain + 2.0**-21) * (q.abs() + (n * c).abs()))
    return out
