"""The operators around a causal language model's blocks, case by case, for timing.

``ops.token_logprobs`` (log probabilities of given tokens with entropy and top
alternatives) and ``ops.token_loss`` (their mean, the training loss),
``ops.embed_tokens`` (the scaled embedding lookup and its gradient), and
``ops.residual_norm`` (a block's output norm and gate, the scaled residual add
and the next block's norm). Vocabulary and hidden sizes are those of the
shipped configurations (32000 and 256 tokens; 256, 1024, 1536 and 2048 wide),
batches those of the benchmark and of the tests, with odd and ragged sizes
beside them.

``run`` computes the plain form in fp32 torch operations, or calls the
framework's operators where ``own`` is set; ``exact`` restates the definitions
in float64.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "cyfa-jittor_amd")
DEV = "cuda"
EPS = 1e-6
IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = 16384 * 32000 * 2  # bytes of the largest listed logits


def listed():
    return [
        # The choice of one decoded token, with five alternatives: the smallest call, all latency.
        _score("score_token", rows=1, vocab=32000, top=5),
        # A decode batch of 64 sequences with twenty alternatives, some rows held to a grammar's tokens.
        _score("score_batch", rows=64, vocab=32000, top=20, masked=True),
        # Scoring a batch of prompts: log probability and entropy of 8 x 2048 tokens.
        _score("score_prompt", rows=16384, vocab=32000),
        # A policy-gradient step: log probabilities and an entropy bonus of sampled tokens, odd vocabulary and row count.
        _score("policy_ragged", rows=1021, vocab=50001, train=True),
        # The loss of a training step at the benchmark's batch, labels ignored past ragged ends.
        _loss("loss_batch", B=8, T=2048, vocab=32000),
        # The tests' small model in fp32, a ragged batch.
        _loss("loss_tiny", B=3, T=37, vocab=256, dtype="fp32"),
        # The next tokens of 64 sequences.
        _embed("embed_token", N=64, vocab=32000, width=1024),
        # A training step's lookup and gradient, 8 x 2048 tokens with natural frequencies.
        _embed("embed_train", N=16384, vocab=32000, width=1024, train=True),
        # fp32 training of the widest configuration, scaled lookup with a padding id, odd token count.
        _embed("embed_wide", N=2999, vocab=32000, width=2048, dtype="fp32", scale=45.25, pad=2, train=True),
        # The join between two blocks for the next tokens of 64 sequences.
        _join("join_token", rows=64, width=1024),
        # A training step's join with an output norm and a gate, 8 x 2048 tokens.
        _join("join_batch", rows=16384, width=1024, post=True, gate=True, train=True),
        # fp32 training of the plain join with a residual scale, 2 x 1500 tokens less one.
        _join("join_fp32", rows=2999, width=1536, dtype="fp32", scale=0.5, train=True),
    ]


def _score(name, rows, vocab, top=0, dtype="bf16", masked=False, train=False):
    return dict(name=name, kind="score", rows=rows, vocab=vocab, top=top, dtype=dtype, masked=masked, train=train)


def _loss(name, B, T, vocab, dtype="bf16"):
    return dict(name=name, kind="loss", B=B, T=T, vocab=vocab, dtype=dtype)


def _embed(name, N, vocab, width, dtype="bf16", scale=1.0, pad=-1, train=False):
    return dict(name=name, kind="embed", N=N, vocab=vocab, width=width, dtype=dtype, scale=scale, pad=pad, train=train)


def _join(name, rows, width, dtype="bf16", scale=1.0, post=False, gate=False, train=False):
    return dict(name=name, kind="join", rows=rows, width=width, dtype=dtype, scale=scale, post=post, gate=gate, train=train)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "score", "loss", "embed", "embed", "join", "join"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    if kind in ("score", "loss"):
        vocab = rng.choice([256, 32000, _log_int(rng, 256, 131072), _log_int(rng, 256, 131072)])
        rows = _log_int(rng, 1, min(16384, LARGEST // (2 * vocab * size)))
        if kind == "score":
            c = _score("", rows, vocab, rng.choice([0, 1, 5, 20]) if rows <= 2048 else 0, dtype,
                       rng.random() < 0.3, rng.random() < 0.4)
        else:
            B = _log_int(rng, 1, min(8, rows))
            c = _loss("", B, max(2, rows // B), vocab, dtype)
    elif kind == "embed":
        c = _embed("", _log_int(rng, 1, 32768), rng.choice([256, 32000, _log_int(rng, 256, 131072)]),
                   rng.choice([256, 1024, 1536, 2048, _log_int(rng, 33, 2048)]), dtype,
                   rng.choice([1.0, 1.0, 32.0]), rng.choice([-1, 2]), rng.random() < 0.6)
    else:
        c = _join("", _log_int(rng, 1, 32768), rng.choice([256, 1024, 1536, 2048, _log_int(rng, 33, 4096)]), dtype,
                  rng.choice([1.0, 1.0, 0.5]), rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.6)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _rand_ids(gen, n, vocab):
    """Token ids with frequencies falling as 1 / (id + 1), as words have them."""
    u = torch.rand(n, device=DEV, generator=gen, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)


def _logits(gen, rows, vocab, dtype, tokens):
    """Logits as a trained model gives them: a broad spread with the given token well ahead in half of the rows."""
    x = torch.empty(rows, vocab, device=DEV, dtype=dtype)
    for i in range(0, rows, 2048):
        part = _randn(gen, min(2048, rows - i), vocab) * 2.5
        ahead = 8 * torch.rand(part.shape[0], device=DEV, generator=gen)
        part.scatter_add_(1, tokens[i:i + 2048, None], (ahead * (ahead > 4))[:, None])
        x[i:i + 2048] = part.to(dtype)
    return x


def prepare(case, seed):
    gen = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["kind"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        tokens = _rand_ids(gen, rows, vocab)
        x = _logits(gen, rows, vocab, dtype, tokens)
        if case["masked"]:  # every third row: nine tokens of ten are outside the grammar
            out = torch.rand(rows, vocab, device=DEV, generator=gen) < 0.9
            out[:, :32] = False
            out.scatter_(1, tokens[:, None], False)
            out[torch.arange(rows, device=DEV) % 3 != 0] = False
            x.masked_fill_(out, -math.inf)
        state.update(logits=x, tokens=tokens)
        if case["train"]:
            state["d_logprob"] = _randn(gen, rows)
            state["d_entropy"] = torch.full((rows,), 0.01, device=DEV)
            if case["top"]:
                state["d_top"] = _randn(gen, rows, case["top"])
            x.requires_grad_(True)
    elif case["kind"] == "loss":
        B, T, vocab = case["B"], case["T"], case["vocab"]
        labels = _rand_ids(gen, B * T, vocab)
        x = _logits(gen, B * T, vocab, dtype, labels).view(B, T, vocab)
        labels = labels.view(B, T)
        lengths = torch.randint(T // 2, T + 1, (B, 1), device=DEV, generator=gen)
        labels = labels.masked_fill(torch.arange(T, device=DEV)[None] >= lengths, IGNORE)
        state.update(logits=x.requires_grad_(True), labels=labels)
    elif case["kind"] == "embed":
        N, vocab, width = case["N"], case["vocab"], case["width"]
        state["ids"] = _rand_ids(gen, N, vocab)
        state["weight"] = (_randn(gen, vocab, width) * 0.02).to(dtype)
        if case["train"]:
            state["weight"].requires_grad_(True)
            state["d_out"] = _randn(gen, N, width).to(dtype)
    else:
        rows, width = case["rows"], case["width"]
        state["x"] = (_randn(gen, rows, width) * 2).to(dtype)
        state["y"] = _randn(gen, rows, width).to(dtype)
        state["gate"] = _randn(gen, rows, width).to(dtype) if case["gate"] else None
        state["weight"] = 1 + 0.1 * _randn(gen, width)
        state["post"] = 1 + 0.1 * _randn(gen, width) if case["post"] else None
        if case["train"]:
            state["d_s"] = _randn(gen, rows, width).to(dtype)
            state["d_h"] = _randn(gen, rows, width).to(dtype)
            for name in ("x", "y", "gate", "weight", "post"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        return _OWN[case["kind"]](case, state)
    with torch.no_grad():
        return _PLAIN[case["kind"]](case, state)


def _ops():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from cyclic_flow_attention import ops

    return ops


def _own_score(case, st):
    if not case["train"]:
        with torch.no_grad():
            r = _ops().token_logprobs(st["logits"], st["tokens"], top_k=case["top"])
        return _score_outputs(case, r)
    r = _ops().token_logprobs(st["logits"], st["tokens"], top_k=case["top"])
    outs, cots = [r.logprob, r.entropy], [st["d_logprob"], st["d_entropy"]]
    if case["top"]:
        outs.append(r.top_logprobs)
        cots.append(st["d_top"])
    (dx,) = torch.autograd.grad(outs, [st["logits"]], cots)
    return [t.detach() for t in _score_outputs(case, r)] + [dx]


def _score_outputs(case, r):
    return [r.logprob, r.entropy, r.top_logprobs, r.top_ids] if case["top"] else [r.logprob, r.entropy]


def _own_loss(case, st):
    loss = _ops().token_loss(st["logits"], st["labels"], ignore_index=IGNORE)
    (dx,) = torch.autograd.grad(loss, [st["logits"]])
    return [loss.detach(), dx]


def _own_embed(case, st):
    pad = None if case["pad"] < 0 else case["pad"]
    if not case["train"]:
        with torch.no_grad():
            return [_ops().embed_tokens(st["ids"], st["weight"], scale=case["scale"], padding_idx=pad)]
    out = _ops().embed_tokens(st["ids"], st["weight"], scale=case["scale"], padding_idx=pad)
    (dw,) = torch.autograd.grad(out, [st["weight"]], st["d_out"])
    return [out.detach(), dw]


def _own_join(case, st):
    def call():
        return _ops().residual_norm(st["x"], st["y"], st["weight"], post_weight=st["post"], gate=st["gate"],
                                    scale=case["scale"], eps=EPS)

    if not case["train"]:
        with torch.no_grad():
            return list(call())
    s, h = call()
    leaves = [st[n] for n in ("x", "y", "gate", "weight", "post") if st[n] is not None]
    return [s.detach(), h.detach(), *torch.autograd.grad([s, h], leaves, [st["d_s"], st["d_h"]])]


_OWN = dict(score=_own_score, loss=_own_loss, embed=_own_embed, join=_own_join)


def _log_softmax(x):
    x = x.float()
    x = x - x.amax(-1, keepdim=True)
    return x - x.exp().sum(-1, keepdim=True).log()


def _plain_score(case, st):
    lp = _log_softmax(st["logits"])
    p = lp.exp()
    plogp = torch.where(p > 0, p * lp, torch.zeros_like(lp))
    logprob = lp.gather(1, st["tokens"][:, None])[:, 0]
    entropy = -plogp.sum(-1)
    outs = [logprob, entropy]
    if case["top"]:
        # keys in the order of (logit, lower index first), all different
        bits = (st["logits"].float() + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        V = case["vocab"]
        keys = bits * (1 << 20) + (V - 1 - torch.arange(V, device=DEV))
        top_ids = V - 1 - (keys.topk(case["top"], -1).values & ((1 << 20) - 1))
        outs += [lp.gather(1, top_ids), top_ids]
    if case["train"]:
        total = st["d_logprob"] + (st["d_top"].sum(-1) if case["top"] else 0)
        dx = -p * total[:, None] - st["d_entropy"][:, None] * (plogp + p * entropy[:, None])
        dx.scatter_add_(1, st["tokens"][:, None], st["d_logprob"][:, None])
        if case["top"]:
            dx.scatter_add_(1, top_ids, st["d_top"])
        outs.append(dx.to(st["logits"].dtype))
    return outs


def _plain_loss(case, st):
    V = case["vocab"]
    lp = _log_softmax(st["logits"]).view(-1, V)
    labels = st["labels"].view(-1)
    kept = labels != IGNORE
    at = labels.clamp(min=0)[:, None]
    count = kept.sum()
    loss = -(lp.gather(1, at)[:, 0] * kept).sum() / count
    g = kept.float() / count
    dx = lp.exp() * g[:, None]
    dx.scatter_add_(1, at, -g[:, None])
    return [loss, dx.to(st["logits"].dtype).view(st["logits"].shape)]


def _plain_embed(case, st):
    w = st["weight"]
    outs = [(w[st["ids"]].float() * case["scale"]).to(w.dtype)]
    if case["train"]:
        d = st["d_out"].float() * case["scale"]
        if case["pad"] >= 0:
            d = d * (st["ids"] != case["pad"])[:, None]
        outs.append(torch.zeros(w.shape, device=DEV).index_add_(0, st["ids"], d).to(w.dtype))
    return outs


def _plain_join(case, st):
    dt, c = st["x"].dtype, case["scale"]
    y = st["y"].float()
    if case["post"]:
        r1 = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        ny = y * r1
        u = ny * st["post"]
    else:
        u = y
    sig = torch.sigmoid(st["gate"].float()) if case["gate"] else None
    s = st["x"].float() + c * (u if sig is None else u * sig)
    r2 = torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS)
    ns = s * r2
    outs = [s.to(dt), (ns * st["weight"]).to(dt)]
    if not case["train"]:
        return outs
    dh = st["d_h"].float()
    dn = dh * st["weight"]
    ds = st["d_s"].float() + r2 * (dn - ns * (dn * ns).mean(-1, keepdim=True))
    db = c * ds
    du = db if sig is None else db * sig
    if case["post"]:
        dny = du * st["post"]
        dy = r1 * (dny - ny * (dny * ny).mean(-1, keepdim=True))
    else:
        dy = du
    outs += [ds.to(dt), dy.to(dt)]
    if sig is not None:
        outs.append((db * u * sig * (1 - sig)).to(dt))
    outs.append((dh * ns).sum(0))
    if case["post"]:
        outs.append((du * ny).sum(0))
    return outs


_PLAIN = dict(score=_plain_score, loss=_plain_loss, embed=_plain_embed, join=_plain_join)


# ---------------------------------------------------------------- work and float64 results


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "score":
        n, rows, k = case["rows"] * case["vocab"], case["rows"], case["top"]
        passes = 2 if case["train"] else 1
        extra = rows * (16 + 12 * k) + (rows * (8 + 4 * k) if case["train"] else 0)
        return dict(bytes=passes * n * size + extra, flops=n * (11 if case["train"] else 5))
    if case["kind"] == "loss":
        n = case["B"] * case["T"] * case["vocab"]
        return dict(bytes=2 * n * size + 8 * case["B"] * case["T"] + 4, flops=7 * n)
    if case["kind"] == "embed":
        N, V, D = case["N"], case["vocab"], case["width"]
        # N draws of ids with weight 1 / (id + 1) meet about this many different rows
        distinct = min(N, V, int(N / math.log(V + 1) * (1 + math.log(max(1.0, V * math.log(V + 1) / N)))) + 1)
        total = (distinct + N) * D * size + 8 * N
        if case["train"]:
            total += (N + V) * D * size
        return dict(bytes=total, flops=N * D * (3 if case["train"] else 1))
    n = case["rows"] * case["width"]
    tensors = 4 + case["gate"]
    flops = 6 + 3 * case["post"] + 4 * case["gate"]
    if case["train"]:
        tensors += 4 + case["gate"]  # d_s, d_h, dx, dy, dgate; x, y and the gate are read once
        flops += 10 + 8 * case["post"] + 6 * case["gate"]
    vectors = (1 + case["post"]) * (2 if case["train"] else 1)
    return dict(bytes=tensors * n * size + vectors * 4 * case["width"], flops=flops * n)


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))


def _exact_score(case, st):
    logits, V, parts = st["logits"].detach(), case["vocab"], []
    step = max(1, (1 << 26) // V)
    for i in range(0, case["rows"], step):
        x = logits[i:i + step].double()
        t = st["tokens"][i:i + step]
        row = torch.arange(x.shape[0], device=DEV)
        lse = torch.logsumexp(x, -1)
        p = torch.softmax(x, -1)
        surprise = torch.where(p > 0, lse[:, None] - x, torch.zeros((), dtype=torch.float64, device=DEV))
        entropy = (p * surprise).sum(-1)
        outs = [x[row, t] - lse, entropy]
        if case["top"]:
            order = torch.sort(x, dim=-1, descending=True, stable=True)
            ids = order.indices[:, :case["top"]]
            outs += [order.values[:, :case["top"]] - lse[:, None], ids]
        if case["train"]:
            onehot = torch.zeros_like(x)
            onehot[row, t] = st["d_logprob"][i:i + step].double()
            if case["top"]:
                d_top = st["d_top"][i:i + step].double()
                for j in range(case["top"]):
                    onehot[row, ids[:, j]] += d_top[:, j]
            dh = st["d_entropy"][i:i + step].double()
            outs.append(onehot - p * onehot.sum(-1, keepdim=True) + p * (surprise - entropy[:, None]) * dh[:, None])
        parts.append(outs)
    return [torch.cat(col) for col in zip(*parts)]


def _exact_loss(case, st):
    logits, V = st["logits"].detach().view(-1, case["vocab"]), case["vocab"]
    labels = st["labels"].view(-1)
    count = int((labels != IGNORE).sum())
    total, parts = 0.0, []
    step = max(1, (1 << 26) // V)
    for i in range(0, logits.shape[0], step):
        x, t = logits[i:i + step].double(), labels[i:i + step]
        p = torch.softmax(x, -1)
        rows = torch.nonzero(t != IGNORE)[:, 0]
        total += float((torch.logsumexp(x, -1)[rows] - x[rows, t[rows]]).sum())
        dx = torch.zeros_like(p)
        dx[rows] = p[rows]
        dx[rows, t[rows]] -= 1
        parts.append(dx / count)
    return [torch.tensor(total / count, dtype=torch.float64, device=DEV), torch.cat(parts).view(st["logits"].shape)]


def _exact_embed(case, st):
    w, ids = st["weight"].detach().double(), st["ids"]
    outs = [w.index_select(0, ids) * case["scale"]]
    if case["train"]:
        keep = torch.nonzero(ids != case["pad"])[:, 0]
        outs.append(torch.zeros_like(w).index_add(0, ids[keep], case["scale"] * st["d_out"][keep].double()))
    return outs


def _exact_join(case, st):
    leaves = {n: st[n].detach().double().requires_grad_(case["train"]) for n in ("x", "y", "gate", "weight", "post")
              if st[n] is not None}
    b = leaves["y"]
    if case["post"]:
        b = b / torch.sqrt(b.square().mean(-1, keepdim=True) + EPS) * leaves["post"]
    if case["gate"]:
        b = b / (1 + torch.exp(-leaves["gate"]))
    s = leaves["x"] + case["scale"] * b
    h = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * leaves["weight"]
    outs = [s.detach(), h.detach()]
    if case["train"]:
        outs += torch.autograd.grad([s, h], list(leaves.values()), [st["d_s"].double(), st["d_h"].double()])
    return outs


_EXACT = dict(score=_exact_score, loss=_exact_loss, embed=_exact_embed, join=_exact_join)
