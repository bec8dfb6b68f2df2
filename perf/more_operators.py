"""What becomes of a causal language model's logits, case by case, for timing.

``ops.adjust_logits`` (penalties for repeated tokens, biases and grammar masks,
and its gradient), ``ops.sample_tokens`` (the choice of a token by temperature,
top-k, top-p and min-p) and ``ops.distill_loss`` (the divergence from a
teacher's most probable tokens, and its gradient). Vocabulary sizes are those of
the shipped configurations (32000 and 256 tokens), batches those of the
benchmark and of the tests, with odd and ragged sizes beside them.

``run`` computes the plain form in torch operations (fp32; float64 for the
sums that decide which token is taken), or calls the framework's operators where
``own`` is set; ``exact`` restates the definitions in float64.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "cyfa-jittor_amd")
DEV = "cuda"
PAD = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = 16384 * 32000 * 2  # bytes of the largest listed logits


def listed():
    return [
        # The next token of one conversation, with penalties for what it has said: the smallest call, all latency.
        _adjust("adjust_token", B=1, vocab=32000, L=512),
        # A decode batch of 64 sequences: penalties of each, a grammar's bit mask for some, 16 biased tokens.
        _adjust("adjust_batch", B=64, vocab=32000, L=2048, bias="tokens", mask="bits"),
        # 256 long sequences, one bias over an odd vocabulary, masks as truth values.
        _adjust("adjust_long", B=256, vocab=50001, L=8191, dtype="fp16", bias="dense", mask="bool"),
        # A policy-gradient step: the logits of 4 x 1024 sampled tokens adjusted as they were when sampled.
        _adjust("adjust_train", B=4, T=1024, vocab=32000, L=1280, train=True),
        # One sampled token, temperature and nucleus.
        _sample("sample_token", rows=1, vocab=32000, p=0.95),
        # A decode batch of 64 sequences, each with settings of its own.
        _sample("sample_batch", rows=64, vocab=32000, k=50, p=0.9, least=0.02, mixed=True),
        # A rollout's tokens drawn from whole fp32 distributions, odd vocabulary and row count.
        _sample("sample_rollout", rows=1021, vocab=50001, dtype="fp32"),
        # Few rows of a large vocabulary, nucleus alone.
        _sample("sample_wide", rows=16, vocab=131072, p=0.9),
        # A step of batched generation: adjust, then sample.
        _adjust("step_batch", kind="step", B=64, vocab=32000, L=1024, mask="bits", k=50, p=0.9),
        # The tests' small model in fp32, a ragged batch against a teacher's eight tokens.
        _distill("distill_tiny", B=3, T=37, vocab=256, k=8, dtype="fp32"),
        # A student's training step at the benchmark's batch, twenty tokens of a softened teacher.
        _distill("distill_batch", B=8, T=2048, vocab=32000, k=20, temperature=2.0),
        # 64 tokens and the rest of the teacher's mass, weighted rows, odd vocabulary and row count.
        _distill("distill_tail", B=1, T=1021, vocab=50001, k=64, tail=True, weights=True, dtype="fp16"),
    ]


def _adjust(name, B, vocab, L, T=1, dtype="bf16", bias="", mask="", train=False, kind="adjust", k=0, p=1.0):
    c = dict(name=name, kind=kind, B=B, T=T, vocab=vocab, L=L, dtype=dtype, bias=bias, mask=mask, train=train)
    return c if kind == "adjust" else dict(c, k=k, p=p)


def _sample(name, rows, vocab, k=0, p=1.0, least=0.0, mixed=False, dtype="bf16"):
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, k=k, p=p, least=least, mixed=mixed, dtype=dtype)


def _distill(name, B, T, vocab, k, temperature=1.0, tail=False, weights=False, dtype="bf16"):
    return dict(name=name, kind="distill", B=B, T=T, vocab=vocab, k=k, temperature=temperature, tail=tail,
                weights=weights, dtype=dtype)


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["adjust", "adjust", "sample", "sample", "step", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    vocab = rng.choice([256, 32000, _log_int(rng, 256, 131072), _log_int(rng, 256, 131072)])
    most = LARGEST // (8 * vocab * size)
    if kind == "adjust" and rng.random() < 0.4:
        B, T = rng.randint(1, 4), _log_int(rng, 1, min(512, most))
        c = _adjust("", B, vocab, T + _log_int(rng, 1, 512), T, dtype, rng.choice(["", "dense", "tokens"]),
                    rng.choice(["", "bool", "bits"]), rng.random() < 0.7)
    elif kind in ("adjust", "step"):
        L = rng.choice([0, _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)])
        c = _adjust("", _log_int(rng, 1, min(256, most)), vocab, L, 1, dtype, rng.choice(["", "dense", "tokens"]),
                    rng.choice(["", "bool", "bits"]), kind=kind, k=rng.choice([0, 1, 50]), p=rng.choice([1.0, 0.9]))
    elif kind == "sample":
        c = _sample("", _log_int(rng, 1, min(1024, most)), vocab, rng.choice([0, 0, 1, 50, 1000]), rng.choice([1.0, 0.95, 0.5]),
                    rng.choice([0.0, 0.0, 0.05]), rng.random() < 0.5, dtype)
    else:
        rows = _log_int(rng, 2, min(8192, 4 * most))
        B = _log_int(rng, 1, min(8, rows // 2))
        tail = rng.random() < 0.4
        c = _distill("", B, rows // B, vocab, rng.choice([1, 8, 20, _log_int(rng, 1, 128)]), 1.0 if tail else rng.choice([1.0, 2.0]),
                     tail, rng.random() < 0.3, dtype)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _rand(gen, *shape):
    return torch.rand(*shape, device=DEV, generator=gen)


def _rand_ids(gen, n, vocab):
    """Token ids with frequencies falling as 1 / (id + 1), as words have them."""
    u = torch.rand(n, device=DEV, generator=gen, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)


def _logits(gen, rows, vocab, dtype, tokens):
    """Logits as a trained model gives them: a broad spread with one token well ahead in half of the rows."""
    x = torch.empty(rows, vocab, device=DEV, dtype=dtype)
    for i in range(0, rows, 2048):
        part = _randn(gen, min(2048, rows - i), vocab) * 2.5
        ahead = 8 * _rand(gen, part.shape[0])
        part.scatter_add_(1, tokens[i:i + 2048, None], (ahead * (ahead > 4))[:, None])
        x[i:i + 2048] = part.to(dtype)
    return x


def prepare(case, seed):
    gen = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case=case)
    vocab = case["vocab"]
    if case["kind"] in ("adjust", "step"):
        B, T, L = case["B"], case["T"], case["L"]
        lead = (B,) if T == 1 else (B, T)
        rows = B * T
        state["logits"] = _logits(gen, rows, vocab, dtype, _rand_ids(gen, rows, vocab)).view(*lead, vocab)
        history = _rand_ids(gen, B * L, vocab).view(B, L)
        if T == 1:  # sequences of ragged lengths, padded
            lengths = torch.randint((L + 1) // 2, L + 1, (B,), device=DEV, generator=gen)
            prompts = (_rand(gen, B) * (lengths + 1)).long()
            history.masked_fill_(torch.arange(L, device=DEV) >= lengths[:, None], PAD)
        else:  # the sequences' own tokens: the position's prefix is its history
            history = history[:, None].expand(B, T, L)
            lengths = (L - T + torch.arange(T, device=DEV)).expand(B, T).contiguous()
            prompts = torch.full((B, T), L - T, device=DEV)
        state.update(history=history, lengths=lengths, prompt_lengths=prompts,
                     repetition=1 + 0.5 * _rand(gen, *lead), presence=_rand(gen, *lead), frequency=0.5 * _rand(gen, *lead))
        if case["bias"] == "dense":
            state["bias"] = _randn(gen, vocab)
        elif case["bias"] == "tokens":
            state["token_bias"] = (_rand_ids(gen, B * 16, vocab).view(*lead[:1], *([1] * (T > 1)), 16), 4 * _randn(gen, *lead[:1], *([1] * (T > 1)), 16))
        if case["mask"]:  # every third sequence: nine tokens of ten are outside the grammar
            allowed = _rand(gen, rows, -(-vocab // 32) * 32) < 0.1
            allowed[:, :16] = True
            allowed[torch.arange(rows, device=DEV) % 3 != 0] = True
            if case["mask"] == "bits":
                words = (allowed.view(rows, -1, 32).long() << torch.arange(32, device=DEV)).sum(-1)
                state["allowed"] = (words - ((words >> 31) << 32)).int().view(*lead, -1)
            else:
                state["allowed"] = allowed[:, :vocab].contiguous().view(*lead, vocab)
        if case["train"]:
            state["d_out"] = _logits(gen, rows, vocab, dtype, _rand_ids(gen, rows, vocab)).view(*lead, vocab)
            state["logits"].requires_grad_(True)
        if case["kind"] == "step":
            state["uniform"] = _rand(gen, rows)
            state["temperature"] = 0.5 + _rand(gen, rows)
    elif case["kind"] == "sample":
        rows, k = case["rows"], case["k"]
        state["logits"] = _logits(gen, rows, vocab, dtype, _rand_ids(gen, rows, vocab))
        state["uniform"] = _rand(gen, rows)
        if case["mixed"]:  # a row's own temperature, top-k, top-p and least share of the first token's weight
            state["options"] = dict(temperature=0.3 + 1.2 * _rand(gen, rows), top_p=1 - (1 - case["p"]) * _rand(gen, rows),
                                    top_k=(k * (0.5 + _rand(gen, rows))).long(), min_p=case["least"] * _rand(gen, rows))
        else:
            state["options"] = dict(temperature=0.8, top_k=k, top_p=case["p"], min_p=case["least"])
    else:
        B, T, k = case["B"], case["T"], case["k"]
        rows = B * T
        x = _logits(gen, rows, vocab, dtype, _rand_ids(gen, rows, vocab))
        ids = torch.empty(rows, k, device=DEV, dtype=torch.int64)
        values = torch.empty(rows, k, device=DEV)
        for i in range(0, rows, 2048):  # a teacher that differs from the student a little
            t = x[i:i + 2048].float()
            t = t + _randn(gen, *t.shape)
            top = t.topk(k, -1)
            ids[i:i + 2048] = top.indices
            values[i:i + 2048] = top.values - torch.logsumexp(t, -1, keepdim=True)
        ends = torch.randint((T + 1) // 2, T + 1, (B, 1), device=DEV, generator=gen)
        ids.view(B, T, k).masked_fill_((torch.arange(T, device=DEV) >= ends)[..., None], PAD)
        state.update(logits=x.view(B, T, vocab).requires_grad_(True), ids=ids.view(B, T, k), values=values.view(B, T, k),
                     weights=_rand(gen, B, T) if case["weights"] else None,
                     # (half precision trains with a scaled loss)
                     d_loss=torch.tensor(2.0**15 if case["dtype"] == "fp16" else 1.0, device=DEV))
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


def _own_adjusted(st):
    return _ops().adjust_logits(st["logits"], st["history"], st["lengths"], st["prompt_lengths"], repetition=st["repetition"],
                                presence=st["presence"], frequency=st["frequency"], bias=st.get("bias"),
                                token_bias=st.get("token_bias"), allowed=st.get("allowed"))


def _own_adjust(case, st):
    if not case["train"]:
        with torch.no_grad():
            return [_own_adjusted(st)]
    y = _own_adjusted(st)
    return [y.detach(), *torch.autograd.grad(y, [st["logits"]], st["d_out"])]


def _own_step(case, st):
    with torch.no_grad():
        y = _own_adjusted(st)
        r = _ops().sample_tokens(y, st["uniform"], temperature=st["temperature"], top_k=case["k"], top_p=case["p"])
    return [y, r.ids, r.logprob]


def _own_sample(case, st):
    with torch.no_grad():
        r = _ops().sample_tokens(st["logits"], st["uniform"], **st["options"])
    return [r.ids, r.logprob]


def _own_distill(case, st):
    loss = _ops().distill_loss(st["logits"], st["ids"], st["values"], temperature=case["temperature"], tail=case["tail"],
                               weights=st["weights"])
    return [loss.detach(), *torch.autograd.grad(loss, [st["logits"]], st["d_loss"])]


_OWN = dict(adjust=_own_adjust, step=_own_step, sample=_own_sample, distill=_own_distill)


def _adjusted(case, st):
    """The adjusted logits in fp32, and their derivative by the logits."""
    x = st["logits"].float()
    V, L = case["vocab"], case["L"]
    lead = x.shape[:-1]
    history, at = st["history"], torch.arange(L, device=DEV)
    inside = (at < st["lengths"][..., None]) & (history >= 0) & (history < V)
    ids = history.clamp(0, V - 1)
    zero = torch.zeros(*lead, V, device=DEV, dtype=torch.int32)
    n = zero.scatter_add(-1, ids, inside.int())
    m = zero.scatter_add(-1, ids, (inside & (at >= st["prompt_lengths"][..., None])).int())
    r = st["repetition"][..., None]
    slope = torch.where(n > 0, torch.where(x > 0, 1 / r, r), torch.ones_like(x))
    y = torch.where(n > 0, torch.where(x > 0, x / r, x * r), x)
    y = y - (m * st["frequency"][..., None] + (m > 0) * st["presence"][..., None])
    if case["bias"] == "dense":
        y = y + st["bias"]
    elif case["bias"] == "tokens":
        to, values = (t.expand(*lead, 16) for t in st["token_bias"])
        y = y + torch.zeros_like(y).scatter_add_(-1, to, values)
    if case["mask"]:
        allowed = st["allowed"]
        if case["mask"] == "bits":
            allowed = ((allowed[..., None] >> torch.arange(32, device=DEV)) & 1).flatten(-2)[..., :V] > 0
        y = torch.where(allowed, y, -math.inf)
        slope = slope * allowed
    return y, slope


def _plain_adjust(case, st):
    y, slope = _adjusted(case, st)
    dtype = st["logits"].dtype
    return [y.to(dtype), (st["d_out"].float() * slope).to(dtype)] if case["train"] else [y.to(dtype)]


def _chosen(x, u, temperature, top_k, top_p, min_p):
    """Ids and log probabilities of the drawn tokens; the options are numbers or [rows, 1]."""
    V = x.shape[-1]
    x = x.double()
    w = torch.exp((x - x.amax(-1, keepdim=True)) / temperature)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(-1, order)
    rank = torch.arange(V, device=DEV)
    first = sorted_w * ((rank < top_k) | (top_k <= 0))
    mass = first.cumsum(-1)
    keep = (first > 0) & ((mass - first < top_p * mass[:, -1:]) | (top_p >= 1)) & (sorted_w >= min_p)
    kept = w * torch.zeros_like(w).scatter_(-1, order, keep.double())
    mass = kept.cumsum(-1)
    ids = (mass <= u.double()[:, None] * mass[:, -1:]).sum(-1)
    return [ids, (kept.gather(-1, ids[:, None])[:, 0] / mass[:, -1]).log().float()]


def _options(st):
    return [v[:, None].double() if isinstance(v, torch.Tensor) else torch.tensor(v, device=DEV, dtype=torch.float64)
            for v in (st["options"][n] for n in ("temperature", "top_k", "top_p", "min_p"))]


def _plain_sample(case, st):
    return _chosen(st["logits"], st["uniform"], *_options(st))


def _plain_step(case, st):
    y = _adjusted(case, st)[0].to(st["logits"].dtype)
    k, p = (torch.tensor(case[n], device=DEV, dtype=torch.float64) for n in ("k", "p"))
    return [y, *_chosen(y, st["uniform"], st["temperature"][:, None].double(), k, p, 0.0)]


def _plain_distill(case, st):
    V, k, temperature = case["vocab"], case["k"], case["temperature"]
    logits = st["logits"].view(-1, V)
    x = logits.float() / temperature
    ids, values = st["ids"].view(-1, k), st["values"].view(-1, k)
    valid = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1)
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    lse = e.sum(-1, keepdim=True).log()
    if case["tail"]:
        p = torch.where(valid, values.double().exp(), 0.0)
        others = e.scatter(-1, torch.where(valid, at, at[:, :1]), 0.0)  # (a row without valid ids does not count)
        log_q_rest = others.sum(-1, keepdim=True).log() - lse
        rest = (1 - p.sum(-1, keepdim=True)).clamp(min=0).float()
        p = p.float()
    else:
        t = torch.where(valid, values / temperature, -math.inf)
        p = torch.where(valid, (t - t.amax(-1, keepdim=True)).exp(), 0.0)
        p = torch.where(valid, p / p.sum(-1, keepdim=True), 0.0)
        rest = torch.zeros_like(lse)
        log_q_rest = torch.zeros_like(lse)
    row = torch.where(p > 0, p * (p.log() - (x.gather(-1, at) - lse)), 0.0).sum(-1)
    row = row + torch.where(rest > 0, rest * (rest.log() - log_q_rest), 0.0)[:, 0]
    counts = valid.any(-1).float()
    if st["weights"] is not None:
        counts = counts * st["weights"].view(-1)
    total = counts.double().sum()
    loss = ((row.double() * counts).sum() / total).float()
    q = (x - lse).exp()
    g = (st["d_loss"] * counts / total.float() / temperature)[:, None]
    dx = q * (p.sum(-1, keepdim=True) + rest)
    if case["tail"]:
        dx = dx - others * (rest / others.sum(-1, keepdim=True))
    dx = torch.where(counts[:, None] > 0, dx.scatter_add_(-1, at, -p) * g, 0.0)
    return [loss, dx.to(logits.dtype).view(st["logits"].shape)]


_PLAIN = dict(adjust=_plain_adjust, step=_plain_step, sample=_plain_sample, distill=_plain_distill)


# ---------------------------------------------------------------- work and float64 results


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    V = case["vocab"]
    if case["kind"] in ("adjust", "step"):
        B, T, L = case["B"], case["T"], case["L"]
        n = B * T * V
        total = n * size * (4 if case["train"] else 2) + B * T * 28
        total += int(B * L * 8 * (0.75 if T == 1 else 1))
        total += {"": 0, "dense": 4 * V, "tokens": 192 * B}[case["bias"]] + {"": 0, "bool": n, "bits": n // 8}[case["mask"]]
        flops = n * (2 if case["train"] else 1) + B * T * L
        if case["kind"] == "step":
            return dict(bytes=total + 20 * B, flops=flops + 20 * n)
        return dict(bytes=total, flops=flops)
    if case["kind"] == "sample":
        rows = case["rows"]
        return dict(bytes=rows * (V * size + 16 + 20 * case["mixed"]), flops=20 * rows * V)
    rows = case["B"] * case["T"]
    n = rows * V
    return dict(bytes=2 * n * size + rows * (12 * case["k"] + 4 * case["weights"]) + 4, flops=7 * n)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["kind"]](case, state)


def _exact_adjust(case, st):
    V, L = case["vocab"], case["L"]
    x = st["logits"].reshape(-1, V).double()
    rows = x.shape[0]
    history = st["history"].reshape(rows, L).cpu().numpy()
    lengths, prompts = (st[n].reshape(-1).cpu().numpy() for n in ("lengths", "prompt_lengths"))
    r, presence, frequency = (st[n].reshape(-1).double().tolist() for n in ("repetition", "presence", "frequency"))
    y, slope = x.clone(), torch.ones_like(x)
    for i in range(rows):
        used = history[i, :lengths[i]]
        seen = torch.from_numpy(np.unique(used[(used >= 0) & (used < V)])).to(DEV)
        slope[i, seen] = torch.where(x[i, seen] > 0, 1 / r[i], r[i]).to(slope)
        y[i] = x[i] * slope[i]
        made = history[i, prompts[i]:lengths[i]]
        made, times = np.unique(made[(made >= 0) & (made < V)], return_counts=True)
        y[i, torch.from_numpy(made).to(DEV)] -= torch.from_numpy(times * frequency[i] + presence[i]).to(DEV)
    if "bias" in st:
        y += st["bias"].double()
    if "token_bias" in st:
        ids, values = (t.expand(*st["logits"].shape[:-1], 16).reshape(rows, 16) for t in st["token_bias"])
        for j in range(16):
            y[torch.arange(rows, device=DEV), ids[:, j]] += values[:, j].double()
    if "allowed" in st:
        allowed = st["allowed"].reshape(rows, -1)
        if case["mask"] == "bits":
            bits = np.unpackbits(np.ascontiguousarray(allowed.cpu().numpy()).view(np.uint8), axis=-1, bitorder="little")
            allowed = torch.from_numpy(bits[:, :V].astype(bool)).to(DEV)
        y[~allowed] = -math.inf
        slope[~allowed] = 0
    shape = st["logits"].shape
    return [y.view(shape), (st["d_out"].double().view(rows, V) * slope).view(shape)] if case["train"] else [y.view(shape)]


def _exact_choice(x, u, temperature, top_k, top_p, min_p):
    """Row by row on the host: x [rows, V], the options lists of numbers."""
    x, u = x.double().cpu().numpy(), u.double().cpu().numpy()
    ids, logprob = [], []
    for i in range(x.shape[0]):
        order = np.lexsort((np.arange(x.shape[1]), -x[i]))
        if top_k[i] > 0:
            order = order[:int(top_k[i])]
        w = np.exp((x[i, order] - x[i, order[0]]) / temperature[i])
        if top_p[i] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)])
            order = order[before[:-1] < top_p[i] * before[-1]]
        order = np.sort(order[w[:len(order)] >= min_p[i]])
        w = np.exp((x[i, order] - x[i].max()) / temperature[i])
        mass = np.cumsum(w)
        j = min(int(np.searchsorted(mass, u[i] * mass[-1], side="right")), len(order) - 1)
        ids.append(int(order[j]))
        logprob.append(math.log(w[j] / mass[-1]))
    return [torch.tensor(ids, device=DEV), torch.tensor(logprob, device=DEV, dtype=torch.float64)]


def _exact_sample(case, st):
    o, rows = st["options"], case["rows"]
    lists = [o[n].tolist() if isinstance(o[n], torch.Tensor) else [o[n]] * rows for n in ("temperature", "top_k", "top_p", "min_p")]
    return _exact_choice(st["logits"], st["uniform"], *lists)


def _exact_step(case, st):
    """Of the token, drawn from the logits as they are rounded, there is no value apart from that rounding."""
    return [_exact_adjust(case, st)[0], None, None]


def _exact_distill(case, st):
    V, k, temperature = case["vocab"], case["k"], case["temperature"]
    logits = st["logits"].view(-1, V)
    ids, values = st["ids"].view(-1, k), st["values"].view(-1, k).double()
    counts = ((ids >= 0) & (ids < V)).any(-1).double()
    if st["weights"] is not None:
        counts = counts * st["weights"].view(-1).double()
    total, loss, parts = counts.sum(), 0.0, []
    step = max(1, (1 << 26) // V)
    for i in range(0, logits.shape[0], step):
        c = counts[i:i + step, None] / total
        valid = (ids[i:i + step] >= 0) & (ids[i:i + step] < V)
        # the teacher's probabilities laid out over the vocabulary
        t = values[i:i + step].masked_fill(~valid, -math.inf)
        p = t.exp() if case["tail"] else torch.softmax(t / temperature, -1)
        p = p.masked_fill(~valid, 0.0)
        logp = torch.log_softmax(logits[i:i + step].double() / temperature, -1)
        given = torch.zeros_like(logp).scatter_add_(1, ids[i:i + step].clamp(0, V - 1), p)
        q = logp.exp()
        loss += float((c * (torch.special.xlogy(p, p).sum(-1, keepdim=True) - (given * logp).sum(-1, keepdim=True))).sum())
        dx = q * p.sum(-1, keepdim=True) - given
        if case["tail"]:
            other = torch.ones_like(q).scatter_(1, torch.where(valid, ids[i:i + step], ids[i:i + step, :1].clamp(min=0)), 0.0)
            q_rest = (q * other).sum(-1, keepdim=True)
            p_rest = (1 - p.sum(-1, keepdim=True)).clamp(min=0)
            loss += float((c * (torch.special.xlogy(p_rest, p_rest) - p_rest * q_rest.log())).sum())
            dx += p_rest * (q - q * other / q_rest)
        parts.append(dx * c * float(st["d_loss"]) / temperature)
    return [torch.tensor(loss, dtype=torch.float64, device=DEV), torch.cat(parts).view(st["logits"].shape)]


_EXACT = dict(adjust=_exact_adjust, step=_exact_step, sample=_exact_sample, distill=_exact_distill)
