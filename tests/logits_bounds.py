"""Float64 results of the operators on a model's logits (adjust_logits,
sample_tokens, distill_loss) from their definitions, row by row, each with a
bound on what fp32 computation and one rounding to the result's dtype may be off
by, counted as in lm_bounds: u = half a step; a product, quotient, sum or
conversion 2^-24 of its value, the hardware exponential 2^-23, its argument t a
further |t| 2^-22, a sum of n terms n 2^-24 of the sum of their magnitudes."""

import math

import numpy as np
import torch

import lm_bounds as lm

INF = float("inf")


def adjust(x, history, lengths, prompts, repetition, presence, frequency, bias, tokens, allowed, dtype, dy=None):
    """(y, bound) or with dy ((y, bound), (dx, bound)) of float64 rows x [rows, V];
    history [rows, L] or None, lengths and prompts lists, the penalties lists of
    numbers, bias [rows, V] or None, tokens a list of lists of (id, value), allowed
    bool [rows, V] or None."""
    rows, V = x.shape
    y, slope, size = x.clone(), torch.ones_like(x), x.abs()
    for r in range(rows):
        seen = [] if history is None else [t for t in history[r][:max(0, lengths[r])] if 0 <= t < V]
        made = [] if history is None else [t for t in history[r][:max(0, lengths[r])][max(0, prompts[r]):] if 0 <= t < V]
        for t in set(seen):
            slope[r, t] = 1 / repetition[r] if x[r, t] > 0 else repetition[r]
            y[r, t] = x[r, t] * slope[r, t] if x[r, t] != 0 else x[r, t]
        size[r] = y[r].abs()
        for t in set(made):
            c = made.count(t)
            y[r, t] -= c * frequency[r] + presence[r]
            size[r, t] += abs(c * frequency[r]) + abs(presence[r])
        if bias is not None:
            y[r] += bias[r]
            size[r] += bias[r].abs()
        for t, v in tokens[r] if tokens else ():
            if 0 <= t < V:
                y[r, t] += v
                size[r, t] += abs(v)
    chain = 6 + (max(map(len, tokens)) if tokens else 0)
    bound = lm.rounded(y, chain * 2.0**-24 * torch.nan_to_num(size, posinf=0.0), dtype)
    if allowed is not None:
        y[~allowed] = -INF
        slope[~allowed] = 0
    if dy is None:
        return y, bound
    dx = torch.where(slope == 0, 0.0, dy * slope)
    return (y, bound), (dx, lm.rounded(dx, 2.0**-22 * dx.abs(), dtype))


def choice(x, u, T, k, p, least):
    """(id, log probability) of one float64 row x (numpy) without NaN or +inf and
    with something finite, from the definition."""
    order = np.lexsort((np.arange(len(x)), -x))
    if not T > 0:
        return int(order[0]), 0.0
    w = np.exp((x[order] - x[order[0]]) / T)
    n = k if 0 < k < len(x) else len(x)
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[:n])])
        n = max(1, int((before[:-1] < p * before[-1]).sum()))
    n = max(1, min(n, int((w >= least).sum())))
    ids = np.sort(order[:n])
    w = np.exp((x[ids] - x[order[0]]) / T)
    mass = np.cumsum(w)
    at = int(np.searchsorted(mass, u * mass[-1], side="right"))
    while w[at] == 0:
        at -= 1
    return int(ids[at]), math.log(w[at] / mass[-1])


def distill(x, ids, values, T, tail, weights, dtype, d_loss=1.0):
    """((loss, bound), (dx, bound)) of float64 rows x [rows, V], ids [rows, k],
    float64 values and weights [rows] (or None)."""
    rows, V = x.shape
    chain = (V / 256 + 64) * 2.0**-24
    loss = err = total = 0.0
    dxs, bounds, counts = torch.zeros_like(x), torch.zeros_like(x), []
    for r in range(rows):
        entries = [(int(i), float(v)) for i, v in zip(ids[r], values[r]) if 0 <= i < V and v != -INF]
        w = (1.0 if weights is None else float(weights[r])) if entries else 0.0
        counts.append(w)
        if w == 0:
            continue
        z = x[r] / T
        lq = lm.log_softmax(z[None])[0]
        q = lq.exp()
        entropy = -(q * torch.where(q == 0, 0.0, lq)).sum()
        e_sum = chain + 2.0**-22 + 2.0**-21 * (entropy + 1)
        t = torch.tensor([v for _, v in entries], dtype=torch.float64)
        at = torch.tensor([i for i, _ in entries])
        lp = t if tail else torch.log_softmax(t / T, 0)
        p = lp.exp()
        e_lq = e_sum + 2.0**-21 * lq[at].abs()
        row, e_row = (p * (lp - lq[at])).sum(), (p * (e_lq + 2.0**-22 * (lp.abs() + lq[at].abs()))).sum()
        given = torch.zeros_like(x[r]).index_add_(0, at, p)
        e_given = torch.zeros_like(x[r]).index_add_(0, at, p * (2.0**-21 * ((t / T).abs() + lp.abs()) + 2.0**-21))
        mass = p.sum()
        dx = q * mass - given
        surprise = torch.where(q == 0, 0.0, -lq)
        e_dx = q * mass * (2.0**-20 + 2 * chain + e_sum + 2.0**-21 * surprise) + e_given + 2.0**-22 * (q * mass + given)
        if tail:
            other = torch.ones(V, dtype=torch.bool)
            other[at] = False
            z = z - z.max()  # (a row of the lowest value would lose log V beside it)
            lr = torch.where(other, z, -INF)
            if (lr > -INF).any():
                rest = max(0.0, 1 - mass.item())
                s = torch.softmax(lr, 0)
                lqr = torch.logsumexp(lr, 0) - torch.logsumexp(z, 0)
                e_lqr = e_sum + chain + 2.0**-22 + 2.0**-21 * (torch.special.entr(s).sum() + 1) + 2.0**-22 * (2 * math.log(V) + lqr.abs() + 1)
                if rest > 0:
                    row = row + rest * (math.log(rest) - lqr)
                    e_row = e_row + rest * (e_lqr + 2.0**-22 * abs(math.log(rest)))
                P = mass + rest
                qr = lqr.exp()
                dx = torch.where(other, s * (qr * P - rest), q * P - given)
                own = s * (qr * P * e_lqr + (qr * P - rest).abs() * (2.0**-20 + 2 * chain + 2.0**-21 * torch.where(s == 0, 0.0, -s.clamp(min=1e-300).log())))
                e_dx = torch.where(other, own + 2.0**-22 * s * (qr * P + rest), e_dx + q * rest * (2.0**-20 + 2 * chain + e_sum + 2.0**-21 * surprise))
        loss = loss + w * row
        err = err + abs(w) * (e_row + 2.0**-23 * abs(row))
        dxs[r], bounds[r] = dx / T, e_dx / T
        total += w
    counts = torch.tensor(counts, dtype=torch.float64)[:, None]
    g = torch.where(counts == 0, 0.0, counts * d_loss / (total or float("nan")))  # (rows that do not count get zeros in any case)
    loss = torch.as_tensor(loss / total if total else float("nan"), dtype=torch.float64)
    err = torch.as_tensor(err / abs(total) if total else 0.0, dtype=torch.float64)
    dx = torch.where(g == 0, 0.0, dxs * g)
    return ((loss, err + 2.0**-23 * loss.abs()),
            (dx, lm.rounded(dx, bounds * g.abs() + 2.0**-21 * dx.abs(), dtype)))
