"""The choice of experts, products with 4-bit weights and the adjusting of logits, in 64 bits on the CPU, with bounds on how far
32-bit sums and the outputs' rounding can move each value.

Roundings as in dense_ref: a value rounded to 16 bits is off by at most eps/2 of itself (plus half the smallest subnormal), a step
of an fp32 sum by at most a unit of 2^-23 of what is summed (a matrix instruction may truncate).
"""
import math

import torch

from dense_ref import U32, half_step, tiny

INF = math.inf


def _order(keys):
    """Indices by descending key, equal ones by index, without those of -inf."""
    return sorted((i for i, k in enumerate(keys) if k > -INF), key=lambda i: (-keys[i], i))


def scores(row, score):
    """fp64 scores of one row; experts that are not there (-inf, NaN) have None."""
    x = [float(v) for v in row]
    there = [v > -INF for v in x]
    if score == "sigmoid":
        return [(1 / (1 + math.exp(-v)) if v > -700 else 0.0) if t else None for v, t in zip(x, there)]
    if not any(there):
        return [None] * len(x)
    top = max(v for v, t in zip(x, there) if t)
    e = [(1.0 if v == top else math.exp(v - top) if top < INF else 0.0) if t else None for v, t in zip(x, there)]
    total = math.fsum(v for v in e if v is not None)
    return [None if v is None else v / total for v in e]


def route(logits, topk, bias=None, score="sigmoid", groups=1, top_groups=1, group_best=2, renorm=True, scale=1.0):
    """(sel, w): lists of rows, plain loops over one row at a time."""
    sels, ws = [], []
    for row in logits.double().cpu():
        s = scores(row, score)
        E, size = len(s), len(s) // groups
        key = [-INF if v is None else v + (0.0 if bias is None else float(bias[i])) for i, v in enumerate(s)]
        key = [-INF if k != k else k for k in key]
        worth = []
        for g in range(groups):
            best = sorted((k for k in key[g * size:(g + 1) * size] if k > -INF), reverse=True)[:group_best]
            worth.append(math.fsum(best) if best else -INF)
        kept = set(_order(worth)[:top_groups])
        by = key if bias is not None or top_groups < groups else [float(v) if s[i] is not None else -INF for i, v in enumerate(row)]
        pick = _order([by[i] if i // size in kept or top_groups == groups else -INF for i in range(E)])[:topk]
        total = math.fsum(s[i] for i in pick) if renorm else 1.0
        sels.append(pick + [-1] * (topk - len(pick)))
        ws.append([scale * s[i] / total if total > 0 else 0.0 for i in pick] + [0.0] * (topk - len(pick)))
    return torch.tensor(sels, dtype=torch.int64).view(-1, topk), torch.tensor(ws, dtype=torch.float64).view(-1, topk)


def route_weights(x, sel, score="sigmoid", renorm=True, scale=1.0):
    """The weights of a given choice as a differentiable function of fp64 logits x [M, E]."""
    p = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, 1)
    s = torch.where(sel >= 0, p.gather(1, sel.clamp(min=0)), 0.0)
    return scale * s / s.sum(1, keepdim=True) if renorm else scale * s


def route_gradient(logits, sel, dw, score="sigmoid", renorm=True, scale=1.0):
    """(value, bound): autograd of route_weights in fp64. The device's terms are fp64, rounded to fp32 and added, then rounded to
    the logits' type."""
    dt = logits.dtype
    x = logits.double().cpu().requires_grad_()
    sel, d = sel.cpu(), dw.double().cpu()
    d = torch.where(sel >= 0, d, 0.0)
    w = route_weights(x, sel, score, renorm, scale)
    value, = torch.autograd.grad((w * d).sum(), x)
    with torch.no_grad():
        p = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, 1)
        s = torch.where(sel >= 0, p.gather(1, sel.clamp(min=0)), 0.0)
        total = s.sum(1, keepdim=True) if renorm else torch.ones_like(s[:, :1])
        mag = abs(scale) * (d.abs() + ((d * s).abs().sum(1, keepdim=True) / total if renorm else 0.0)) / total
        terms = torch.zeros_like(p).scatter_add_(1, sel.clamp(min=0), torch.where(sel >= 0, mag, 0.0)) * p
        whole = p * (mag * s).sum(1, keepdim=True)
        if score == "softmax" and not renorm:
            terms = terms + whole
        # the fp64 value itself is off by some 2^-53 of its terms: at experts that are not picked the gradient of a
        # renormalised softmax is 0, and autograd's terms cancel to that
        err = 4 * 2.0 ** -24 * terms + 2.0 ** -48 * whole
    return value, err + half_step(dt) * (value.abs() + err) + tiny(dt)


# ---------------------------------------------------------------------------------------------------------------

PLACE = [0, 2, 4, 6, 1, 3, 5, 7]


def unpack(q, K):
    """Values [N, K] from packed rows, word by word as the header describes them."""
    words = q.cpu().contiguous().view(torch.int32).long() & 0xFFFFFFFF     # [N, blocks * 16]
    out = torch.zeros((q.shape[0], q.shape[1] * 2), dtype=torch.int64)
    for at in range(words.shape[1]):
        block, g, j = at // 16, at % 16 // 4, at % 4
        for p in range(8):
            out[:, block * 128 + 32 * j + 8 * g + PLACE[p]] = words[:, at] >> (4 * p) & 15
    return out[:, :K]


def weight(q, scale, zero, K, group):
    of = torch.arange(K) // group
    s = scale.double().cpu().t()[:, of]
    z = zero.double().cpu().t()[:, of] if zero is not None else 8.0
    return (unpack(q, K).double() - z) * s


def quant(w, group, zeros):
    """(values, scale, zero) by the header's rule: fp32 quotients of the rounded scale."""
    dt, (N, K) = w.dtype, w.shape
    n = (K + group - 1) // group
    full = torch.zeros((N, n * group))
    full[:, :K] = w.float().cpu()
    f = full.view(N, n, group)
    lo, hi = f.amin(2).clamp(max=0), f.amax(2).clamp(min=0)
    s = ((hi - lo) / 15 if zeros else torch.maximum(-lo, hi) / 7).to(dt)
    sf = s.float()[:, :, None]
    some = sf > 0
    z = torch.where(some, torch.round(-lo[:, :, None] / sf).clamp(max=15) if zeros else torch.full_like(sf, 8.0), 8.0)
    v = torch.where(some, (torch.round(f / sf) + z).clamp(0, 15), 8.0)
    return v.view(N, -1)[:, :K].long(), s.t(), z[:, :, 0].t().to(torch.uint8) if zeros else None


def linear(x, q, scale, zero, K, group, out_dt, exact, whole=False):
    """(value, bound) of x w^T. exact: the weights enter as whole numbers, a group as s (sum x (16 + v) - (16 + z) sum x); else they
    are rounded to x's type first. whole: the tokens are whole numbers small enough that a group's sums are exact."""
    xd, w = x.double().cpu(), weight(q, scale, zero, K, group)
    value = xd @ w.t()
    if not exact:
        mag = xd.abs() @ w.abs().t()
        err = (half_step(x.dtype) + (K + 2) * U32 * (1 + half_step(x.dtype))) * mag + tiny(x.dtype) * xd.abs().sum(1)[:, None]
    else:
        n = (K + group - 1) // group
        pad = torch.zeros((xd.shape[0], n * group), dtype=torch.float64)
        pad[:, :K] = xd.abs()
        ax = pad.view(-1, n, group).sum(2)                       # sum |x| of a group
        s = scale.double().cpu().abs()                           # [n, N]
        top = 16.0 + (15.0 if zero is None else float(zero.max()))   # of 16 + v and 16 + z
        size = ax @ s * 2 * max(top, 31.0)
        # a group's two sums, its two multiply-adds, then the sums over groups, at most 16 waves and parts of a call
        err = ((0 if whole else group + 2) + 3 + n + 32) * U32 * size
    return value, err + half_step(out_dt) * (value.abs() + err) + tiny(out_dt)


# ---------------------------------------------------------------------------------------------------------------

def adjust(logits, history=None, lengths=None, prompt=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias=None,
           allowed=None):
    """(value, bound), a row at a time with lists."""
    B, V = logits.shape
    value, mag = logits.double().cpu().clone(), logits.double().cpu().abs()
    of = lambda t, b, off: off if t is None else float(t[b])
    for b in range(B):
        h = [] if history is None else history[b].tolist()
        n = len(h) if lengths is None else min(max(int(lengths[b]), 0), len(h))
        p = 0 if prompt is None else min(max(int(prompt[b]), 0), n)
        r, f, q = of(repetition, b, 1.0), of(frequency, b, 0.0), of(presence, b, 0.0)
        count = {}
        for i in h[p:n]:
            count[i] = count.get(i, 0) + 1
        for i in set(h[:n]):
            if not 0 <= i < V:
                continue
            y = float(value[b, i])
            if r > 0:
                y = y / r if y > 0 else y * r
            c = count.get(i, 0)
            mag[b, i] = mag[b, i] + abs(y) + 2 * abs(f) * c + 2 * (abs(q) if c else 0.0)
            value[b, i] = y - f * c - (q if c else 0.0)
        last = {}
        if bias_ids is not None:
            for i, v in zip(bias_ids[b].tolist(), bias[b].tolist()):
                last[i] = v
        for i, v in last.items():
            if 0 <= i < V:
                mag[b, i] += 2 * abs(v)
                value[b, i] += v
        if allowed is not None:
            bits = (allowed[b].cpu().long()[:, None] >> torch.arange(32) & 1).view(-1)[:V]
            value[b][bits == 0] = -INF
    dt = logits.dtype
    err = torch.where(torch.isfinite(value), 4 * 2.0 ** -24 * mag, 0.0)
    return value, torch.where(torch.isfinite(value), err + half_step(dt) * (value.abs() + err) + tiny(dt), 0.0)


def same(got, want, bound, name=""):
    """Within the bound where the value is finite; infinities and NaN as they are."""
    got = got.double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    bad = torch.where(fine, ~((got - want).abs() <= bound), ~((got == want) | (got.isnan() & want.isnan())))
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside, first at {at}: {float(got[at])} for "
                             f"{float(want[at])} +- {float(bound[at])}")
