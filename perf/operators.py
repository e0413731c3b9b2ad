"""The dense side of a served MoE model's step, as cases that can be timed and compared: the gated feed-forward block of
its dense layers and unquantised shared experts (serving, and training with its gradients), the product in 8-bit integers
of its other projections and its head, and the sampling of tokens from the head's logits.

Kinds of case:
  ffn     y = (min(silu(x Wg^T), L) * clamp(u, -L, L)) Wd^T with u = x Wu^T; L = act_limit, 0 = off
  train   the same forward, then the gradients of x and of the three weights for a given dy
  linear  x quantised per token, times an int8 weight with a scale per channel
  gemm    the product alone, of two int8 matrices with scales for each token and channel
  sample  temperature, top-k, top-p and min-p for each row, then the draw for a given uniform number

With `own` false a pass is the plain form, elementary torch operations in 32 bits (64 where 32 lose what matters); with
`own` true it makes the calls of glm-flash-lite_amd/_native.py. Weights are in hand before a pass, as nn.Linear keeps them.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "glm-flash-lite_amd")
DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _native():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import _native as n
    return n


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------

def _ffn(name, kind, M, H, I, **kw):
    return dict(dict(name=name, kind=kind, M=M, H=H, I=I, type="bf16", act_limit=0.0, strided=False), **kw)


def _int8(name, kind, M, K, N, **kw):
    return dict(dict(name=name, kind=kind, M=M, K=K, N=N, type="bf16", out="bf16"), **kw)


def _sample(name, B, V, **kw):
    return dict(dict(name=name, kind="sample", B=B, V=V, type="f32", mode="mixed", masked=0.0, pad=0), **kw)


def listed():
    return [
        # the shared expert of a decode step of one token, unquantised, at the benchmark's layer shape
        _ffn("ffn-1", "ffn", 1, 5120, 1536, type="f16"),
        # speculative decode of six tokens through a shared expert at the served model's shape, with the SwiGLU clamp
        _ffn("ffn-6", "ffn", 6, 4096, 2048, act_limit=10.0),
        # batched decode of an odd batch through a dense layer, the tokens a slice of a wider buffer
        _ffn("ffn-101", "ffn", 101, 5120, 12288, strided=True),
        # a prompt chunk through a dense layer
        _ffn("ffn-4096", "ffn", 4096, 5120, 12288),
        # a short ragged batch of a fine-tuning step on a small dense layer, fp16
        _ffn("train-333", "train", 333, 2048, 5500, type="f16"),
        # a training step of 8,192 tokens through a dense layer
        _ffn("train-8192", "train", 8192, 4096, 11008),
        # a projection of one token, decode
        _int8("linear-1", "linear", 1, 5120, 5120, type="f16", out="f16"),
        # the head for nine users: logits in fp32
        _int8("head-9", "linear", 9, 4096, 65536, out="f32"),
        # a prompt chunk through a projection whose input another layer quantised
        _int8("gemm-4001", "gemm", 4001, 5120, 12288),
        # one user's token from 131,072 logits, nucleus sampling
        _sample("sample-1", 1, 131072, mode="top_p"),
        # a small server's batch over an odd vocabulary, bf16 logits, each user's own settings, a grammar's mask
        _sample("sample-24", 24, 100003, type="bf16", masked=0.5, pad=5),
        # the largest batch
        _sample("sample-256", 256, 131072, masked=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A matrix size: a multiple of 64 most of the time, else of 8, now and then any number."""
    n, r = _log_int(rng, lo, hi), rng.random()
    return n if r < 0.1 else max(8, n // 8 * 8) if r < 0.35 else max(64, n // 64 * 64)


def draw(rng):
    kind = rng.choice(["ffn", "ffn", "train", "linear", "gemm", "sample", "sample"])
    if kind in ("ffn", "train"):
        band = rng.choice(["decode", "batch", "prompt"])
        M = {"decode": rng.randint(1, 16), "batch": _log_int(rng, 17, 512), "prompt": _log_int(rng, 513, 8192)}[band]
        return dict(kind=kind, M=M, H=_size(rng, 256, 4096), I=_size(rng, 256, 11008), type=rng.choice(["f16", "bf16"]),
                    act_limit=rng.choice([0.0, 0.0, 10.0]), strided=rng.random() < 0.3)
    if kind in ("linear", "gemm"):
        M = rng.choice([rng.randint(1, 16), _log_int(rng, 17, 512), _log_int(rng, 513, 8192)])
        N = _size(rng, 4096, 65536) if M <= 64 and rng.random() < 0.4 else _size(rng, 64, 12288)
        return dict(kind=kind, M=M, K=_size(rng, 128, 8192), N=N, type=rng.choice(["f16", "bf16"]),
                    out=rng.choice(["f16", "bf16", "f32"]))
    return dict(kind="sample", B=_log_int(rng, 1, 256), V=_log_int(rng, 1000, 131072),
                type=rng.choice(["f32", "f32", "bf16", "f16"]),
                mode=rng.choice(["mixed", "mixed", "top_p", "top_k", "min_p", "plain", "greedy"]),
                masked=rng.choice([0.0, 0.1, 0.5, 0.999]), pad=rng.choice([0, 0, 5, 64]))


# ---------------------------------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 29)
    return g


def _randn(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV).mul_(scale)


def _tokens(g, M, K, dt, strided=False, scale=1.0):
    """Activations: normal, one channel in 128 eight times as large, as the residual stream of a trained model has."""
    x = _randn(g, (M, K), scale)
    x[:, torch.randint(0, K, (max(1, K // 128),), generator=g, device=DEV)] *= 8.0
    if not strided:
        return x.to(dt)
    wide = torch.zeros((M, K + 64), dtype=dt, device=DEV)
    wide[:, 32:32 + K] = x.to(dt)
    return wide[:, 32:32 + K]


def prepare(case, seed):
    if own:
        _native().load()
    c, g = case, _gen(seed)
    if c["kind"] in ("ffn", "train"):
        M, H, I, dt = c["M"], c["H"], c["I"], TYPES[c["type"]]
        wide = 3.0 if c["act_limit"] else 1.0       # some gates and ups reach the clamp
        s = dict(case=c, x=_tokens(g, M, H, dt, c["strided"]),
                 wg=_randn(g, (I, H), 0.8 * wide / math.sqrt(H)).to(dt),
                 wu=_randn(g, (I, H), 0.8 * wide / math.sqrt(H)).to(dt),
                 wd=_randn(g, (H, I), 1.0 / math.sqrt(I)).to(dt))
        if c["kind"] == "train":
            s["dy"] = _randn(g, (M, H)).to(dt)
        return s
    if c["kind"] in ("linear", "gemm"):
        M, K, N = c["M"], c["K"], c["N"]
        s = dict(case=c, w=torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8),
                 sw=(torch.rand((N,), generator=g, device=DEV) + 0.5) / (127 * math.sqrt(K)))
        if c["kind"] == "linear":
            s["x"] = _tokens(g, M, K, TYPES[c["type"]])
        else:
            s["a"] = _randn(g, (M, K), 30.0).round_().clamp_(-127, 127).to(torch.int8)
            s["sa"] = (torch.rand((M,), generator=g, device=DEV) + 0.5) / 30.0
        return s
    B, V = c["B"], c["V"]
    x = _randn(g, (B, V), 2.5)
    peak = torch.randint(0, V, (B, 12), generator=g, device=DEV)       # the tokens the context makes likely
    x.scatter_add_(1, peak, 8.0 + 4.0 * torch.rand((B, 12), generator=g, device=DEV))
    if c["masked"]:
        x[torch.rand((B, V), generator=g, device=DEV) < c["masked"]] = float("-inf")
    logits = torch.zeros((B, V + c["pad"]), dtype=TYPES[c["type"]], device=DEV)[:, :V]
    logits.copy_(x)
    rnd = lambda: torch.rand((B,), generator=g, device=DEV)
    on = {"mixed": ("t", "k", "p", "m"), "top_p": ("t", "p"), "top_k": ("t", "k"), "min_p": ("t", "m"), "plain": ("t",),
          "greedy": ()}[c["mode"]]
    s = dict(case=c, logits=logits, u=rnd(), t=0.5 + rnd() if "t" in on else torch.zeros(B, device=DEV),
             k=torch.exp(rnd() * math.log(400.0)).int() if "k" in on else None,
             p=0.7 + 0.3 * rnd() if "p" in on else None, m=0.15 * rnd() if "m" in on else None)
    if c["mode"] == "mixed":                        # each user's own settings: some leave a filter off, some are greedy
        s["k"][rnd() < 0.3] = 0
        s["p"][rnd() < 0.3] = 1.0
        s["m"][rnd() < 0.3] = 0.0
        s["t"][rnd() < 0.1] = 0.0
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------

def _act(g, u, limit):
    """(silu(g) and u, both clamped; the sigmoid)"""
    sg = 1.0 / (1.0 + torch.exp(-g))
    a = g * sg
    if limit:
        return a.clamp(max=limit), u.clamp(-limit, limit), sg, a
    return a, u, sg, a


def _plain_ffn(s):
    c = s["case"]
    dt, L = TYPES[c["type"]], c["act_limit"]
    x, wg, wu, wd = (s[n].float() for n in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    a, b, sg, raw = _act(g, u, L)
    h = a * b
    y = (h @ wd.t()).to(dt)
    if c["kind"] == "ffn":
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    da, db = dh * b, dh * a
    if L:
        da = da * (raw <= L)
        db = db * (u.abs() <= L)
    dg = da * (sg * (1.0 + g * (1.0 - sg)))
    return y, (dg @ wg + db @ wu).to(dt), (dg.t() @ x).to(dt), (db.t() @ x).to(dt), (dy.t() @ h).to(dt)


def _plain_int8(s):
    c = s["case"]
    if c["kind"] == "linear":
        x = s["x"].float()
        amax = x.abs().amax(1, keepdim=True)
        a = torch.round(x * 127.0 / torch.where(amax > 0, amax, torch.ones_like(amax)))
        sa = amax[:, 0] / 127.0
    else:
        a, sa = s["a"], s["sa"]
    acc = a.double() @ s["w"].double().t()          # whole numbers beyond 2^24: exact in 64 bits only
    return (acc.float() * sa[:, None] * s["sw"][None, :]).to(TYPES[c["out"]])


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    t = s["t"].double()[:, None]
    best = x.amax(1, keepdim=True)
    w = torch.exp((x - best) / torch.where(t > 0, t, torch.ones_like(t)))
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    ws = w.gather(1, order)
    cum = torch.cumsum(ws, 1)
    n = torch.full((B, 1), V, dtype=torch.int64, device=x.device)
    if s["k"] is not None:
        k = s["k"].long()[:, None]
        n = torch.where(k > 0, torch.minimum(k, n), n)
    if s["p"] is not None:
        p = s["p"].double()[:, None]
        short = (cum < p * cum.gather(1, n - 1)).sum(1, keepdim=True) + 1
        n = torch.where(p < 1, torch.minimum(short, n), n)
    if s["m"] is not None:
        m = s["m"].double()[:, None]
        n = torch.where(m > 0, torch.minimum((ws >= m).sum(1, keepdim=True).clamp(min=1), n), n)
    n = torch.where(t > 0, n, torch.ones_like(n))
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(V, device=x.device).expand(B, V))
    w = torch.where(rank < n, w, torch.zeros_like(w))
    cum = torch.cumsum(w, 1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    last = V - 1 - (w > 0).flip(1).int().argmax(1, keepdim=True)
    token = torch.minimum(token, last)
    prob = (w.gather(1, token) / total).float()
    return token[:, 0], prob[:, 0]


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return _plain_ffn(s) if kind in ("ffn", "train") else _plain_sample(s) if kind == "sample" else _plain_int8(s)
    n, c = _native(), s["case"]
    if kind == "ffn":
        return n.ffn_forward(s["x"], s["wg"], s["wu"], s["wd"], act_limit=c["act_limit"])
    if kind == "train":
        y, g, u = n.ffn_forward(s["x"], s["wg"], s["wu"], s["wd"], act_limit=c["act_limit"], save=True)
        return (y,) + tuple(n.ffn_backward(s["dy"], s["x"], g, u, s["wg"], s["wu"], s["wd"], act_limit=c["act_limit"]))
    if kind == "linear":
        return n.linear_i8(s["x"], s["w"], s["sw"], dtype=TYPES[c["out"]])
    if kind == "gemm":
        return n.gemm_i8(s["a"], s["sa"], s["w"], s["sw"], dtype=TYPES[c["out"]])
    return n.sample(s["logits"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"])


def work(case):
    c = case
    if c["kind"] == "ffn":
        M, H, I = c["M"], c["H"], c["I"]
        return {"bytes": 2 * (2 * M * H + 3 * H * I), "flops": 6 * M * H * I}
    if c["kind"] == "train":
        M, H, I = c["M"], c["H"], c["I"]
        return {"bytes": 2 * (4 * M * H + 6 * H * I), "flops": 18 * M * H * I}
    if c["kind"] in ("linear", "gemm"):
        M, K, N = c["M"], c["K"], c["N"]
        xb = 2 * M * K if c["kind"] == "linear" else M * K + 4 * M
        return {"bytes": xb + N * K + 4 * N + M * N * (4 if c["out"] == "f32" else 2), "flops": 2 * M * N * K}
    B, V = c["B"], c["V"]
    return {"bytes": B * V * (4 if c["type"] == "f32" else 2) + 32 * B, "flops": 4 * B * V}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def _exact_ffn(s):
    c = s["case"]
    x, wg, wu, wd = (s[n].to(torch.float64) for n in ("x", "wg", "wu", "wd"))
    L = c["act_limit"] or math.inf
    g, u = torch.mm(x, wg.T), torch.mm(x, wu.T)
    sig = torch.sigmoid(g)
    silu = g * sig
    act, up = torch.clamp(silu, max=L), torch.clamp(u, min=-L, max=L)
    h = act * up
    y = torch.mm(h, wd.T)
    if c["kind"] == "ffn":
        return y
    dy = s["dy"].to(torch.float64)
    dh = torch.mm(dy, wd)
    dg = torch.where(silu > L, 0.0, dh * up * (sig + silu * (1.0 - sig)))
    du = torch.where(u.abs() > L, 0.0, dh * act)
    return y, torch.mm(dg, wg) + torch.mm(du, wu), torch.mm(dg.T, x), torch.mm(du.T, x), torch.mm(dy.T, h)


def _exact_int8(s):
    if "x" in s:
        x = s["x"].to(torch.float64)
        top = torch.max(torch.abs(x), dim=1).values
        a = torch.where(top[:, None] > 0, torch.round(127.0 * x / top[:, None]), 0.0)
        sa = top / 127.0
    else:
        a, sa = s["a"].to(torch.float64), s["sa"].to(torch.float64)
    return torch.mm(a * sa[:, None], (s["w"].to(torch.float64) * s["sw"].to(torch.float64)[:, None]).T)


def _exact_sample(s):
    """Row by row on the sorted values: the kept set is the first n of the descending order."""
    tokens, probs = [], []
    for b in range(s["logits"].shape[0]):
        x = s["logits"][b].to(torch.float64)
        val, idx = torch.sort(-x, stable=True)
        val = -val
        t = float(s["t"][b])
        if t <= 0:
            tokens.append(idx[0])
            probs.append(torch.ones((), dtype=torch.float64, device=x.device))
            continue
        e = torch.exp((val - val[0]) / t)
        n = x.numel()
        if s["k"] is not None and int(s["k"][b]) > 0:
            n = min(n, int(s["k"][b]))
        m = n
        if s["p"] is not None and float(s["p"][b]) < 1:
            mass = torch.cumsum(e[:n], 0)
            m = min(m, int(torch.searchsorted(mass, float(s["p"][b]) * mass[-1])) + 1)
        if s["m"] is not None and float(s["m"][b]) > 0:
            m = min(m, max(1, int((e >= float(s["m"][b])).sum())))
        keep, at = torch.sort(idx[:m])
        e = e[:m][at]
        mass = torch.cumsum(e, 0)
        i = min(int(torch.searchsorted(mass, float(s["u"][b]) * mass[-1], right=True)), m - 1)
        while i > 0 and float(e[i]) == 0.0:
            i -= 1
        tokens.append(keep[i])
        probs.append(e[i] / mass[-1])
    return torch.stack(tokens), torch.stack(probs)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    return _exact_ffn(s) if kind in ("ffn", "train") else _exact_sample(s) if kind == "sample" else _exact_int8(s)
