"""What a served or fine-tuned MoE model computes next to its experts and its dense layers, as cases that can be timed and
compared: the choice of experts from the router's logits, products with 4-bit weights, and the adjusting of the head's logits
before a token is drawn.

Kinds of case:
  route   scores (sigmoid or softmax), a bias for balance, groups, top-k, weights: the picks of each token
  train   the same, then the gradient of the logits for a given gradient of the weights
  linear  a linear layer whose weight has 4 bits, with a scale (and a zero point) for each group of inputs
  dx      the gradient of that layer's input for a given gradient of its output
  logits  penalties for tokens that were there before, biases, a grammar's mask

With `own` false a pass is the plain form, elementary torch operations in 32 bits (64 where 32 lose what matters: values next to
the border of a choice); with `own` true it makes the calls of glm-flash-lite_amd/_native.py. Weights are in hand before a pass,
in the layout that those calls read.
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
INF = float("inf")


def _native():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import _native as n
    return n


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------

def _route(name, kind, M, E, **kw):
    return dict(dict(name=name, kind=kind, M=M, E=E, topk=8, type="f32", score="sigmoid", bias=True, groups=1, top_groups=1,
                     group_best=2, renorm=True, scale=1.0, wtype="f16", off=0.0), **kw)


def _linear(name, kind, M, K, N, **kw):
    return dict(dict(name=name, kind=kind, M=M, K=K, N=N, type="bf16", out="bf16", group=128, zeros=False, strided=False), **kw)


def _logits(name, B, V, L, **kw):
    return dict(dict(name=name, kind="logits", B=B, V=V, L=L, type="f32", nbias=0, masked=-1.0, pad=0), **kw)


def listed():
    return [
        # one token of a decode step through the served model's router: 288 experts, a bias for balance
        _route("route-1", "route", 1, 288),
        # a prompt chunk through a router of eight groups, four of which a token may use
        _route("route-8192", "route", 8192, 256, groups=8, top_groups=4, scale=2.5),
        # a fine-tuning step's tokens, softmax scores that are not renormalised: every logit has a gradient
        _route("route-train-16384", "train", 16384, 128, type="bf16", score="softmax", bias=False, renorm=False, scale=16.0,
               wtype="f32"),
        # a projection of one token
        _linear("linear4-1", "linear", 1, 5120, 5120),
        # five draft tokens through a layer of odd sizes, small groups with zero points, the tokens a slice of a wider buffer
        _linear("linear4-5", "linear", 5, 4072, 11007, type="f16", out="f16", group=64, zeros=True, strided=True),
        # the head for nine users: logits in fp32
        _linear("head4-9", "linear", 9, 4096, 65536, out="f32"),
        # a batch of users through a down projection, the smallest groups
        _linear("linear4-50", "linear", 50, 12288, 5120, group=32, type="f16", out="f16"),
        # a prompt chunk
        _linear("linear4-4096", "linear", 4096, 5120, 12288),
        # the step back through a frozen 4-bit layer in fine-tuning
        _linear("dx-1001", "dx", 1001, 4096, 11008, zeros=True),
        # one user's logits, an answer of some hundred tokens after a short prompt
        _logits("logits-1", 1, 131072, 2000),
        # a small server's batch over an odd vocabulary, bf16, a grammar that allows few tokens, biases
        _logits("logits-24", 24, 100003, 9000, type="bf16", nbias=40, masked=0.99, pad=5),
        # the largest batch, long prompts
        _logits("logits-256", 256, 131072, 30000, nbias=300, masked=0.3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A matrix size: a multiple of 128 most of the time, else of 8, now and then any number."""
    n, r = _log_int(rng, lo, hi), rng.random()
    return n if r < 0.1 else max(8, n // 8 * 8) if r < 0.35 else max(128, n // 128 * 128)


def draw(rng):
    kind = rng.choice(["route", "route", "train", "linear", "linear", "linear", "dx", "logits", "logits"])
    if kind in ("route", "train"):
        groups = rng.choice([1, 1, 1, 4, 8])
        E = rng.choice([groups * rng.randint(4, 32), 8 * _log_int(rng, 2, 64), 288])
        E = max(16, E // groups * groups)
        top_groups = rng.randint(1, groups)
        topk = min(rng.choice([1, 2, 4, 6, 8, 8, 8, 16]), E // groups * top_groups)
        score = rng.choice(["sigmoid", "softmax"])
        M = rng.choice([rng.randint(1, 16), _log_int(rng, 17, 512), min(_log_int(rng, 513, 16384), 16384 * 128 // E)])
        # one pick that is renormalised weighs 1 whatever its logit: nothing to train
        renorm = rng.random() < 0.7 and not (kind == "train" and topk == 1)
        return dict(kind=kind, M=M, E=E, topk=topk,
                    type=rng.choice(["f32", "f32", "bf16", "f16"]), score=score, bias=rng.random() < 0.6, groups=groups,
                    top_groups=top_groups, group_best=rng.choice([1, 2]), renorm=renorm,
                    scale=rng.choice([1.0, 1.0, 2.5]), wtype="f32" if kind == "train" else rng.choice(["f16", "f32", "bf16"]),
                    off=rng.choice([0.0, 0.0, 0.05]))
    if kind in ("linear", "dx"):
        M = rng.choice([rng.randint(1, 16), _log_int(rng, 17, 512), _log_int(rng, 513, 4096)])
        N = _size(rng, 4096, 65536) if M <= 64 and rng.random() < 0.4 else _size(rng, 64, 12288)
        t = rng.choice(["f16", "bf16"])
        K = _size(rng, 128, 4096 if N > 12288 else 12288 if M <= 64 else 5120)
        return dict(kind=kind, M=M, K=K, N=N, type=t,
                    out=t if kind == "dx" else rng.choice([t, t, "f32"]), group=rng.choice([32, 64, 128, 128]),
                    zeros=rng.random() < 0.5, strided=rng.random() < 0.3)
    return dict(kind=kind, B=_log_int(rng, 1, 256), V=_log_int(rng, 1000, 131072), L=rng.choice([0, 1, _log_int(rng, 2, 30000)]),
                type=rng.choice(["f32", "f32", "bf16", "f16"]), nbias=rng.choice([0, 0, 7, 300]),
                masked=rng.choice([-1.0, -1.0, 0.0, 0.3, 0.99, 1.0]), pad=rng.choice([0, 0, 5, 64]))


# ---------------------------------------------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 31)
    return g


def _randn(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV).mul_(scale)


def _rand(g, shape):
    return torch.rand(shape, generator=g, device=DEV)


def _tokens(g, M, K, dt, strided):
    """Activations: normal, one channel in 128 eight times as large, as the residual stream of a trained model has."""
    x = _randn(g, (M, K))
    x[:, torch.randint(0, K, (max(1, K // 128),), generator=g, device=DEV)] *= 8.0
    if not strided:
        return x.to(dt)
    wide = torch.zeros((M, K + 64), dtype=dt, device=DEV)
    wide[:, 32:32 + K] = x.to(dt)
    return wide[:, 32:32 + K]


def _pack(v):
    """Values 0..15 [N, K] as the products read them: each 128 inputs 64 bytes, of which the 32-bit word j of the 16-byte piece g
    holds the inputs 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7), four bits each from the lowest on."""
    N, K = v.shape
    blocks = (K + 127) // 128
    full = torch.zeros((N, blocks * 128), dtype=torch.uint8, device=v.device)
    full[:, :K] = v
    e = full.view(N, blocks, 4, 4, 4, 2)                     # block, j, g, pair, of a pair
    e = e.permute(0, 1, 3, 2, 5, 4).reshape(N, blocks * 64, 2)   # block, g, j, first or second of all pairs, pair
    return (e[..., 0] | (e[..., 1] << 4)).contiguous()


def _unpack(q, K):
    N = q.shape[0]
    e = torch.stack((q & 15, q >> 4), -1).view(N, -1, 4, 4, 2, 4)   # block, g, j, first or second, pair
    return e.permute(0, 1, 3, 2, 5, 4).reshape(N, -1)[:, :K]


def _weight4(g, N, K, group, zeros, dt):
    """A normal weight rounded to 4 bits: (packed, scale [groups, N], zero [groups, N] or None)."""
    n = (K + group - 1) // group
    w = torch.zeros((N, n * group), device=DEV)
    w[:, :K] = _randn(g, (N, K), 1.0 / math.sqrt(K))
    w = w.view(N, n, group)
    if zeros:
        lo, hi = w.amin(2, keepdim=True).clamp(max=0), w.amax(2, keepdim=True).clamp(min=0)
        s = ((hi - lo) / 15).to(dt).float()
        z = torch.round(-lo / s)
    else:
        s = (w.abs().amax(2, keepdim=True) / 7).to(dt).float()
        z = torch.full_like(s, 8.0)
    v = (torch.round(w / s) + z).clamp_(0, 15).view(N, n * group)[:, :K].to(torch.uint8)
    rows = lambda t: t[:, :, 0].t().contiguous()
    return _pack(v), rows(s).to(dt), rows(z).to(torch.uint8) if zeros else None


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] in ("route", "train"):
        M, E = c["M"], c["E"]
        logits = _randn(g, (M, E), 1.5).add_(_randn(g, (1, E), 0.5))     # some experts are liked by all
        if c["off"]:
            logits[:, _rand(g, (E,)) < c["off"]] = -INF                  # experts that are out of service
        s = dict(case=c, logits=logits.to(TYPES[c["type"]]), bias=_randn(g, (E,), 0.05) if c["bias"] else None)
        if c["kind"] == "train":
            s["dw"] = _randn(g, (M, c["topk"])).to(TYPES[c["wtype"]])
        return s
    if c["kind"] in ("linear", "dx"):
        M, K, N, dt = c["M"], c["K"], c["N"], TYPES[c["type"]]
        q, scale, zero = _weight4(g, N, K, c["group"], c["zeros"], dt)
        return dict(case=c, q=q, scale=scale, zero=zero, x=_tokens(g, M, K if c["kind"] == "linear" else N, dt, c["strided"]))
    B, V, L = c["B"], c["V"], c["L"]
    x = _randn(g, (B, V), 2.5)
    peak = torch.randint(0, V, (B, 12), generator=g, device=DEV)
    x.scatter_add_(1, peak, 8.0 + 4.0 * _rand(g, (B, 12)))
    logits = torch.zeros((B, V + c["pad"]), dtype=TYPES[c["type"]], device=DEV)[:, :V]
    logits.copy_(x)
    # text: few tokens often, many now and then
    history = (V * _rand(g, (B, L)).double().pow(4)).long().clamp_(max=V - 1).int()
    lengths = (L * (0.5 + 0.5 * _rand(g, (B,)))).round().int()
    s = dict(case=c, logits=logits, history=history, lengths=lengths, prompt=(lengths * _rand(g, (B,))).int(),
             repetition=1.0 + 0.3 * _rand(g, (B,)), frequency=0.5 * _rand(g, (B,)), presence=_rand(g, (B,)) - 0.2,
             bias_ids=None, bias=None, allowed=None)
    s["repetition"][_rand(g, (B,)) < 0.3] = 1.0       # each user's own settings: some leave a penalty off
    s["frequency"][_rand(g, (B,)) < 0.3] = 0.0
    s["presence"][_rand(g, (B,)) < 0.3] = 0.0
    if c["nbias"]:
        s["bias_ids"] = torch.randint(-1, V, (B, c["nbias"]), generator=g, device=DEV, dtype=torch.int32)
        s["bias"] = _randn(g, (B, c["nbias"]), 5.0)
    if c["masked"] >= 0:
        words = (V + 31) // 32
        bits = torch.zeros((B, words * 32), dtype=torch.int64, device=DEV)
        bits[:, :V] = _rand(g, (B, V)) >= c["masked"]
        m = (bits.view(B, words, 32) << torch.arange(32, device=DEV)).sum(2)
        s["allowed"] = torch.where(m >= 2 ** 31, m - 2 ** 32, m).int()
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------

def _plain_route(s):
    c = s["case"]
    x, k = s["logits"].double(), c["topk"]
    M, E = x.shape
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    biased = score + s["bias"].double() if c["bias"] else score
    there = x > -INF
    biased = torch.where(there, biased, -INF)
    key = biased if c["bias"] else torch.where(there, x, -INF)      # without a bias the logits are in the scores' order
    if c["groups"] > 1:
        by = torch.sort(biased.view(M, c["groups"], -1), dim=2, descending=True)[0][:, :, :c["group_best"]]
        worth = torch.where(by[:, :, 0] > -INF, torch.where(by > -INF, by, 0.0).sum(2), -INF)
        order = torch.sort(worth, dim=1, descending=True, stable=True)[1]
        kept = torch.zeros((M, c["groups"]), dtype=torch.bool, device=x.device).scatter_(1, order[:, :c["top_groups"]], True)
        key = torch.where(kept.repeat_interleave(E // c["groups"], dim=1), key, -INF)
    val, idx = torch.sort(key, dim=1, descending=True, stable=True)
    picked, sel = val[:, :k] > -INF, idx[:, :k]
    p = torch.where(picked, score.gather(1, sel), 0.0)
    total = p.sum(1, keepdim=True) if c["renorm"] else torch.ones_like(p[:, :1])
    w = c["scale"] * p / torch.where(total > 0, total, 1.0)
    out = torch.where(picked, sel, -1), w.to(TYPES[c["wtype"]])
    if c["kind"] == "route":
        return out
    dw = torch.where(picked, s["dw"].double() * c["scale"], 0.0)
    if c["renorm"]:
        dw = (dw - (dw * p).sum(1, keepdim=True) / total) / total
    ds = torch.zeros_like(x).scatter_add_(1, sel, torch.where(picked, dw, 0.0))
    if c["score"] == "sigmoid":
        dx = ds * score * (1.0 - score)
    else:
        dx = score * (ds - (ds * score).sum(1, keepdim=True))
    return out + (dx.to(s["logits"].dtype),)


def _plain_weight(s, K):
    c = s["case"]
    of = torch.arange(K, device=DEV) // c["group"]
    v = _unpack(s["q"], K).float()
    scale = s["scale"].float().t()
    zero = s["zero"].float().t() if c["zeros"] else torch.full_like(scale, 8.0)
    return (v - zero[:, of]) * scale[:, of]


def _plain_linear(s):
    c = s["case"]
    w = _plain_weight(s, c["K"])
    return (s["x"].float() @ (w.t() if c["kind"] == "linear" else w)).to(TYPES[c["out"]])


def _plain_logits(s):
    c = s["case"]
    B, V = s["logits"].shape
    y = s["logits"].float()
    at = torch.arange(c["L"], device=DEV)[None, :]
    ids, there = s["history"].long(), at < s["lengths"][:, None]
    zeros = lambda: torch.zeros((B, V), dtype=torch.int32, device=DEV)
    seen = zeros().scatter_add_(1, ids, there.int()) > 0
    count = zeros().scatter_add_(1, ids, (there & (at >= s["prompt"][:, None])).int())
    r = s["repetition"][:, None]
    y = torch.where(seen, torch.where(y > 0, y / r, y * r), y)
    y = y - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if c["nbias"]:
        # the last entry of an id counts
        n = torch.arange(1, c["nbias"] + 1, device=DEV, dtype=torch.int32).expand(B, -1)
        n = torch.where(s["bias_ids"] >= 0, n, 0)
        last = zeros().scatter_reduce_(1, s["bias_ids"].long().clamp(min=0), n, "amax").long()
        y = y + torch.where(last > 0, s["bias"].gather(1, (last - 1).clamp(min=0)), 0.0)
    if s["allowed"] is not None:
        v = torch.arange(V, device=DEV)
        y = torch.where((s["allowed"][:, v // 32] >> (v % 32) & 1) > 0, y, -INF)
    return y.to(s["logits"].dtype)


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return (_plain_route if kind in ("route", "train") else _plain_linear if kind in ("linear", "dx") else _plain_logits)(s)
    n = _native()
    if kind in ("route", "train"):
        sel, w = n.route_experts(s["logits"], c["topk"], bias=s["bias"], score=c["score"], groups=c["groups"],
                                 top_groups=c["top_groups"], group_best=c["group_best"], renorm=c["renorm"], scale=c["scale"],
                                 dtype=TYPES[c["wtype"]])
        if kind == "route":
            return sel, w
        return sel, w, n.route_experts_backward(s["dw"], s["logits"], sel, score=c["score"], renorm=c["renorm"], scale=c["scale"])
    if kind == "linear":
        return n.linear_i4(s["x"], s["q"], s["scale"], zero=s["zero"], group=c["group"], dtype=TYPES[c["out"]])
    if kind == "dx":
        return n.linear_i4_dx(s["x"], s["q"], s["scale"], c["K"], zero=s["zero"], group=c["group"])
    return n.adjust_logits(s["logits"], history=s["history"], lengths=s["lengths"], prompt=s["prompt"],
                           repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                           bias_ids=s["bias_ids"], bias=s["bias"], allowed=s["allowed"])


def work(case):
    c = case
    size = lambda t: 4 if t == "f32" else 2
    if c["kind"] in ("route", "train"):
        M, E, k = c["M"], c["E"], c["topk"]
        b = M * E * size(c["type"]) + M * k * (8 + size(c["wtype"])) + 4 * E * c["bias"]
        if c["kind"] == "train":
            b += M * E * size(c["type"]) + M * k * size(c["wtype"])
        return {"bytes": b, "flops": M * E * (16 if c["kind"] == "train" else 8)}
    if c["kind"] in ("linear", "dx"):
        M, K, N = c["M"], c["K"], c["N"]
        groups = (K + c["group"] - 1) // c["group"]
        io = 2 * M * K + size(c["out"]) * M * N if c["kind"] == "linear" else 2 * M * (K + N)
        return {"bytes": io + N * K // 2 + N * groups * (3 if c["zeros"] else 2), "flops": 2 * M * N * K}
    B, V = c["B"], c["V"]
    b = 2 * B * V * size(c["type"]) + 3 * B * c["L"] + 8 * B * c["nbias"] + 20 * B + (B * V // 8 if c["masked"] >= 0 else 0)
    return {"bytes": b, "flops": 4 * B * V}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def _ranks(v):
    """[..., n]: how many come before each: larger ones, and equal ones with a lower index."""
    a, b = v[..., :, None], v[..., None, :]
    i = torch.arange(v.shape[-1], device=v.device)
    return ((b > a) | ((b == a) & (i[None, :] < i[:, None]))).sum(-1)


def _exact_route_rows(c, logits, bias, dw):
    x = logits.to(torch.float64)
    M, E = x.shape
    p = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, dim=1)
    b = p if bias is None else p + bias.to(torch.float64)[None, :]
    dead = torch.isneginf(x)
    rank_by = (x if bias is None else b).masked_fill(dead, -INF)
    if c["groups"] > 1:
        size = E // c["groups"]
        v = b.masked_fill(dead, -INF).reshape(M, c["groups"], size)
        best = _ranks(v) < min(c["group_best"], size)
        worth = torch.where(best & ~torch.isneginf(v), v, 0.0).sum(2).masked_fill(dead.reshape(v.shape).all(2), -INF)
        out = _ranks(worth) >= c["top_groups"]
        rank_by = rank_by.masked_fill(out[:, :, None].expand(-1, -1, size).reshape(M, E), -INF)
    rank = _ranks(rank_by)
    rank = torch.where(torch.isneginf(rank_by), E, rank)
    hit = rank[:, None, :] == torch.arange(c["topk"], device=x.device)[None, :, None]      # token, place, expert
    some = hit.any(2)
    sel = torch.where(some, hit.to(torch.uint8).argmax(2), -1)
    h = hit.to(torch.float64)
    s = (h * p[:, None, :]).sum(2)
    total = s.sum(1, keepdim=True) if c["renorm"] else torch.ones((M, 1), dtype=torch.float64, device=x.device)
    w = torch.where(total > 0, c["scale"] * s / total, 0.0)
    if dw is None:
        return sel, w
    up = dw.to(torch.float64) * some
    if c["renorm"]:      # dw_j / ds_i = (scale delta_ij - w_j) / total
        ds = (c["scale"] * up - (up * w).sum(1, keepdim=True)) / total
    else:
        ds = c["scale"] * up
    of = (h * ds[:, :, None]).sum(1)
    if c["score"] == "sigmoid":
        return sel, w, of * p * torch.sigmoid(-x)
    return sel, w, p * of - p * (p * of).sum(1, keepdim=True)


def _exact_route(s):
    c = s["case"]
    step = max(1, (1 << 26) // c["E"] ** 2)
    parts = []
    for i in range(0, c["M"], step):
        parts.append(_exact_route_rows(c, s["logits"][i:i + step], s["bias"],
                                       s["dw"][i:i + step] if c["kind"] == "train" else None))
    return tuple(torch.cat(t) for t in zip(*parts))


def _exact_linear(s):
    c = s["case"]
    K, N, G = c["K"], c["N"], c["group"]
    n = (K + G - 1) // G
    low, high = s["q"] % 16, s["q"] // 16
    v = torch.zeros((N, (K + 127) // 128, 128), dtype=torch.float64, device=DEV)
    for byte in range(64):
        g, j, at = byte // 16, byte % 16 // 4, byte % 4
        for half, t in ((0, low), (1, high)):
            place = 2 * at + half                                 # of the word's eight values
            v[:, :, 32 * j + 8 * g + (0, 2, 4, 6, 1, 3, 5, 7)[place]] = t[:, byte::64].double()
    v = v.reshape(N, -1)[:, :K]
    pad = torch.zeros((N, n * G), dtype=torch.float64, device=DEV)
    pad[:, :K] = v
    zero = 8.0 if s["zero"] is None else s["zero"].double().T[:, :, None]
    w = ((pad.reshape(N, n, G) - zero) * s["scale"].double().T[:, :, None]).reshape(N, n * G)[:, :K]
    return torch.mm(s["x"].double(), w.T.contiguous() if c["kind"] == "linear" else w.contiguous())


def _exact_logits(s):
    """Row by row, with each row's own lists."""
    c = s["case"]
    rows = []
    host = {n: s[n].cpu() for n in ("lengths", "prompt")}
    for b in range(c["B"]):
        n, p = int(host["lengths"][b]), int(host["prompt"][b])
        y = s["logits"][b].double()
        count = torch.bincount(s["history"][b, p:n].long(), minlength=c["V"]).double() if n > p else torch.zeros_like(y)
        seen = torch.unique(s["history"][b, :n].long())
        r = s["repetition"][b].double()
        y[seen] = torch.maximum(y[seen], torch.zeros_like(y[seen])) / r + torch.minimum(y[seen], torch.zeros_like(y[seen])) * r
        y = y - count * s["frequency"][b].double() - torch.clamp(count, max=1.0) * s["presence"][b].double()
        if c["nbias"]:
            ids, by = s["bias_ids"][b].long(), s["bias"][b].double()
            i = torch.arange(len(ids), device=DEV)
            again = ((ids[:, None] == ids[None, :]) & (i[None, :] > i[:, None])).any(1)
            ok = (ids >= 0) & ~again
            y[ids[ok]] += by[ok]
        if s["allowed"] is not None:
            bits = (s["allowed"][b].long() & 0xFFFFFFFF)[:, None] // (2 ** torch.arange(32, device=DEV)) % 2
            y[bits.reshape(-1)[:c["V"]] == 0] = -INF
        rows.append(y)
    return torch.stack(rows)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    return _exact_route(s) if kind in ("route", "train") else _exact_linear(s) if kind in ("linear", "dx") else _exact_logits(s)
