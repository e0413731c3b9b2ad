"""The dense operators in 64 bits, on the CPU, with bounds on how far 32-bit sums and 16-bit roundings can move each output.

Roundings: a value rounded to 16 bits is off by at most eps/2 of itself (plus half the smallest subnormal); an fp32 sum of n
products by at most n + 2 units of 2^-23 of the sum of the products' magnitudes (a matrix instruction may truncate where an
fp32 add rounds, so a whole unit counts per step). The device's sigmoid (v_exp_f32, v_rcp_f32, each within a unit
in the last place of its fp32 argument's result) is off by at most (8 + 2|g|) 2^-23 of itself.
"""
import math

import torch

U32 = 2.0 ** -23


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dt]


def _mm(a, b):
    return a @ b.t()


class FFN:
    """The block and its gradients for float64 copies of the inputs: value, bound for each output. err_* are bounds on the
    device's intermediate values."""

    def __init__(self, x, wg, wu, wd, L=0.0, out_dt=None, f32_h=False):
        dt = x.dtype
        self.dt, self.L = dt, L or math.inf
        u = half_step(dt)
        x, wg, wu, wd = (t.double().cpu() for t in (x, wg, wu, wd))
        self.x, self.wg, self.wu, self.wd = x, wg, wu, wd
        H, I = x.shape[1], wg.shape[0]
        self.g, self.u = _mm(x, wg), _mm(x, wu)
        self.eg = (H + 2) * U32 * _mm(x.abs(), wg.abs())
        self.eu = (H + 2) * U32 * _mm(x.abs(), wu.abs())
        self.s = torch.sigmoid(self.g)
        self.raw = self.g * self.s
        self.t, self.v = self.raw.clamp(max=self.L), self.u.clamp(-self.L, self.L)
        self.h = self.t * self.v
        et = 1.1 * self.eg + (8 + 2 * self.g.abs()) * U32 * self.raw.abs()
        self.eh = et * (self.v.abs() + self.eu) + self.eu * self.t.abs() + 2 * U32 * self.h.abs()
        self.eh16 = self.eh + u * (self.h.abs() + self.eh) + tiny(dt)
        eh = self.eh if f32_h else self.eh16
        self.y = _mm(self.h, wd)
        o = out_dt or dt
        self.ey = _mm(eh, wd.abs()) + (I + 2) * U32 * _mm(self.h.abs() + eh, wd.abs())
        self.ey = self.ey + half_step(o) * (self.y.abs() + self.ey) + tiny(o)

    def backward(self, dy):
        dt, u, L = self.dt, half_step(self.dt), self.L
        dy = dy.double().cpu()
        M, H, I = self.x.shape[0], self.x.shape[1], self.wg.shape[0]
        dh = dy @ self.wd
        edh = (H + 2) * U32 * (dy.abs() @ self.wd.abs())
        k = self.s + self.raw * (1 - self.s)
        pass_g, pass_u = self.raw <= L, self.u.abs() <= L
        dg = torch.where(pass_g, dh * self.v * k, 0.0)
        du = torch.where(pass_u, dh * self.t, 0.0)
        eg, eu = self.eg, self.eu
        ek = 0.5 * eg + (8 + 2 * self.g.abs()) * U32 * (2 + self.g.abs())
        et = 1.1 * eg + (8 + 2 * self.g.abs()) * U32 * self.raw.abs()
        a, b, c = dh.abs() + edh, self.v.abs() + eu, k.abs() + ek
        edg = edh * b * c + a * eu * c + a * b * ek + 3 * U32 * dg.abs()
        edu = edh * (self.t.abs() + et) + a * et + 3 * U32 * du.abs()
        # a value so near the clamp that fp32 may see it on the other side
        near_g = (self.raw - L).abs() <= 1.1 * self.eg + (8 + 2 * self.g.abs()) * U32 * self.raw.abs() if L < math.inf else None
        near_u = (self.u.abs() - L).abs() <= self.eu if L < math.inf else None
        if L < math.inf:
            edg = torch.where(near_g, a * b * c, torch.where(pass_g, edg, 0.0))
            edu = torch.where(near_u, a * (self.t.abs() + et), torch.where(pass_u, edu, 0.0))
        r = lambda v, e: e + u * (v.abs() + e) + tiny(dt)
        edg, edu = r(dg, edg), r(du, edu)
        eh = et * b + eu * self.t.abs() + 2 * U32 * self.h.abs()
        eh = r(self.h, eh)
        A = lambda v, e: v.abs() + e

        def out(value, err, n, mag):
            e = err + (n + 2) * U32 * mag
            return value, e + u * (value.abs() + e) + tiny(dt)

        dx = out(dg @ self.wg + du @ self.wu, edg @ self.wg.abs() + edu @ self.wu.abs(), 2 * I,
                 A(dg, edg) @ self.wg.abs() + A(du, edu) @ self.wu.abs())
        xa = self.x.abs()
        dwg = out(dg.t() @ self.x, edg.t() @ xa, M, A(dg, edg).t() @ xa)
        dwu = out(du.t() @ self.x, edu.t() @ xa, M, A(du, edu).t() @ xa)
        dwd = out(dy.t() @ self.h, dy.abs().t() @ eh, M, dy.abs().t() @ A(self.h, eh))
        return dx, dwg, dwu, dwd


def within(got, want, bound, name=""):
    got = got.double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside, first at {at}: {float(got[at])} for "
                             f"{float(want[at])} +- {float(bound[at])}")


def quant(x):
    x = x.double().cpu()
    top = x.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.round(x * 127 / torch.where(top > 0, top, 1.0)), 0.0)
    return q, top[..., 0] / 127


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """Row by row: (token, prob, margin): margin is the smallest distance, relative to the weights' sum, between a border
    of the row and the value that is compared with it."""
    logits = logits.double().cpu()
    out = []
    for b in range(logits.shape[0]):
        x = torch.where(torch.isnan(logits[b]), -math.inf, logits[b])
        val, idx = torch.sort(x, descending=True, stable=True)
        T = 1.0 if temperature is None else float(temperature[b])
        if float(val[0]) == -math.inf:
            out.append((-1, 0.0, 1.0))
            continue
        if not T > 0:
            out.append((int(idx[0]), 1.0, 1.0))
            continue
        e = torch.where(val == val[0], 1.0, torch.where((val == -math.inf) | (val[0] == math.inf), 0.0,
                                                        torch.exp((val - val[0]) / T)))   # T = inf: all the finite ones weigh 1
        n, margin = len(x), 1.0
        if top_k is not None and int(top_k[b]) > 0:
            n = min(n, int(top_k[b]))
        m = n
        p = 1.0 if top_p is None else float(top_p[b])
        if p < 1:
            cum = torch.cumsum(e[:n], 0)
            goal = p * float(cum[-1])
            i = int((cum < goal).sum())
            m = min(m, i + 1)
            if i > 0 or goal > 0:
                # a border only matters where another value is near: equal weights step by more than the margin
                margin = min(margin, float((cum - goal).abs().min() / cum[-1]))
        q = 0.0 if min_p is None else float(min_p[b])
        if q > 0:
            m = min(m, max(1, int((e >= q).sum())))
            if q < 1:
                # compared as fp64 values, each off by some 2^-50 of itself: the distance counts relative to q
                margin = min(margin, float((e - q).abs().min()) / q)
        keep, at = torch.sort(idx[:m])
        w = e[:m][at]
        cum = torch.cumsum(w, 0)
        goal = float(u[b]) * float(cum[-1])
        i = min(int((cum <= goal).sum()), m - 1)
        while i > 0 and float(w[i]) == 0:
            i -= 1
        if goal > 0:
            margin = min(margin, float((cum - goal).abs().min() / cum[-1]))
        out.append((int(keep[i]), float(w[i] / cum[-1]), margin))
    return out
