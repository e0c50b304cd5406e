"""8-bit weights, quantised activations, routing and routed experts in 64 bits, straight from their formulas."""
from __future__ import annotations

import torch

B = 128
F64 = torch.float64


def blocks_of(x):
    """x [n, K] as [n, ceil(K / 128), 128], zeros behind."""
    n, K = x.shape
    out = torch.zeros(n, -(-K // B) * B, dtype=F64, device=x.device)
    out[:, :K] = x
    return out.view(n, -1, B)


def scales_of(x):
    """[n, blocks]: the smallest power of two s >= 2^-100 with max |x| of the block <= 448 s; NaN where the block is not finite."""
    amax = blocks_of(x).abs().amax(dim=2)
    s = torch.full_like(amax, 2.0 ** -100)
    finite = torch.isfinite(amax)
    while True:
        small = finite & (448.0 * s < amax)
        if not small.any():
            break
        s = torch.where(small, 2.0 * s, s)
    return torch.where(finite, s, torch.full_like(s, float("nan")))


def to_grid(v):
    """The nearest e4m3 value (ties to even) of |v| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0) - 3.0)
    return torch.round(v / step) * step


def quantised(x):
    """(values q [n, K], scales [n, blocks]) of x [n, K] float64."""
    s = scales_of(x)
    q = to_grid(blocks_of(x) / s[:, :, None])
    return q.reshape(x.shape[0], -1)[:, :x.shape[1]], s


def quantised_values(x):
    q, s = quantised(x)
    return (blocks_of(q) * s[:, :, None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def weight_values(q, scales):
    M, K = q.shape
    return q.to(F64) * scales.to(F64).repeat_interleave(B, 0)[:M].repeat_interleave(B, 1)[:, :K]


def product_bound(x, w):
    """How far the 32-bit sums may be from x . w^T: a block's 128 exact products are added in 32-bit (each addition rounds or truncates the running
    sum: a step of 2^-23), every block's sum and scale product then once more."""
    return (x.abs() @ w.abs().t()) * ((B + 2 * -(-x.shape[1] // B) + 4) * 2.0 ** -23)


def silu(g):
    return g / (1.0 + torch.exp(-g))


def gated(x, gate, up):
    """silu(x gate^T) * (x up^T) and how far 32-bit may be from it: silu's slope lies within +-1.1, its exponential and division are a few units in the
    last place each (the exponential's argument is rounded: |g| more of them)."""
    g, u = x @ gate.t(), x @ up.t()
    eg, eu = product_bound(x, gate), product_bound(x, up)
    z = silu(g) * u
    return z, 1.1 * eg * (u.abs() + eu) + silu(g).abs() * eu + z.abs() * (8.0 + 2.0 * g.abs()) * 2.0 ** -23


def requantised_slack(z, ez):
    """How far the quantised values of a z that is off by up to ez may be from the quantised z: one step where the value or its block's scale can fall
    on the other side of a border, nothing elsewhere."""
    s = scales_of(z)
    bz, be = blocks_of(z), blocks_of(ez)
    v, e = bz / s[:, :, None], be / s[:, :, None] + 2.0 ** -22 * (bz / s[:, :, None]).abs()
    near = (to_grid((v + e).clamp(-448, 448)) != to_grid((v - e).clamp(-448, 448)))
    amax, eamax = bz.abs().amax(dim=2), be.amax(dim=2) + 2.0 ** -22 * bz.abs().amax(dim=2)
    border = (448.0 * s < amax + eamax) | ((224.0 * s >= amax - eamax) & (s > 2.0 ** -100))
    step = torch.maximum(2.0 ** -3 * bz.abs(), 2.0 ** -8 * s[:, :, None])
    slack = torch.where(near | border[:, :, None], step, torch.zeros_like(step))
    return slack.reshape(z.shape[0], -1)[:, :z.shape[1]]


def experts(x, choice, weights, gate, up, down):
    """(out, bound): choice [n, top], weights [top, n], lists of float64 matrices; ids outside the lists have no term."""
    n, top = choice.shape
    W = down[0].shape[0]
    out, bound = torch.zeros(n, W, dtype=F64, device=x.device), torch.zeros(n, W, dtype=F64, device=x.device)
    xv = quantised_values(x)
    for e in range(len(down)):
        rows, ks = torch.nonzero(choice == e, as_tuple=True)
        if rows.numel() == 0:
            continue
        z, ez = gated(xv[rows], gate[e], up[e])
        zv = quantised_values(z)
        w = weights[ks, rows].to(F64)[:, None]
        y = zv @ down[e].t()
        b = product_bound(zv, down[e]) + requantised_slack(z, ez) @ down[e].abs().t()
        out.index_add_(0, rows, w * y)
        bound.index_add_(0, rows, w.abs() * (b + (top + 2) * 2.0 ** -24 * y.abs()))
    return out, bound


def route(z, top, score, bias=None, groups=1, top_groups=1, group_best=2, renormalise=True, scale=1.0):
    """Row by row, from the definition: (choice [n][top], weights [top, n] float64)."""
    z = z.to(F64)
    n, E = z.shape
    choice, weights = [], torch.zeros(top, n, dtype=F64)
    for t in range(n):
        row = [min(float(v), 3.4028234663852886e38) if v == v else float("-inf") for v in z[t].tolist()]
        is_open = [v > float("-inf") for v in row]
        if score == "softmax":
            high = max((v for v, o in zip(row, is_open) if o), default=0.0)
            s = [float(torch.exp(torch.tensor(v - high, dtype=F64))) if o else 0.0 for v, o in zip(row, is_open)]
            total = sum(s)
            s = [v / total if total > 0 else 0.0 for v in s]
        else:
            s = torch.where(torch.tensor(is_open), 1.0 / (1.0 + torch.exp(-torch.tensor(row, dtype=F64))), torch.zeros(E, dtype=F64)).tolist()
        b = [0.0] * E if bias is None else [float(v) for v in bias]
        is_open = [o and bv > float("-inf") for o, bv in zip(is_open, b)]
        c = [sv + bv for sv, bv in zip(s, b)]
        if groups > 1:
            size = E // groups
            judged = []
            for g in range(groups):
                best = sorted((c[e] for e in range(g * size, (g + 1) * size) if is_open[e]), reverse=True)[:group_best]
                judged.append(sum(best) if best else float("-inf"))
            kept = sorted(range(groups), key=lambda g: (-judged[g], g))[:top_groups]
            is_open = [o and e // size in kept for e, o in enumerate(is_open)]
        order = sorted((e for e in range(E) if is_open[e]), key=lambda e: (-c[e], e))[:top]
        total = sum(s[e] for e in order)
        for k, e in enumerate(order):
            weights[k, t] = s[e] * scale / (total + 1e-20) if renormalise else s[e] * scale
        choice.append(order + [-1] * (top - len(order)))
    return torch.tensor(choice, dtype=torch.int32).view(n, top), weights
