"""Plain float64 restatement of the group norm with an activation (value, first and second gradient) and of the counter-based dropout:
loops over clouds, formulas written out, no code shared with the package.  Checked on the CPU against torch's autograd, finite
differences and the generator's published vectors (tests/test_norm_drop_oracle.py); the GPU tests compare the kernels with it.

Besides every result it returns the size of the terms that result was summed from (``scale``): an fp32 evaluation can be off by a number
of half steps of THAT, however much the terms cancel."""
from __future__ import annotations

import math

import numpy as np
import torch

SLOPES = {"none": 1.0, "relu": 0.0}


# ---------------------------------------------------------------------------------------------------------------- random words
def philox4x32(ctr, key, rounds=10):
    """ctr [..., 4], key [2]: uint32 words; returns the block's words [..., 4] (Salmon et al. 2011)."""
    c = [np.asarray(ctr[..., i], dtype=np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, -1).astype(np.uint32)


def keep_mask(rows, C, p, seed, call, first_row=0):
    """Truth values [rows, C]: what dropout keeps of the rows first_row, first_row + 1, ..."""
    quads = (C + 3) // 4
    at = np.arange(rows * quads, dtype=np.uint64) + np.uint64(first_row * quads)
    seed, call = int(seed) % 2 ** 64, int(call) % 2 ** 64
    ctr = np.stack([at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.full_like(at, call & 0xFFFFFFFF), np.full_like(at, call >> 32)], -1)
    words = philox4x32(ctr, (seed & 0xFFFFFFFF, seed >> 32)).reshape(rows, 4 * quads)[:, :C]
    return torch.from_numpy(words.astype(np.float64) >= round(p * 2.0 ** 32))


def dropout(x, p, seed, call):
    """(value, mask) in float64 for x of any shape, rows = all but the last dimension."""
    C = x.shape[-1]
    keep = keep_mask(x.numel() // max(C, 1), C, p, seed, call).reshape(x.shape)
    return torch.where(keep, x.double() / (1 - p) if p < 1 else torch.zeros_like(x.double()), torch.zeros((), dtype=torch.float64)), keep


# ------------------------------------------------------------------------------------------------------------------ activations
def act(name, u, slope=0.01):
    """phi, phi', phi''."""
    if name in ("none", "relu", "leaky_relu"):
        s = SLOPES.get(name, slope)
        return torch.where(u > 0, u, u * s), torch.where(u > 0, torch.ones_like(u), torch.full_like(u, s)), torch.zeros_like(u)
    if name == "silu":
        s = torch.sigmoid(u)
        return u * s, s * (1 + u * (1 - s)), s * (1 - s) * (2 + u * (1 - 2 * s))
    cdf, pdf = torch.special.ndtr(u), torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    return u * cdf, cdf + u * pdf, pdf * (2 - u * u)


# ------------------------------------------------------------------------------------------------------------------- group norm
def group_norm(x, seg_off, G, w=None, b=None, eps=1e-5, name="none", slope=0.01, D=None, dy=None, ggx=None, ggw=None, ggb=None, order=0):
    """Everything up to ``order`` (0 value, 1 gradient, 2 second gradient) as a dict name -> (result, scale), float64.  ``D`` [M, C]: dropout's
    factors (0 or 1 / (1 - p))."""
    x = x.detach().double().cpu()
    M, C = x.shape
    Cg, seg = C // G, [int(v) for v in seg_off]
    vec = lambda t, d: torch.full((C,), d, dtype=torch.float64) if t is None else t.detach().double().cpu().reshape(-1)  # noqa: E731
    mat = lambda t: torch.zeros(M, C, dtype=torch.float64) if t is None else t.detach().double().cpu()  # noqa: E731
    w, b, D = vec(w, 1.0), vec(b, 0.0), torch.ones(M, C, dtype=torch.float64) if D is None else D.double()
    dy, P, q, s = mat(dy), mat(ggx), vec(ggw, 0.0), vec(ggb, 0.0)
    new = lambda: (torch.zeros(M, C, dtype=torch.float64), torch.zeros(M, C, dtype=torch.float64))  # noqa: E731
    y, dx, ddy, ddx = new(), new(), new(), new()
    par = {k: (torch.zeros(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)) for k in ("dw", "db", "ddw", "ddb")}
    cond = torch.ones(M, C, dtype=torch.float64)

    def put(to, rows, cols, value, scale):
        to[0][rows, cols], to[1][rows, cols] = value, scale.max()

    def add(to, cols, value):
        to[0][cols] += value.sum(0)
        to[1][cols] += value.abs().sum(0)

    for r0, r1 in zip(seg[:-1], seg[1:]):
        if r1 <= r0:
            continue
        for g in range(G):
            rows, cols = slice(r0, r1), slice(g * Cg, (g + 1) * Cg)
            X, wc, bc, Dc = x[rows, cols], w[cols], b[cols], D[rows, cols]
            mean = X.mean()
            r = 1 / torch.sqrt(((X - mean) ** 2).mean() + eps)
            cond[rows, cols] = 1 + X.abs().max() * r
            xh = (X - mean) * r
            f, f1, f2 = act(name, wc * xh + bc, slope)
            put(y, rows, cols, f * Dc, (f * Dc).abs() + Dc * ((wc * xh).abs() + bc.abs()))
            if order == 0:
                continue
            dyD = dy[rows, cols] * Dc
            gr = dyD * f1
            h = gr * wc
            m1, m2 = h.mean(), (h * xh).mean()
            put(dx, rows, cols, r * (h - m1 - xh * m2), r * (h.abs() + h.abs().mean() + xh.abs() * (h * xh).abs().mean()) + r * (dyD * wc).abs())
            add(par["dw"], cols, gr * xh)
            add(par["db"], cols, gr)
            par["dw"][1][cols] += (dyD * xh).abs().sum(0)
            par["db"][1][cols] += dyD.abs().sum(0)
            if order == 1:
                continue
            Pc = P[rows, cols]
            mp, mp2, mph = Pc.mean(), (Pc * xh).mean(), (Pc * h).mean()
            v = r * (Pc - mp - xh * mp2)
            va = r * (Pc.abs() + Pc.abs().mean() + xh.abs() * (Pc * xh).abs().mean())
            gb = wc * v + q[cols] * xh + s[cols]
            gba = wc.abs() * va + (q[cols] * xh).abs() + s[cols].abs()
            ub, uba = gb * dyD * f2, gba * dyD.abs()
            Xh = -r * (h * mp2 + Pc * m2) + q[cols] * gr + wc * ub
            ga = dyD.abs()                        # |phi'| <= 1.13, |phi''| <= 0.8 for every activation here
            ha = ga * wc.abs()
            Xa = r * (ha * (Pc * xh).abs().mean() + Pc.abs() * (ha * xh.abs()).mean()) + q[cols].abs() * ga + wc.abs() * uba
            cross = mph - mp * m1 - mp2 * m2
            crossa = (Pc.abs() * ha).mean() + Pc.abs().mean() * ha.mean() + (Pc * xh).abs().mean() * (ha * xh.abs()).mean()
            put(ddy, rows, cols, gb * f1 * Dc, gba * Dc)
            put(ddx, rows, cols, r * (Xh - Xh.mean() - xh * ((Xh * xh).mean() + r * cross)),
                r * (Xa + Xa.mean() + xh.abs() * ((Xa * xh.abs()).mean() + r * crossa)))
            add(par["ddw"], cols, gr * v + ub * xh)
            add(par["ddb"], cols, ub)
            par["ddw"][1][cols] += (ga * va + uba * xh.abs()).sum(0)
            par["ddb"][1][cols] += uba.sum(0)
    out = {"y": y}
    if order >= 1:
        out |= {"dx": dx, "dw": par["dw"], "db": par["db"]}
    if order >= 2:
        out |= {"ddy": ddy, "ddx": ddx, "ddw": par["ddw"], "ddb": par["ddb"]}
    out["cond"] = (cond, cond)
    return out


# half steps of fp32 on the way to one result, counted generously: statistics (a sum over up to 2^20 elements in partial sums, two rounds)
# 24, normalising and the affine map 6, an activation with its exponential and reciprocal 24, dropout's scale 2 -> 56; a gradient adds the
# derivative and two more means: 2 x 56; the second gradient adds three means and the product of two gradients: 6 x 56
ROUNDINGS = {"y": 56, "dx": 112, "dw": 112, "db": 112, "ddy": 168, "ddx": 336, "ddw": 336, "ddb": 336}


def off(name, got, ref, dtype, cond):
    """Largest |got - ref| over what the count above and one rounding to ``dtype`` allow (<= 1 is a pass); rows' conditioning included."""
    want, scale = ref[name]
    got = got.detach().double().cpu().reshape(want.shape)
    kappa = cond if want.dim() == 2 else cond.max()
    allow = torch.finfo(dtype).eps / 2 * want.abs() + ROUNDINGS[name] * 2.0 ** -24 * kappa * scale + torch.finfo(dtype).tiny
    if dtype == torch.float16:
        allow = allow + 2.0 ** -25      # half a step among fp16's subnormal numbers
    bad = (got - want).abs() / allow
    return float(torch.where(torch.isfinite(got), bad, torch.full_like(bad, math.inf)).max()) if want.numel() else 0.0
