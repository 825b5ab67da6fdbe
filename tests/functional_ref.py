"""64-bit references of ivid_amd.functional and the error bounds its tests use, derived here once.

Bounds.  u = 2^-24 is half a step of fp32.  A stored result is off by at most half a step of its type, HALF[t] relative, plus the
error of the fp32 evaluation behind it.  That one is bounded by K * u times the sum of the absolute values that enter it:

  * a sum over a tile is at most 32 additions in a thread, 64 in the tree behind it and one division, so a mean, a sum of squares or
    a channel's sum is off by at most about 100 u times the sum of absolute values (K_SUM = 128; the sums over tiles are 64-bit);
  * xhat = (x - mean) * rstd, the affine map, FiLM and the dropout scale are at most 10 operations: with the mean's and rstd's
    errors in front, |dv| <= K_SUM u ((|xhat| + mean|x| rstd) |gamma gain| + |bias gain| + |shift|) =: Ev;
  * sigmoid: the exponent is a rounded product (|v| u relative error of the exponential), exp2, add and reciprocal are good to 1 ulp
    each, so d silu <= 1.1 Ev + |v| sigma (|v| + 8) u  (|silu'| <= 1.1) and  d silu' <= Ev / 2 + (|v| + 2)(|v| + 8) sigma u  (|silu''| <= 1/2);
  * the gradient of x is a difference of three terms: its error is bounded by those of the terms, nothing cancels the bound.
"""
import math
import os
import sys

import numpy as np
import torch

U = 2.0 ** -24
K_SUM = 128
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Floor near zero: the smallest subnormal for fp16; for the others the hardware exponential and reciprocal stop at the normal range
# (exp(-v) overflows for v < -88.7, where |v| exp(v) is below 89 * 2.9e-39 < 2^-121).
TINY = {torch.float32: 2.0 ** -121, torch.bfloat16: 2.0 ** -121, torch.float16: 2.0 ** -24}


def draws(n, rng, first=0):
    """Draws first .. first + n - 1 of the dropout stream (numpy), from the published generator in oracle/."""
    from oracle.philox_oracle import philox4x32_10
    seed, sid = rng
    j = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    ctr = np.stack([j & np.uint64(0xFFFFFFFF), j >> np.uint64(32), np.full(len(j), sid & 0xFFFFFFFF, np.uint64),
                    np.full(len(j), sid >> 32, np.uint64)], -1)
    w = philox4x32_10(ctr, (seed & 0xFFFFFFFF, (seed >> 32) ^ 0x44524F50))
    h = np.stack([w & np.uint32(0xFFFF), w >> np.uint32(16)], -1).reshape(-1)
    return h[first % 8:first % 8 + n]


def threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def drop_factor(n, p, rng, first=0):
    t = threshold(p)
    f = 65536 / (65536 - t) if t < 65536 else 0.0
    return torch.from_numpy((draws(n, rng, first) >= t) * f)


def gn_act(x, groups, weight, bias, film=None, skip=None, act="silu", eps=1e-5, p=0.0, rng=None, dy=None):
    """(outputs, bounds): dicts y, stats and, with dy, dx, dskip, dweight, dbias, dfilm in float64 on the CPU, computed from the
    values as stored."""
    d = lambda t: None if t is None else t.detach().double().cpu()
    dt = x.dtype
    film_dt = None if film is None else film.dtype
    c0 = x.shape[-1]
    shape = x.shape[:-1]
    x, weight, bias, film, skip, dy = d(x), d(weight), d(bias), d(film), d(skip), d(dy)
    if skip is not None:
        x = torch.cat([x, skip], -1)
    n, c = x.shape[0], x.shape[-1]
    x = x.reshape(n, -1, c)
    hw = x.shape[1]
    grouped = lambda t: t.reshape(n, hw, groups, c // groups)
    spread = lambda t: t.expand(n, hw, groups, c // groups).reshape(n, hw, c)
    mean_g = grouped(x).mean((1, 3), keepdim=True)
    var = ((grouped(x) - mean_g) ** 2).mean((1, 3), keepdim=True)
    rstd_g = 1 / (var + eps).sqrt()
    mean, rstd = spread(mean_g), spread(rstd_g)
    absx = spread(grouped(x.abs()).mean((1, 3), keepdim=True))
    xhat = (x - mean) * rstd
    gain = 1 + film[:, None, :c] if film is not None else torch.ones(n, 1, c, dtype=torch.float64)
    shift = film[:, None, c:] if film is not None else torch.zeros(n, 1, c, dtype=torch.float64)
    u = xhat * weight + bias
    v = u * gain + shift
    ex = K_SUM * U * (xhat.abs() + absx * rstd)
    ev = ex * (weight * gain).abs() + K_SUM * U * ((bias * gain).abs() + shift.abs())
    sig = 1 / (1 + torch.exp(-v)) if act == "silu" else torch.ones_like(v)
    keep = drop_factor(n * hw * c, p, rng).reshape(n, hw, c) if p > 0 else torch.ones_like(v)
    y = v * sig * keep
    ey = (1.1 * ev + v.abs() * sig * (v.abs() + 8) * U) * keep if act == "silu" else ev * keep

    def rounded(val, err, t):
        return err * (1 + 2 * HALF[t]) + HALF[t] * val.abs() * 1.001 + TINY[t]

    out = {"y": y.reshape(*shape, c), "stats": torch.stack([mean_g.reshape(n, groups), rstd_g.reshape(n, groups)], -1)}
    bound = {"y": rounded(y, ey, dt).reshape(*shape, c),
             "stats": torch.stack([K_SUM * U * absx.reshape(n, hw, groups, -1)[:, 0, :, 0], K_SUM * U * rstd_g.reshape(n, groups)], -1)}
    if dy is None:
        return out, bound
    dy = dy.reshape(n, hw, c)
    slope = sig * (1 + v * (1 - sig)) if act == "silu" else torch.ones_like(v)
    eslope = (ev / 2 + (v.abs() + 2) * (v.abs() + 8) * sig * U) if act == "silu" else torch.zeros_like(v)
    gv = dy * keep * slope
    egv = (dy * keep).abs() * eslope + 8 * U * gv.abs()
    a, b = gv.sum(1), (gv * xhat).sum(1)
    ea = egv.sum(1) + K_SUM * U * gv.abs().sum(1)
    eb = (egv * xhat.abs() + gv.abs() * ex).sum(1) + K_SUM * U * (gv * xhat).abs().sum(1)
    gain2 = gain[:, 0]
    w = weight * gain
    g, eg = gv * w, egv * w.abs() + 4 * U * (gv * w).abs()
    m = hw * (c // groups)
    gsum = lambda t: spread(t.reshape(n, 1, groups, c // groups).sum(3, keepdim=True)) / m
    m1, m2 = gsum(a * w[:, 0]), gsum(b * w[:, 0])
    em1, em2 = gsum(ea * w[:, 0].abs()), gsum(eb * w[:, 0].abs())
    dx = rstd * (g - m1 - xhat * m2)
    edx = rstd * (eg + em1 + xhat.abs() * em2 + ex * m2.abs()) + K_SUM * U * rstd * (g.abs() + m1.abs() + (xhat * m2).abs())
    ddx = rounded(dx, edx, dt)
    out["dx"], bound["dx"] = dx[..., :c0].reshape(*shape, c0), ddx[..., :c0].reshape(*shape, c0)
    if skip is not None:
        out["dskip"], bound["dskip"] = dx[..., c0:].reshape(*shape, c - c0), ddx[..., c0:].reshape(*shape, c - c0)
    out["dweight"], out["dbias"] = (gain2 * b).sum(0), (gain2 * a).sum(0)
    bound["dweight"] = (gain2.abs() * eb).sum(0) + K_SUM * U * (gain2 * b).abs().sum(0) + TINY[torch.float32]
    bound["dbias"] = (gain2.abs() * ea).sum(0) + K_SUM * U * (gain2 * a).abs().sum(0) + TINY[torch.float32]
    if film is not None:
        ds, dt_ = weight * b + bias * a, a
        out["dfilm"] = torch.cat([ds, dt_], 1)
        eds = weight.abs() * eb + bias.abs() * ea + 4 * U * ((weight * b).abs() + (bias * a).abs())
        bound["dfilm"] = rounded(out["dfilm"], torch.cat([eds, ea], 1), film_dt)
    return out, bound


def check(got, want, bound, what=""):
    """Every entry of `want` within its bound; returns the worst ratio."""
    worst = 0.0
    for k, ref in want.items():
        if got.get(k) is None:
            raise AssertionError(f"{what}: {k} is missing")
        g = got[k].detach().double().cpu()
        assert g.shape == ref.shape, (what, k, g.shape, ref.shape)
        assert torch.isfinite(g).all(), (what, k, "not finite")
        off = (g - ref).abs()
        r = torch.where(off == 0, 0.0, off / bound[k]).max().item() if ref.numel() else 0.0      # (0 / 0 where a bound is 0)
        assert r <= 1.0, f"{what}: {k} is {r:.3f} times its bound off"
        worst = max(worst, r)
    return worst
