"""Plain float64 statements of the 16-bit feed-forward operators and their
gradients, with elementwise bounds on what a kernel may be off by.

A kernel sums in float32 and rounds its result once: an output is off by at
most ``u |y|`` (``u`` half a step of its type, plus half the smallest
subnormal) and by the float32 sum's error, ``(n + 16) 2^-23`` times the sum of
the terms' magnitudes for ``n`` terms (twice the textbook ``n 2^-24``: matrix
cores add in groups, and an activation adds a few ulp of its own). The backward
passes of an activation start from its input kept to ``2^-16`` of itself:
that and the sum's error move a slope by at most ``max|act''|`` (below 1.2 for
every activation here) times themselves and a value by ``max|act'|`` (below
1.2), and the products' operand ``dz`` is rounded to 16 bits once.
"""

from __future__ import annotations

import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -127}
CUT = 2.0 ** -16   # of a pre-activation kept for the backward pass
BEND = 1.2   # bounds |act'| and |act''| of every activation


def act(z: torch.Tensor, name: str):
    """The activation of float64 ``z`` and its slope."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        q = 2.0 * math.sqrt(2.0 / math.pi)
        s = torch.sigmoid(q * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * q * (1 + 3 * 0.044715 * z * z)
    q = {"silu": 1.0, "quick_gelu": 1.702}[name]
    s = torch.sigmoid(q * z)
    return z * s, s + q * z * s * (1 - s)


def _round(v, dt):
    return U[dt] * v.abs() + TINY[dt]


def _sum(n, magnitude):
    return (n + 16) * 2.0 ** -23 * magnitude


def linear(x, w, b, name, res, dt, dy=None, bias_dt=None):
    """Outputs and bounds of ``linear_act`` on float64 tensors (``x [M, K]``):
    ``{name: (value, bound)}`` of y and, with ``dy``, of dx, dw and db."""
    M, K = x.shape
    N = w.shape[0]
    z = x @ w.T
    mag = x.abs() @ w.abs().T
    if b is not None:
        z, mag = z + b, mag + b.abs()
    y, slope = act(z, name)
    if res is not None:
        y = y + res
    ez = _sum(K, mag)
    out = {"y": (y, _round(y, dt) + BEND * ez + 2.0 ** -20 * (y.abs() + (0 if res is None else res.abs())))}
    if dy is not None:
        dz = dy * slope
        edz32 = 2.0 ** -20 * dz.abs()
        if name != "none":
            edz32 = edz32 + dy.abs() * BEND * (ez + CUT * z.abs())
        edz = edz32 + (_round(dz, dt) if name != "none" else 0)
        out.update(_grads(x, [w], [dz], [edz], [edz32], dt, bias_dt or dt))
        out["dres"] = (dy, torch.zeros_like(dy))
    return out


def _grads(x, ws, dzs, edzs, edz32s, dt, bias_dt):
    M, N = dzs[0].shape
    dx = sum(dz @ w for dz, w in zip(dzs, ws))
    mag = sum(dz.abs() @ w.abs() for dz, w in zip(dzs, ws))
    edx = sum(e @ w.abs() for e, w in zip(edzs, ws)) + _sum(N * len(ws), mag)
    out = {"dx": (dx, _round(dx, dt) + edx)}
    for i, (dz, e, e32) in enumerate(zip(dzs, edzs, edz32s)):
        dw = dz.T @ x
        out["dw" if i == 0 else "dwg"] = (dw, _round(dw, dt) + e.T @ x.abs() + _sum(M, dz.abs().T @ x.abs()))
        db = dz.sum(0)
        out["db" if i == 0 else "dbg"] = (db, _round(db, bias_dt) + e32.sum(0) + _sum(M, dz.abs().sum(0)))
    return out


def gated(x, wv, wg, bv, bg, name, dt, dy=None, bias_dt=None):
    """The same of ``gated_linear`` (weights ``[N, K]`` each): y, dx, dw, dwg, db, dbg."""
    K = x.shape[1]
    v, g = x @ wv.T, x @ wg.T
    mv, mg = x.abs() @ wv.abs().T, x.abs() @ wg.abs().T
    if bv is not None:
        v, mv = v + bv, mv + bv.abs()
    if bg is not None:
        g, mg = g + bg, mg + bg.abs()
    ev, eg = _sum(K, mv), _sum(K, mg)
    a, slope = act(g, name)
    y = v * a
    out = {"y": (y, _round(y, dt) + ev * a.abs() + BEND * eg * v.abs() + BEND * ev * eg + 2.0 ** -20 * y.abs())}
    if dy is not None:
        dv, dg = dy * a, dy * v * slope
        rv, rg = ev + CUT * v.abs(), eg + CUT * g.abs()
        ev32 = 2.0 ** -20 * dv.abs() + dy.abs() * BEND * rg
        eg32 = 2.0 ** -20 * dg.abs() + dy.abs() * (rv * slope.abs() + (v.abs() + rv) * BEND * rg)
        out.update(_grads(x, [wv, wg], [dv, dg], [ev32 + _round(dv, dt), eg32 + _round(dg, dt)], [ev32, eg32], dt,
                          bias_dt or dt))
    return out


def layer_norm(x, w, b, eps, dt, dy=None, w_dt=None):
    """The same of ``layer_norm``: y and, with ``dy``, dx, dw, db. The float32
    mean is off by ``(D + 16) 2^-23 mean|x|`` at most, which the deviations
    carry in full; the variance's error is relative (a sum of squares), and the
    mean's enters it squared."""
    M, D = x.shape
    mean = x.mean(1, keepdim=True)
    dev = x - mean
    var = (dev * dev).mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    emean = _sum(D, x.abs().mean(1, keepdim=True))
    rel = _sum(D, 1.0) + emean ** 2 * rstd ** 2   # of rstd: half the variance's, and slack
    xh = dev * rstd
    exh = (emean + 2.0 ** -22 * (x.abs() + mean.abs())) * rstd + xh.abs() * rel
    ww = torch.ones(D, dtype=x.dtype, device=x.device) if w is None else w
    y = xh * ww + (0 if b is None else b)
    out = {"y": (y, _round(y, dt) + exh * ww.abs() + 2.0 ** -22 * ((xh * ww).abs() + y.abs()))}
    if dy is not None:
        g = dy * ww
        s1, s2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        dx = rstd * (g - s1 - xh * s2)
        es1 = _sum(D, g.abs().mean(1, keepdim=True))
        es2 = _sum(D, (g * xh).abs().mean(1, keepdim=True)) + (g.abs() * exh).mean(1, keepdim=True)
        inner = 2.0 ** -21 * (g.abs() + s1.abs() + (xh * s2).abs()) + es1 + exh * s2.abs() + (xh.abs() + exh) * es2
        out["dx"] = (dx, _round(dx, dt) + rstd * inner + rel * dx.abs() + rstd * rel * inner)
        wt = w_dt or dt
        dw, db = (dy * xh).sum(0), dy.sum(0)
        out["dw"] = (dw, _round(dw, wt) + (dy.abs() * exh).sum(0) + _sum(M, (dy * xh).abs().sum(0)))
        out["db"] = (db, _round(db, wt) + _sum(M, dy.abs().sum(0)))
    return out
