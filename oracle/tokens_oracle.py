"""Plain 64-bit forms of the token operators (layer norm, linear with epilogue, gated feed-forward block), their gradients, and how far a correct kernel may be from them.

The bounds count roundings.  u = 2^-24 is half a step of f32, h = finfo(T).eps / 2 half a step of the operand type.  A sum of n terms in f32, in any order with at most `depth`
additions on a term's way, is off by at most depth * u * sum |terms| (a product of two bf16 or f32 values that an MFMA adds contributes one more u).  An activation's derivative is at most
1.13 (gelu, gelu_tanh, silu), its second derivative at most 1.13, and its evaluation with the hardware's exp2 / reciprocal is off by at most 2^-20 (1 + |z|)."""
import math

import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def act(name, z):
    """(f(z), f'(z)) in 64 bits"""
    one = torch.ones_like(z)
    if name in (None, "none"):
        return z, one
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "gelu":
        c = torch.special.ndtr(z)
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        return z / 2 * (1 + t), (1 + t) / 2 + z / 2 * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return (s, s * (1 - s)) if name == "sigmoid" else (z * s, s * (1 + z * (1 - s)))


def _d(t):
    return None if t is None else t.detach().double()


def layer_norm(x, w, b, eps, dy=None):
    """dict of (value, bound): y, and with dy: dx, dw, db.  x (M, D) in its own type."""
    h = half(x.dtype)
    x, w, b, dy = _d(x), _d(w), _d(b), _d(dy)
    M, D = x.shape
    n = D / 64 + 32                              # additions on a term's way: a row is summed by at least 64 lanes, then across them
    g = torch.ones(D, dtype=x.dtype, device=x.device) if w is None else w
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = d * rstd
    dmean = n * U * x.abs().mean(1, keepdim=True) + U * mean.abs()
    rel = 0.5 * ((n + 8) * U * var + dmean * dmean + 4 * U * d.abs().mean(1, keepdim=True) * x.abs().amax(1, keepdim=True)) * rstd * rstd + 4 * U          # of rstd
    dxh = (dmean + U * x.abs()) * rstd + xh.abs() * (rel + 2 * U)
    y = xh * g + (0 if b is None else b)
    out = {"y": (y, g.abs() * dxh + 4 * U * (xh * g).abs() + 2 * U * y.abs() + h * y.abs())}
    if dy is not None:
        t = dy * g
        m1, m2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
        dm1 = n * U * t.abs().mean(1, keepdim=True)
        dm2 = n * U * (t * xh).abs().mean(1, keepdim=True) + (t.abs() * dxh).mean(1, keepdim=True)
        dx = rstd * (t - m1 - xh * m2)
        edx = rstd * (dm1 + xh.abs() * dm2 + m2.abs() * dxh + 6 * U * (t.abs() + m1.abs() + (xh * m2).abs())) + dx.abs() * rel + h * dx.abs()
        n2 = M / 512 + 256                       # additions on a row's way into a column sum
        out["dx"] = (dx, edx)
        out["dw"] = ((dy * xh).sum(0), (dy.abs() * dxh).sum(0) + n2 * U * (dy * xh).abs().sum(0))
        out["db"] = (dy.sum(0), n2 * U * dy.abs().sum(0))
    return out


def _product(a, b, bias):
    """(a b^T + bias, its bound in f32)"""
    z, s = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        z, s = z + bias, s + bias.abs()
    return z, (a.shape[1] + 4) * U * s


def _activated(name, z, ez):
    """f, bound of f, f', bound of f'"""
    f, fp = act(name, z)
    if name in (None, "none"):
        return f, ez, fp, torch.zeros_like(z)
    e = 2.0 ** -20 * (1 + z.abs())
    efp = 1.13 * ez + e
    if name == "relu":
        return f, ez, fp, (z.abs() <= ez).to(z.dtype)          # on the border either side is right
    return f, 1.13 * ez + e * 0.25, fp, efp


def _back(dz, edz, h, w, x, rounded):
    """(dx, dw, db) with their bounds from dz and its bound before the rounding to the operand type"""
    e = edz + h * (dz.abs() + edz) if rounded else edz
    a = dz.abs() + e
    N, M = dz.shape[1], dz.shape[0]
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    return ((dx, e @ w.abs() + (N + 4) * U * (a @ w.abs()) + h * dx.abs()), (dw, e.t() @ x.abs() + (M + 4) * U * (a.t() @ x.abs()) + h * dw.abs()),
            (db, edz.sum(0) + (M / 512 + 256) * U * (dz.abs() + edz).sum(0)))


def linear(x, w, b, name, res, dy=None):
    h = half(x.dtype)
    x, w, b, res, dy = _d(x), _d(w), _d(b), _d(res), _d(dy)
    z, ez = _product(x, w, b)
    f, ef, fp, efp = _activated(name, z, ez)
    y = f if res is None else f + res
    out = {"y": (y, (ef + U * y.abs()) * (1 + h) + h * y.abs())}
    if dy is not None:
        rounded = name not in (None, "none")
        dz = dy * fp
        out["dx"], out["dw"], out["db"] = _back(dz, dy.abs() * efp + 2 * U * dz.abs() * rounded, h, w, x, rounded)
        out["dres"] = (dy, torch.zeros_like(dy))
    return out


def gated(x, wg, wu, bg, bu, name, dy=None):
    h = half(x.dtype)
    x, wg, wu, bg, bu, dy = _d(x), _d(wg), _d(wu), _d(bg), _d(bu), _d(dy)
    (g, eg), (u, eu) = _product(x, wg, bg), _product(x, wu, bu)
    f, ef, fp, efp = _activated(name, g, eg)
    y = f * u
    out = {"y": (y, (ef * u.abs() + eu * f.abs() + ef * eu + U * y.abs()) * (1 + h) + h * y.abs())}
    if dy is not None:
        dg, du = dy * u * fp, dy * f
        edg = dy.abs() * (u.abs() * efp + eu * fp.abs() + eu * efp) + 3 * U * dg.abs()
        edu = dy.abs() * ef + 2 * U * du.abs()
        (dxg, exg), out["dwg"], out["dbg"] = _back(dg, edg, h, wg, x, True)
        (dxu, exu), out["dwu"], out["dbu"] = _back(du, edu, h, wu, x, True)
        # one sum over 2 F terms instead of two over F, rounded once: twice the longer bounds cover it
        out["dx"] = (dxg + dxu, 2 * (exg + exu))
    return out


def check(got, want, what):
    """`got` within want's bound, element by element"""
    value, bound = want
    g = got.detach().double()
    assert g.shape == value.shape, f"{what}: shape {tuple(g.shape)}, expected {tuple(value.shape)}"
    off = (g - value).abs()
    bad = ~(off <= bound + 1e-300)
    if bad.any():
        i = tuple(int(v) for v in (bad.nonzero()[0]))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values outside their bound; first at {i}: {float(g[i])} against {float(value[i])} +- {float(bound[i])}")
