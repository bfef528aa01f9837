"""64-bit norms, rotations and causal attention, and how far a kernel may be off.

u is the unit roundoff of fp32 (2^-24), b half a step of the stored type.
Norm and rotation, dh elements a head:
  r = 1 / sqrt(mean x^2 + eps)   off by (dh + 8) u relatively (a sum of dh
           squares in any order, a mean, an addition, a root, a reciprocal)
  cos, sin off by 6 u mag: the reduced angle (at most pi / 4) rounded once, a
           polynomial of six steps, the factor
  y        turned from n = x r w: ((dh + 8) + 3 + 6 + 3) u mag (|n_a| + |n_b|) + b |y|
  dn       turned back from dy:   9 u mag (|dy_a| + |dy_b|) =: e
  dx       r (dn w - x m), m = r^2 mean(dn w x): with f = (dh + 12) u,
           r (e |w| + f |dn w|) + r |x| r^2 (mean((e + f |dn|) |w x|) + 2 f mean|dn w x|) + b |dx|
  dw       sum |x r| (e + f |dn|) + terms u sum |dn x r|
"""
import math

import torch

U = 2.0 ** -24
TINY = 1e-37


def half_step(t):
    return torch.finfo(t).eps / 2


def frequencies(rot, base=10000.0, scaling=0, factor=8.0, length=4096.0, fast=32.0, slow=1.0):
    b = base * factor ** (rot / (rot - 2)) if scaling == 2 and rot > 2 else base
    f = [b ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == 1:
        f = [x / factor for x in f]
    if scaling == 3:
        keep = [min(1.0, max(0.0, (length * x / (2 * math.pi) - slow) / (fast - slow))) for x in f]
        f = [x * k + x / factor * (1 - k) for x, k in zip(f, keep)]
    return f, 0.1 * math.log(factor) + 1 if scaling == 3 else 1.0


def _pairs(rot, inter):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)


def turn(x, pos, freq, mag, inter, back=False):
    """x (rows, heads, dh) in 64 bits, turned; and mag (|x_a| + |x_b|) per element (|x| where nothing turns)."""
    rot = 2 * len(freq)
    y, span = x.clone(), x.abs()
    if rot == 0:
        return y, span
    ia, ib = _pairs(rot, inter)
    ang = pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = mag * torch.cos(ang), mag * torch.sin(ang) * (-1 if back else 1)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    both = abs(mag) * (a.abs() + b.abs())
    span[..., ia], span[..., ib] = both, both
    return y, span


def norm_rope(x, w, eps, pos, freq, mag, inter, t, dy=None):
    """x (rows, heads, dh): {name: (value, bound)} of y, and of dx, dw where dy is given."""
    b, dh = half_step(t), x.shape[-1]
    x = x.double()
    r = torch.ones_like(x[..., :1]) if w is None else (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    w64 = torch.ones(dh, dtype=torch.float64, device=x.device) if w is None else w.double()
    y, span = turn(x * r * w64, pos, freq, mag, inter)
    res = {"y": (y, (dh + 20) * U * span + b * y.abs() + TINY)}
    if dy is None:
        return res
    dn, dspan = turn(dy.double(), pos, freq, mag, inter, back=True)
    e, f = 9 * U * dspan, (dh + 12) * U
    if w is None:
        res["dx"] = (dn, e + b * dn.abs() + TINY)
        return res
    g, gerr = dn * w64, (e + f * dn.abs()) * w64.abs()
    m = r * r * (g * x).mean(-1, keepdim=True)
    merr = r * r * ((gerr * x.abs()).mean(-1, keepdim=True) + 2 * f * (g * x).abs().mean(-1, keepdim=True))
    dx = r * (g - x * m)
    res["dx"] = (dx, r * (gerr + f * g.abs() + x.abs() * (merr + f * m.abs())) + b * dx.abs() + TINY)
    terms = x.shape[0] * x.shape[1]
    dw = (dn * x * r).sum((0, 1))
    res["dw"] = (dw, (((e + f * dn.abs()) * (x * r).abs()).sum((0, 1)) + terms * U * (dn * x * r).abs().sum((0, 1)))
                 + U * dw.abs() + TINY)
    return res


def within(name, got, want, err):
    """got is within err of want element by element (infinities and NaN exact)."""
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.nan_to_num(got[~fin], nan=7.0), torch.nan_to_num(want[~fin], nan=7.0)), \
        f"{name}: infinities differ"
    assert torch.isfinite(got[fin]).all(), f"{name}: not finite"
    over = (got - want).abs()[fin] / err[fin]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound"
    return worst
