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
Attention with its gradients, lk keys:
  scores   |ds| <= (dh + 4) u scale sum|q||k|; an exponential adds 4 u and the
           shifted argument's rounding |s - m| u: a probability is off by
           e_i = 2 max_j|ds_ij| + (8 + 4 max|s| + lk) u, relatively
  out      sum_j P|v| (e + p) + b |out|, p = 2^-8 in bf16 (P rounded for the
           product), 0 in fp32
  D        sum_d |do| err(out)_d + dh u sum|do||out|
  dS       P (err(D) + (dh + 4) u sum|do||v|) + |dS| (e + p + 4 u)
  dq, dk   scale sum err(dS) |k|, |q| (+ the sum's own u per term) + b |.|
  dv       sum_i P |do| (e + p + rows u) + b |dv|
Underflow: an exponential below 2^-126 may come out as 0, so P is off by up to
2^-126 absolutely as well, and so is every product made from it.
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


FLUSH = 2.0 ** -126


def sees(qpos, kpos, window, sinks):
    """(rows, keys): which keys a row sees."""
    q, k = qpos[:, None], kpos[None]
    return (k <= q) & ((q - k < (window or 1 << 62)) | (k < sinks))


def attention(q, k, v, see, scale, do=None, bf16=False):
    """One sequence in 64 bits: q (lq, H, d), k, v (lk, KV, d), see (lq, lk) bool.
    Returns {name: (value, bound)}; lse's bound is absolute too."""
    t = torch.bfloat16 if bf16 else torch.float32
    b, p_round = half_step(t), (2.0 ** -8 if bf16 else 0.0)
    q, k, v = q.double(), k.double(), v.double()
    unseen = ~see.any(0)
    k, v = k.masked_fill(unseen[:, None, None], 0.0), v.masked_fill(unseen[:, None, None], 0.0)
    lq, H, d = q.shape
    lk, KV = k.shape[0], k.shape[1]
    G = H // KV
    live = see.any(1)
    qh = q.transpose(0, 1).masked_fill(~live[None, :, None], 0.0)
    kh, vh = (x.transpose(0, 1).repeat_interleave(G, 0) for x in (k, v))
    s = (scale * qh @ kh.transpose(1, 2)).masked_fill(~see, -math.inf)
    sabs = (scale * qh.abs() @ kh.abs().transpose(1, 2)).masked_fill(~see, 0.0)
    lse = torch.logsumexp(s, 2) if lk else torch.full((H, lq), -math.inf, dtype=torch.float64, device=q.device)
    P = torch.exp(s - torch.where(live, lse, 0.0)[..., None])
    top = sabs.amax(2, keepdim=True) if lk else torch.zeros(H, lq, 1, dtype=torch.float64, device=q.device)
    e = (2 * (d + 4) * U * top + (8 + 4 * top + lk) * U) * live[None, :, None]
    out = P @ vh
    out_err = (P @ vh.abs()) * (e + p_round) * (1 + p_round) + b * out.abs() + TINY
    out_err = out_err + FLUSH * (see.double() @ vh.abs())
    res = {"out": (out.transpose(0, 1), out_err.transpose(0, 1)),
           "lse": (lse, e[..., 0] + 4 * U * (1 + lse.abs().nan_to_num(posinf=0.0)))}
    if do is None:
        return res
    doh = do.double().transpose(0, 1).masked_fill(~live[None, :, None], 0.0)
    dP = doh @ vh.transpose(1, 2)
    D = (doh * out).sum(2, keepdim=True)
    D_err = (doh.abs() * out_err).sum(2, keepdim=True) + d * U * (doh.abs() * out.abs()).sum(2, keepdim=True)
    dS = P * (dP - D)
    dP_err = (d + 4) * U * doh.abs() @ vh.abs().transpose(1, 2)
    dS_err = P * (D_err + dP_err) * (1 + p_round) + dS.abs() * (e + p_round + 4 * U)
    dS_err = dS_err + FLUSH * (dP.abs() + D.abs() + 1) * see
    fold = lambda x: x.unflatten(0, (KV, G)).sum(1)
    rows = lq * G

    def pair(val, err, terms, absum):
        return val.transpose(0, 1), (err + terms * U * absum + b * val.abs() + TINY).transpose(0, 1)

    res["dq"] = pair(scale * dS @ kh, scale * dS_err @ kh.abs(), lk + 4, scale * dS.abs() @ kh.abs())
    res["dk"] = pair(scale * fold(dS.transpose(1, 2) @ qh), scale * fold(dS_err.transpose(1, 2) @ qh.abs()), rows + 4,
                     scale * fold(dS.abs().transpose(1, 2) @ qh.abs()))
    res["dv"] = pair(fold(P.transpose(1, 2) @ doh),
                     fold((P * (e + p_round) + FLUSH * see).transpose(1, 2) @ doh.abs()), rows + 4,
                     fold(P.transpose(1, 2) @ doh.abs()))
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
