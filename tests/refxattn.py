"""64-bit cross attention with its gradients, and how far a kernel may be off.

Bounds follow the arithmetic, element by element.  u is the unit roundoff of
fp32 (2^-24), b half a step of the stored type (bf16 2^-8, fp32 2^-24).
  scores   |ds| <= (dh + 4) u scale sum|q||k|; an exponential adds 4 u and the
           shifted argument's rounding |s - m| u: a probability is off by
           e_i = 2 max_j|ds_ij| + (8 + 4 max|s| + lk) u, relatively.
  out      sum_j P|v| (e + p) + b |out|, p = 2^-8 in bf16 (P rounded for the
           product), 0 in fp32.
  D        sum_d |do| err(out)_d + dh u sum|do||out|
  dS       P (err(D) + (dh + 4) u sum|do||v|) + |dS| (e + p + 4 u)
  dq, dk   scale sum err(dS) |k|, |q| (+ the sum's own u per term) + b |.|
  dv       sum_i P |do| (e + p + rows u) + b |dv|
Underflow: an exponential below 2^-126 may come out as 0 (v_exp_f32 and the
bf16 products flush subnormals), so P is off by up to t = 2^-126 absolutely as
well, and so is every product made from it: t enters P's error wherever P does
(t |v|, t (|dP| + |D| + 1), t |do|), besides 1e-37 for a stored result itself.
"""
import math

import torch

U = 2.0 ** -24
TINY = 2.0 ** -126


def half_step(t):
    return torch.finfo(t).eps / 2


def reference(q, k, v, keep, scale, do=None, bf16=False):
    """One sample in 64 bits: q (lq, H, d), k, v (lk, KV, d), keep (lk) bool.
    Returns {name: (value, bound)}; lse's bound is absolute too."""
    t = torch.bfloat16 if bf16 else torch.float32
    b, p_round = half_step(t), (2.0 ** -8 if bf16 else 0.0)
    q, k, v = q.double(), k.double(), v.double()
    lq, H, d = q.shape
    lk, KV = k.shape[0], k.shape[1]
    k, v = k.masked_fill(~keep[:, None, None], 0.0), v.masked_fill(~keep[:, None, None], 0.0)
    G = H // KV
    qh = q.transpose(0, 1)
    kh, vh = (x.transpose(0, 1).repeat_interleave(G, 0) for x in (k, v))
    s = scale * qh @ kh.transpose(1, 2)
    sabs = scale * qh.abs() @ kh.abs().transpose(1, 2)
    s = s.masked_fill(~keep, -math.inf)
    empty = not bool(keep.any())
    if empty:
        P = torch.zeros_like(s)
        lse = torch.full((H, lq), -math.inf, dtype=torch.float64, device=q.device)
        e = torch.zeros(H, lq, 1, dtype=torch.float64, device=q.device)
    else:
        lse = torch.logsumexp(s, 2)
        P = torch.exp(s - lse[..., None])
        top = sabs.masked_fill(~keep, 0.0).amax(2, keepdim=True)
        e = 2 * (d + 4) * U * top + (8 + 4 * top + lk) * U
    out = P @ vh
    out_err = (P @ vh.abs()) * (e + p_round) * (1 + p_round) + b * out.abs() + 1e-37
    out_err = out_err + TINY * vh.abs().sum(1, keepdim=True)
    res = {"out": (out.transpose(0, 1), out_err.transpose(0, 1)),
           "lse": (lse, e[..., 0] + 4 * U * (1 + lse.abs().nan_to_num(posinf=0.0)))}
    if do is None:
        return res
    doh = do.double().transpose(0, 1)
    dP = doh @ vh.transpose(1, 2)
    D = (doh * out).sum(2, keepdim=True)
    D_err = (doh.abs() * out_err).sum(2, keepdim=True) + d * U * (doh.abs() * out.abs()).sum(2, keepdim=True)
    dS = P * (dP - D)
    dP_err = (d + 4) * U * doh.abs() @ vh.abs().transpose(1, 2)
    dS_err = P * (D_err + dP_err) * (1 + p_round) + dS.abs() * (e + p_round + 4 * U)
    dS_err = dS_err + TINY * (dP.abs() + D.abs() + 1)
    fold = lambda x: x.unflatten(0, (KV, G)).sum(1)
    rows = lq * G

    def pair(val, err, terms, absum):
        return val.transpose(0, 1), (err + terms * U * absum + b * val.abs() + 1e-37).transpose(0, 1)

    res["dq"] = pair(scale * dS @ kh, scale * dS_err @ kh.abs(), lk + 4, scale * dS.abs() @ kh.abs())
    res["dk"] = pair(scale * fold(dS.transpose(1, 2) @ qh), scale * fold(dS_err.transpose(1, 2) @ qh.abs()), rows + 4,
                     scale * fold(dS.abs().transpose(1, 2) @ qh.abs()))
    res["dv"] = pair(fold(P.transpose(1, 2) @ doh), fold((P * (e + p_round) + TINY).transpose(1, 2) @ doh.abs()), rows + 4,
                     fold(P.transpose(1, 2) @ doh.abs()))
    return res


def within(name, got, want, err):
    """got is within err of want element by element (infinities and zeros exact)."""
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin]), f"{name}: infinities differ"
    assert torch.isfinite(got[fin]).all(), f"{name}: not finite"
    over = (got - want).abs()[fin] / err[fin]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound"
    return worst
