"""Performance cases of the attention-to-encoder, embedding and 8-bit checkpoint operators.

A decoder over option tokens next to the policy's trunk: option tokens are
looked up in a table, attend to the trunk's encoded tokens, and pass through
layers whose activations are kept for the backward pass in 8 bits.

kinds
  xattn   cross attention to an encoder's states: samples of lq query rows
          and lk key rows, padded (with a key mask or per-sample key counts)
          or packed end to end; the forward, or forward and backward.
  embed   embedding lookup with scaling; the forward, or with the table's
          gradient.
  store   an activation stored in 8 bits and restored (power-of-two scale per
          group of 32 along the row, e4m3 values).
  gelu    a GELU layer's backward from its 8-bit pre-activation.
  dw      a linear layer's weight and bias gradient from its 8-bit input.

Plain forms compute in fp32 with elementary torch operations and round once.
"""
import ctypes
import importlib
import math

import torch

own = False

GROUP = 32


def _native():
    return importlib.import_module("kaggle-ptcg-ai-battle_amd.native")


def listed():
    return [
        # acting for a few environments: options attend to the board's tokens, latency
        dict(name="xattn_act_16", kind="xattn", n=16, lq=64, lk=97, heads=4, kv=4, dh=64, prec="fp32", mask="keep",
             bwd=False),
        # the same for all environments at once, mixed precision
        dict(name="xattn_act_8192", kind="xattn", n=8192, lq=64, lk=97, heads=4, kv=4, dh=64, prec="bf16",
             mask="keep", bwd=False),
        # one new token per sample against a long cache of encoder states, shared kv heads
        dict(name="xattn_token_long", kind="xattn", n=4, lq=1, lk=50001, heads=8, kv=2, dh=128, prec="bf16",
             mask="len", bwd=False),
        # the training minibatch of the benchmark model
        dict(name="xattn_train_512", kind="xattn", n=512, lq=64, lk=97, heads=4, kv=4, dh=64, prec="fp32",
             mask="keep", bwd=True),
        # packed samples of very different lengths, mixed precision, shared kv heads
        dict(name="xattn_train_packed", kind="xattn", n=16, lq=1501, lk=4003, heads=8, kv=2, dh=128, prec="bf16",
             mask="packed", bwd=True),
        # a few tokens' rows: latency
        dict(name="embed_64", kind="embed", rows=64, vocab=2048, d=256, table="fp32", out="fp32", zipf=False, bwd=False),
        # card ids of a training minibatch, a quarter of the slots padding
        dict(name="embed_train", kind="embed", rows=49152, vocab=2048, d=256, table="fp32", out="fp32", zipf=False,
             bwd=True),
        # a large table under a skewed distribution, mixed precision
        dict(name="embed_large", kind="embed", rows=300007, vocab=100003, d=1024, table="fp32", out="bf16", zipf=True,
             bwd=True),
        # a trunk activation of a training minibatch kept in 8 bits
        dict(name="store_fp32", kind="store", rows=37391, d=256, prec="fp32"),
        # the FFN's GELU backward, mixed precision
        dict(name="gelu_bf16", kind="gelu", rows=149504, d=1024, prec="bf16"),
        # the FFN's first weight gradient of a training minibatch
        dict(name="dw_fp32", kind="dw", rows=37391, k=256, n=1024, prec="fp32"),
        # a wide layer's weight gradient, mixed precision
        dict(name="dw_bf16_wide", kind="dw", rows=65539, k=4096, n=1024, prec="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["xattn", "xattn", "xattn", "embed", "store", "gelu", "dw", "dw"])
    prec = rng.choice(["fp32", "bf16"])
    if kind == "xattn":
        form = rng.choice(["act", "token", "train", "packed"])
        kv, group = rng.choice([(4, 1), (8, 1), (2, 4), (1, 8), (2, 3)])
        c = dict(kind=kind, heads=kv * group, kv=kv, dh=rng.choice([32, 64, 64, 128, 128, 40, 96]), prec=prec)
        if form == "token":
            lk = _log(rng, 200, 60000)
            return dict(c, n=min(64, _log(rng, 1, 1 + 300000 // lk)), lq=1, lk=lk,
                        mask=rng.choice(["len", "keep", "none"]), bwd=False)
        if form == "packed":
            return dict(c, n=rng.randint(1, 12), lq=_log(rng, 1, 1200), lk=_log(rng, 16, 2500), mask="packed",
                        bwd=rng.random() < 0.7)
        n = _log(rng, 1, 1500)
        return dict(c, n=n, lq=rng.randint(1, 96), lk=rng.randint(1, 260), mask=rng.choice(["keep", "len", "none"]),
                    bwd=form == "train")
    if kind == "embed":
        return dict(kind=kind, rows=_log(rng, 1, 200000), vocab=_log(rng, 16, 60000),
                    d=rng.choice([32, 64, 128, 256, 512, 1024, 300, 77]), table=rng.choice(["fp32", "bf16"]),
                    out=rng.choice(["fp32", "bf16"]), zipf=rng.random() < 0.5, bwd=rng.random() < 0.7)
    if kind == "dw":
        return dict(kind=kind, rows=_log(rng, 40, 60000), k=rng.choice([128, 256, 512, 1024, 2048, 634, 200]),
                    n=rng.choice([64, 128, 256, 512, 768, 1024, 136]), prec=prec)
    return dict(kind=kind, rows=_log(rng, 1, 100000), d=rng.choice([128, 256, 512, 1024, 634, 200]), prec=prec)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 29)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _lengths(n, hi, step):
    """Sample lengths over [hi/4, hi], spread by a low-discrepancy sequence."""
    return [max(1, hi - int((i * step) % 1.0 * 0.75 * hi)) for i in range(n)]


def _offsets(lens):
    off = [0]
    for x in lens:
        off.append(off[-1] + x)
    return off


def _xattn_inputs(c, seed):
    g, t = _gen(seed), _type(c["prec"])
    n, lq, lk, H, KV, dh = (c[x] for x in ("n", "lq", "lk", "heads", "kv", "dh"))
    s = dict(keep=None, k_len=None, q_off=None, k_off=None)
    if c["mask"] == "packed":
        qo, ko = _offsets(_lengths(n, lq, 0.618034)), _offsets(_lengths(n, lk, 0.414214))
        q_shape, k_shape = (qo[-1], H, dh), (ko[-1], KV, dh)
        s["q_off"] = torch.tensor(qo, dtype=torch.int32, device="cuda")
        s["k_off"] = torch.tensor(ko, dtype=torch.int32, device="cuda")
    else:
        q_shape, k_shape = (n, lq, H, dh), (n, lk, KV, dh)
        live = lk - (torch.rand(n, generator=g, device="cuda") * (lk // 2 + 1)).int()
        if c["mask"] == "len":
            s["k_len"] = live
        elif c["mask"] == "keep":    # a valid prefix, holes in it
            hole = torch.rand(n, lk, generator=g, device="cuda") < 0.05
            s["keep"] = ((torch.arange(lk, device="cuda")[None] < live[:, None]) & ~hole).float()
    for name, shape in (("q", q_shape), ("k", k_shape), ("v", k_shape)):
        s[name] = _randn(g, *shape).to(t)
    if c["bwd"]:
        s["do"] = _randn(g, *q_shape).to(t)
    return s


def _embed_inputs(c, seed):
    g = _gen(seed)
    u = torch.rand(c["rows"], generator=g, device="cuda", dtype=torch.float64)
    ids = (c["vocab"] ** u - 1 if c["zipf"] else c["vocab"] * u).long().clamp(0, c["vocab"] - 1)
    pad = torch.rand(c["rows"], generator=g, device="cuda") < 0.25
    s = dict(ids=torch.where(pad, -1, ids).int(), table=_randn(g, c["vocab"], c["d"]).to(_type(c["table"])))
    if c["bwd"]:
        s["dout"] = _randn(g, c["rows"], c["d"]).to(_type(c["out"]))
    return s


def _activations(g, rows, d):
    """Rows of different magnitude with a few outlying features."""
    x = _randn(g, rows, d) * torch.exp(_randn(g, rows, 1))
    return x * torch.where(torch.rand(d, generator=g, device="cuda") < 0.02, 12.0, 1.0)


def _group_exponent(x):
    """e of each group's scale 2^e: the least with max |x| <= 448 2^e, within [-110, 119]."""
    rows, d = x.shape
    x = torch.nn.functional.pad(x, (0, -d % GROUP)).view(rows, -1, GROUP)
    m, e = torch.frexp(x.abs().amax(2))           # amax = m 2^e, m in [1/2, 1)
    e = e - 9 + (m > 0.875).int()
    return torch.where(m > 0, e, -200).clamp(-110, 119)


def _per_value(e, d):
    return torch.exp2(e.float()).repeat_interleave(GROUP, 1)[:, :d]


def _round_e4m3(y):
    """y (|y| <= 448) to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp(min=-6).float() - 3)
    return torch.round(y / step) * step


def _codes(v):
    """e4m3 codes of e4m3 values."""
    a = v.abs()
    _, e = torch.frexp(a)
    e = (e - 1).clamp(min=-6)
    frac = (a * torch.exp2(3 - e.float())).int()    # in 1/8 of 2^e: 8..15, below 8 for subnormals
    code = torch.where(frac >= 8, (e + 7) * 8 + frac - 8, frac)
    return (code + torch.where(v < 0, 128, 0)).to(torch.uint8)


def _packed(x):
    """What the forward pass left of an activation: codes and scale bytes."""
    e = _group_exponent(x)
    return _codes(_round_e4m3(x / _per_value(e, x.shape[1]))), (e + 127).to(torch.uint8)


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind == "xattn":
        s = _xattn_inputs(c, seed)
    elif kind == "embed":
        s = _embed_inputs(c, seed)
    else:
        g = _gen(seed)
        t = _type(c["prec"])
        if kind == "store":
            s = dict(x=_activations(g, c["rows"], c["d"]).to(t))
        elif kind == "gelu":
            q, sc = _packed(_randn(g, c["rows"], c["d"]) * 1.5)
            s = dict(q=q, sc=sc, dy=_randn(g, c["rows"], c["d"]).to(t))
        else:
            q, sc = _packed(_activations(g, c["rows"], c["k"]))
            s = dict(q=q, sc=sc, dy=(_randn(g, c["rows"], c["n"]) * 1e-3).to(t))
    s["case"] = c
    if own:     # the output buffers, workspace and argument lists that a training program keeps
        PLANS[kind](c, s)
    return s


# ------------------------------------------------------------------ the framework's calls
def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _bytes(n):
    return torch.zeros(max(int(n), 16), dtype=torch.uint8, device="cuda")


def _plan_xattn(c, s):
    nv = _native()
    L = nv.lib()
    H, KV, dh = c["heads"], c["kv"], c["dh"]
    a = nv.CPtcgCrossAttn(n=c["n"], lq=c["lq"], lk=c["lk"], heads=H, kv_heads=KV, dh=dh,
                          bf16=int(c["prec"] == "bf16"), scale=1 / math.sqrt(dh))
    for name, h, l in (("q", H, c["lq"]), ("k", KV, c["lk"]), ("v", KV, c["lk"]), ("o", H, c["lq"])):
        setattr(a, name, nv.CPtcgHeadLayout(sn=l * h * dh, sl=h * dh, sh=dh))
    a.q_off, a.k_off, a.k_len = _p(s["q_off"]), _p(s["k_off"]), _p(s["k_len"])
    a.keep, a.keep_sn = _p(s["keep"]), c["lk"]
    s["desc"] = a
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(c["n"], H, c["lq"], device="cuda") if c["bwd"] else None
    ref = ctypes.byref(a)
    wb = [L.ptcg_kernel_cross_attention_ws_bytes(ref, 0)]
    if c["bwd"]:
        wb.append(L.ptcg_kernel_cross_attention_ws_bytes(ref, 1))
        s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[x]) for x in "qkv")
    s["ws"] = _bytes(max(wb))
    nb = s["ws"].numel()
    q, k, v, o = (_p(s[x]) for x in ("q", "k", "v", "out"))
    s["calls"] = [(L.ptcg_kernel_cross_attention_fwd, (ref, q, k, v, o, _p(s["lse"]), _p(s["ws"]), nb))]
    s["result"] = dict(out=s["out"])
    if c["bwd"]:
        s["calls"].append((L.ptcg_kernel_cross_attention_bwd,
                           (ref, q, k, v, o, _p(s["lse"]), _p(s["do"]), _p(s["dq"]), _p(s["dk"]), _p(s["dv"]),
                            _p(s["ws"]), nb)))
        s["result"].update(dq=s["dq"], dk=s["dk"], dv=s["dv"])


def _plan_embed(c, s):
    L = _native().lib()
    rows, V, d = c["rows"], c["vocab"], c["d"]
    ob = int(c["out"] == "bf16")
    s["out"] = torch.empty(rows, d, dtype=_type(c["out"]), device="cuda")
    s["calls"] = [(L.ptcg_kernel_embedding_fwd,
                   (_p(s["ids"]), rows, _p(s["table"]), d, int(c["table"] == "bf16"), V, d, math.sqrt(d), _p(s["out"]),
                    d, ob))]
    s["result"] = dict(out=s["out"])
    if c["bwd"]:
        s["ws"] = _bytes(L.ptcg_kernel_embedding_bwd_ws_bytes(rows, V, d))
        s["dtable"] = torch.empty(V, d, device="cuda")
        s["calls"].append((L.ptcg_kernel_embedding_bwd,
                           (_p(s["ids"]), rows, _p(s["dout"]), d, ob, V, d, math.sqrt(d), _p(s["dtable"]), d,
                            _p(s["ws"]), s["ws"].numel())))
        s["result"].update(dtable=s["dtable"])


def _plan_store(c, s):
    L = _native().lib()
    rows, d, bf = c["rows"], c["d"], int(c["prec"] == "bf16")
    gs = -(-d // GROUP)
    s["q8"] = torch.empty(rows, d, dtype=torch.uint8, device="cuda")
    s["s8"] = torch.empty(rows, gs, dtype=torch.uint8, device="cuda")
    s["out"] = torch.empty_like(s["x"])
    s["calls"] = [(L.ptcg_kernel_ckpt8_pack, (_p(s["x"]), d, bf, rows, d, _p(s["q8"]), d, _p(s["s8"]), gs)),
                  (L.ptcg_kernel_ckpt8_unpack, (_p(s["q8"]), d, _p(s["s8"]), gs, rows, d, _p(s["out"]), d, bf))]
    s["result"] = dict(out=s["out"])


def _plan_gelu(c, s):
    L = _native().lib()
    rows, d, bf = c["rows"], c["d"], int(c["prec"] == "bf16")
    s["dz"], s["a"] = torch.empty_like(s["dy"]), torch.empty_like(s["dy"])
    s["calls"] = [(L.ptcg_kernel_ckpt8_gelu_bwd,
                   (_p(s["q"]), d, _p(s["sc"]), -(-d // GROUP), rows, d, _p(s["dy"]), d, _p(s["dz"]), d, _p(s["a"]),
                    d, bf))]
    s["result"] = dict(dz=s["dz"], a=s["a"])


def _plan_dw(c, s):
    L = _native().lib()
    rows, k, n, bf = c["rows"], c["k"], c["n"], int(c["prec"] == "bf16")
    s["dW"], s["db"] = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    s["ws"] = _bytes(L.ptcg_kernel_ckpt8_dw_ws_bytes(rows, k, n, bf))
    s["calls"] = [(L.ptcg_kernel_ckpt8_dw,
                   (rows, k, n, _p(s["dy"]), n, bf, _p(s["q"]), k, _p(s["sc"]), -(-k // GROUP), _p(s["dW"]),
                    _p(s["db"]), _p(s["ws"]), s["ws"].numel()))]
    s["result"] = dict(dW=s["dW"], db=s["db"])


PLANS = dict(xattn=_plan_xattn, embed=_plan_embed, store=_plan_store, gelu=_plan_gelu, dw=_plan_dw)


def _run_own(s):
    check, stream = _native().check, _stream()
    for f, args in s["calls"]:
        check(f(*args, stream))
    return s["result"]


# ------------------------------------------------------------------ plain forms
def _pad_rows(x, off, L):
    """Packed rows (total, h, dh) as (n, L, h, dh), the row index of each and whether it is one."""
    pos = torch.arange(L, device=x.device)[None]
    valid = pos < (off[1:] - off[:-1])[:, None]
    idx = (off[:-1, None] + pos).clamp(max=x.shape[0] - 1).long()
    return x[idx], idx, valid


def _unpad_rows(y, idx, valid, total):
    """(n, L, h, dh) back to packed rows; padding goes to a row behind them that is cut off."""
    out = y.new_zeros(total + 1, *y.shape[2:])
    out[torch.where(valid, idx, total)] = y
    return out[:total]


def _plain_xattn(s):
    c = s["case"]
    n, lq, lk, H, KV, dh = (c[x] for x in ("n", "lq", "lk", "heads", "kv", "dh"))
    G, t, scale = H // KV, s["q"].dtype, 1 / math.sqrt(dh)
    names = ["q", "k", "v"] + (["do"] if c["bwd"] else [])
    x = {m: s[m].float() for m in names}
    packed = c["mask"] == "packed"
    keep = torch.ones(n, lk, dtype=torch.bool, device="cuda")
    if packed:
        x["q"], qi, qv = _pad_rows(x["q"], s["q_off"], lq)
        x["k"], ki, keep = _pad_rows(x["k"], s["k_off"], lk)
        x["v"] = _pad_rows(x["v"], s["k_off"], lk)[0]
        if c["bwd"]:
            x["do"] = _pad_rows(x["do"], s["q_off"], lq)[0] * qv[..., None, None]
    elif s["keep"] is not None:
        keep = s["keep"] != 0
    elif s["k_len"] is not None:
        keep = torch.arange(lk, device="cuda")[None] < s["k_len"][:, None]
    rows = lambda y: y.view(n, lq, KV, G, dh).permute(0, 2, 3, 1, 4).reshape(n, KV, G * lq, dh)
    cols = lambda y: y.permute(0, 2, 1, 3).contiguous()
    q, k, v = rows(x["q"]), cols(x["k"]), cols(x["v"])
    live = keep[:, None, None, :]
    sc = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(~live, -math.inf)
    m = sc.amax(3, keepdim=True).clamp(min=-1e30)
    p = sc.sub_(m).exp_()
    z = p.sum(3, keepdim=True)
    p = p.div_(torch.where(z > 0, z, 1.0))
    o = torch.matmul(p, v)
    back = lambda y: y.view(n, KV, G, lq, dh).permute(0, 3, 1, 2, 4).reshape(n, lq, H, dh)
    keys = lambda y: y.permute(0, 2, 1, 3).contiguous()
    qout = (lambda y: _unpad_rows(back(y), qi, qv, s["q"].shape[0])) if packed else back
    kout = (lambda y: _unpad_rows(keys(y), ki, keep, s["k"].shape[0])) if packed else keys
    res = dict(out=qout(o).to(t))
    if c["bwd"]:
        do = rows(x["do"])
        dv = torch.matmul(p.transpose(2, 3), do)
        ds = torch.matmul(do, v.transpose(2, 3)).sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(scale)
        res.update(dq=qout(torch.matmul(ds, k)).to(t), dk=kout(torch.matmul(ds.transpose(2, 3), q)).to(t),
                   dv=kout(dv).to(t))
    return res


def _plain_embed(s):
    c = s["case"]
    ids, scale = s["ids"].long(), math.sqrt(c["d"])
    live = ids >= 0
    out = s["table"].float()[ids.clamp(min=0)] * scale * live[:, None]
    res = dict(out=out.to(_type(c["out"])))
    if c["bwd"]:
        acc = torch.zeros(c["vocab"] + 1, c["d"], device="cuda")
        acc.index_add_(0, torch.where(live, ids, c["vocab"]), s["dout"].float())
        res["dtable"] = acc[:c["vocab"]] * scale
    return res


def _values(s, d):
    """The activation that codes and scale bytes stand for."""
    code = torch.arange(256, device="cuda")
    e, m = (code >> 3) & 15, (code & 7).float()
    v = torch.where(e > 0, (8 + m) * torch.exp2(e.float() - 10), m * 2.0 ** -9)
    v = torch.where(code > 127, -v, v)
    return v[s["q"].long()] * _per_value(s["sc"].int() - 127, d)


def _plain_store(s):
    x = s["x"].float()
    w = _per_value(_group_exponent(x), x.shape[1])
    return dict(out=(_round_e4m3(x / w) * w).to(s["x"].dtype))


def _plain_gelu(s):
    z, t = _values(s, s["case"]["d"]), s["dy"].dtype
    cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    grad = cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return dict(dz=(s["dy"].float() * grad).to(t), a=(z * cdf).to(t))


def _plain_dw(s):
    dy = s["dy"].float()
    return dict(dW=torch.matmul(dy.t(), _values(s, s["case"]["k"])), db=dy.sum(0))


PLAIN = dict(xattn=_plain_xattn, embed=_plain_embed, store=_plain_store, gelu=_plain_gelu, dw=_plain_dw)


def run(state):
    if own:
        return _run_own(state)
    return PLAIN[state["case"]["kind"]](state)


# ------------------------------------------------------------------ work
def work(case):
    c, kind = case, case["kind"]
    if kind == "xattn":
        n, lq, lk, H, KV, dh = (c[x] for x in ("n", "lq", "lk", "heads", "kv", "dh"))
        e = 2 if c["prec"] == "bf16" else 4
        if c["mask"] == "packed":
            ql, kl = _lengths(n, lq, 0.618034), _lengths(n, lk, 0.414214)
            tq, tk, pairs = sum(ql), sum(kl), sum(a * b for a, b in zip(ql, kl))
        else:
            share = 1.0 if c["mask"] == "none" else (lk - lk // 4) / lk * (0.95 if c["mask"] == "keep" else 1.0)
            tq, tk, pairs = n * lq, n * lk * share, n * lq * lk * share
        qb, kb = tq * H * dh * e, tk * KV * dh * e
        by, fl = 2 * qb + 2 * kb, 4.0 * pairs * H * dh
        if c["bwd"]:    # out and the scores' statistics again, do, dq; dk and dv
            by, fl = by + 4 * qb + 4 * kb + 8.0 * tq * H, fl + 10.0 * pairs * H * dh
        return dict(bytes=float(by), flops=fl)
    if kind == "embed":
        rows, V, d = c["rows"], c["vocab"], c["d"]
        te, oe = (2 if c[x] == "bf16" else 4 for x in ("table", "out"))
        live = 0.75 * rows
        touched = V * (1 - math.exp(-live / V))
        if c["zipf"]:   # id + 1 log-uniform over the vocabulary
            touched = sum(1 - math.exp(-live * math.log((i + 2) / (i + 1)) / math.log(V)) for i in range(V))
        by = 4.0 * rows + touched * d * te + rows * d * oe
        if c["bwd"]:
            by += 4.0 * rows + live * d * oe + V * d * 4.0
        return dict(bytes=by, flops=rows * d * (2.0 if c["bwd"] else 1.0))
    rows = c["rows"]
    e = 2 if c["prec"] == "bf16" else 4
    if kind == "store":
        d = c["d"]
        return dict(bytes=rows * (2.0 * d * e + 2 * (d + -(-d // GROUP))), flops=4.0 * rows * d)
    if kind == "gelu":
        d = c["d"]
        return dict(bytes=rows * (3.0 * d * e + d + -(-d // GROUP)), flops=20.0 * rows * d)
    k, n = c["k"], c["n"]
    return dict(bytes=rows * (n * e + k + -(-k // GROUP) + 0.0) + 4.0 * n * (k + 1), flops=2.0 * rows * k * n)


# ------------------------------------------------------------------ exact
def _exact_xattn(c, seed):
    """Sample by sample in 64 bits; the gradients from the softmax's definition."""
    s = _xattn_inputs(c, seed)
    n, lq, lk, H, KV, dh = (c[x] for x in ("n", "lq", "lk", "heads", "kv", "dh"))
    packed = c["mask"] == "packed"
    if packed:
        ql, kl = _lengths(n, lq, 0.618034), _lengths(n, lk, 0.414214)
        qo, ko = _offsets(ql), _offsets(kl)
        part = lambda t, off, i: t[off[i]:off[i + 1]][None]
        groups = [(part(s["q"], qo, i), part(s["k"], ko, i), part(s["v"], ko, i),
                   part(s["do"], qo, i) if c["bwd"] else None, None) for i in range(n)]
    else:
        keep = torch.ones(n, lk, device="cuda", dtype=torch.bool)
        if s["keep"] is not None:
            keep = s["keep"] > 0
        if s["k_len"] is not None:
            keep = torch.stack([torch.arange(lk, device="cuda") < x for x in s["k_len"]])
        step = max(1, int(2e8 // (H * lq * lk)))
        groups = [(s["q"][i:i + step], s["k"][i:i + step], s["v"][i:i + step],
                   s["do"][i:i + step] if c["bwd"] else None, keep[i:i + step]) for i in range(0, n, step)]
    got = dict(out=[], dq=[], dk=[], dv=[])
    for q, k, v, do, kp in groups:
        q, k, v = (x.double().transpose(1, 2) for x in (q, k, v))
        ke, ve = (x.repeat_interleave(H // KV, 1) for x in (k, v))
        w = q @ ke.transpose(2, 3) / math.sqrt(dh)
        if kp is not None:
            w = w.masked_fill(~kp[:, None, None], -math.inf)
        w = torch.nan_to_num(torch.softmax(w, 3), nan=0.0)
        got["out"].append((w @ ve).transpose(1, 2))
        if do is None:
            continue
        do = do.double().transpose(1, 2)
        dw = do @ ve.transpose(2, 3)
        dv = (w.transpose(2, 3) @ do).unflatten(1, (KV, H // KV)).sum(2)
        dsc = w * (dw - (w * dw).sum(3, keepdim=True)) / math.sqrt(dh)
        dk = (dsc.transpose(2, 3) @ q).unflatten(1, (KV, H // KV)).sum(2)
        for name, x in (("dq", dsc @ ke), ("dk", dk), ("dv", dv)):
            got[name].append(x.transpose(1, 2))
    join = lambda x: torch.cat([y[0] for y in x] if packed else x)
    return {m: join(x) for m, x in got.items() if x}


def _exact_codes(q, sc):
    v = q.view(torch.float8_e4m3fn).double()
    rows, d = q.shape
    return torch.cat([torch.ldexp(v[:, i:i + GROUP], sc[:, i // GROUP:i // GROUP + 1].double() - 127)
                      for i in range(0, d, GROUP)], 1)


def exact(case, seed):
    c, kind = case, case["kind"]
    if kind == "xattn":
        return _exact_xattn(c, seed)
    if kind == "embed":
        s = _embed_inputs(c, seed)
        ids, f = s["ids"].long(), float(c["d"]) ** 0.5
        table = torch.cat([s["table"].double(), torch.zeros(1, c["d"], dtype=torch.float64, device="cuda")])
        res = dict(out=torch.index_select(table, 0, torch.where(ids < 0, c["vocab"], ids)) * f)
        if c["bwd"]:
            order = torch.argsort(ids, stable=True)
            run = torch.cumsum(s["dout"].double()[order], 0)
            run = torch.cat([torch.zeros(1, c["d"], dtype=torch.float64, device="cuda"), run])
            at = torch.searchsorted(ids[order].contiguous(), torch.arange(c["vocab"] + 1, device="cuda"))
            res["dtable"] = (run[at[1:]] - run[at[:-1]]) * f
        return res
    s = prepare(c, seed)
    if kind == "store":
        x = s["x"].double()
        out = torch.zeros_like(x)
        for i in range(0, c["d"], GROUP):
            y = x[:, i:i + GROUP]
            top = y.abs().amax(1, keepdim=True)
            e = torch.ceil(torch.log2((top / 448).clamp(min=1e-300))).clamp(-110, 119)
            e = torch.where(top > torch.ldexp(torch.full_like(e, 448.0), e), e + 1, e)     # log2 may be a hair off
            e = torch.where(top <= torch.ldexp(torch.full_like(e, 224.0), e), e - 1, e).clamp(-110, 119)
            v = torch.ldexp(y, -e).float().to(torch.float8_e4m3fn).double()
            out[:, i:i + GROUP] = torch.ldexp(v, e)
        return dict(out=out)
    if kind == "gelu":
        z = _exact_codes(s["q"], s["sc"])
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return dict(dz=s["dy"].double() * (cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)), a=z * cdf)
    dy = s["dy"].double()
    return dict(dW=dy.t() @ _exact_codes(s["q"], s["sc"]), db=dy.sum(0))
