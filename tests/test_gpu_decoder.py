"""The decoder's operators as a program runs them: a training step of a windowed
self-attention layer (norms and rotation, attention, both backwards) against
64-bit autograd, and acting over the paged cache, prompt by chunks and then token
by token, against the same layer over the whole sequence."""
import ctypes
import math

import pytest
import torch

from ptcg_amd import native
from refseq import frequencies, sees

pytestmark = pytest.mark.gpu

LAY = native.CPtcgHeadLayout


class Layer:
    """q, k norms, rotation and causal attention of rows qkv (T, H + 2 KV, dh), sequences packed."""

    def __init__(self, lens, H, KV, dh, rot, inter, bf16, window, sinks):
        self.t = torch.bfloat16 if bf16 else torch.float32
        g = torch.Generator(device="cuda").manual_seed(5)
        self.lens, self.H, self.KV, self.dh, self.rot, self.inter = lens, H, KV, dh, rot, inter
        self.window, self.sinks, self.bf16 = window, sinks, int(bf16)
        self.first = [sum(lens[:i]) for i in range(len(lens) + 1)]
        T = self.first[-1]
        self.T = T
        self.qkv = torch.randn(T, H + 2 * KV, dh, generator=g, device="cuda").to(self.t)
        self.wq, self.wk = (1 + 0.2 * torch.randn(dh, generator=g, device="cuda") for _ in range(2))
        self.do = torch.randn(T, H, dh, generator=g, device="cuda").to(self.t)
        self.pos = torch.cat([torch.arange(m) for m in lens]).int().cuda()
        self.off = torch.tensor(self.first, dtype=torch.int32, device="cuda")
        f, mag = (ctypes.c_double * (rot // 2))(), ctypes.c_float()
        native.check(native.lib().ptcg_rope_frequencies(rot, 10000.0, 3, 8.0, 256.0, 32.0, 1.0, f, ctypes.byref(mag)))
        self.mag = mag.value
        self.freq = torch.tensor(list(f), dtype=torch.float64, device="cuda")
        self.scale = 1 / math.sqrt(dh)

    def rope(self, pos):
        return native.CPtcgRope(rot=self.rot, interleaved=int(self.inter), mag=self.mag, freq=self.freq.data_ptr(),
                                pos=pos)

    def lay(self, h, l):
        return LAY(sn=l * h * self.dh, sl=h * self.dh, sh=self.dh)

    def ptrs(self, x):
        e = x.element_size() * self.dh
        return x.data_ptr(), x.data_ptr() + self.H * e, x.data_ptr() + (self.H + self.KV) * e

    def train(self, stream=None):
        """One step's forward and backward: out, and the gradients of qkv and of the norms' weights."""
        L, T, H, KV, dh = native.lib(), self.T, self.H, self.KV, self.dh
        w = self.lay(H + 2 * KV, T)
        new = lambda *s: torch.empty(*s, dtype=self.t, device="cuda")
        q, k, v = self.ptrs(self.qkv)
        qo, ko, out, dqo, dko = new(T, H, dh), new(T, KV, dh), new(T, H, dh), new(T, H, dh), new(T, KV, dh)
        lse, dqkv = torch.empty(len(self.lens), H, max(self.lens), device="cuda"), new(T, H + 2 * KV, dh)
        dw = torch.empty(2, dh, device="cuda")
        r = native.CPtcgQkRope(n=1, l=T, heads=H, kv_heads=KV, dh=dh, bf16=self.bf16, eps=1e-6, q=w, k=w,
                               qo=self.lay(H, T), ko=self.lay(KV, T), wq=self.wq.data_ptr(), wk=self.wk.data_ptr(),
                               rope=self.rope(self.pos.data_ptr()))
        # v and its gradient lie in the packed matrices
        a = native.CPtcgWindowAttn(n=len(self.lens), l=max(self.lens), heads=H, kv_heads=KV, dh=dh, bf16=self.bf16,
                                   scale=self.scale, window=self.window, sinks=self.sinks, q=self.lay(H, T),
                                   k=self.lay(KV, T), v=w, o=self.lay(H, T), off=self.off.data_ptr())
        rr, ra = ctypes.byref(r), ctypes.byref(a)
        nb = max(L.ptcg_kernel_qk_norm_rope_bwd_ws_bytes(rr), *[L.ptcg_kernel_window_attention_ws_bytes(ra, x)
                                                               for x in (0, 1)])
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        p = lambda x: x.data_ptr()
        dq, dk, dv = self.ptrs(dqkv)

        def step(stream):
            for rc in (
                    L.ptcg_kernel_qk_norm_rope_fwd(rr, q, k, p(qo), p(ko), stream),
                    L.ptcg_kernel_window_attention_fwd(ra, p(qo), p(ko), v, p(out), p(lse), p(ws), nb, stream),
                    L.ptcg_kernel_window_attention_bwd(ra, p(qo), p(ko), v, p(out), p(lse), p(self.do), p(dqo), p(dko), dv,
                                                       p(ws), nb, stream),
                    L.ptcg_kernel_qk_norm_rope_bwd(rr, q, k, p(dqo), p(dko), dq, dk, p(dw[0]), p(dw[1]), p(ws), nb, stream)):
                native.check(rc)

        self.hold = (r, a, qo, ko, dqo, dko, lse, ws)
        return step, dict(out=out, dqkv=dqkv, dw=dw)

    def exact(self):
        """The same in 64 bits, gradients by autograd."""
        H, KV, dh = self.H, self.KV, self.dh
        x = self.qkv.double().requires_grad_()
        ws = [w.double().requires_grad_() for w in (self.wq, self.wk)]
        freq, mag = frequencies(self.rot, scaling=3, length=256.0)
        ang = self.pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
        c, s = mag * torch.cos(ang), mag * torch.sin(ang)
        h = self.rot // 2

        def turned(y, w):
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
            a, b = (y[..., 0:self.rot:2], y[..., 1:self.rot:2]) if self.inter else (y[..., :h], y[..., h:self.rot])
            a, b = a * c - b * s, a * s + b * c
            z = torch.stack((a, b), -1).flatten(-2) if self.inter else torch.cat((a, b), -1)
            return torch.cat((z, y[..., self.rot:]), -1)

        q, k, v = turned(x[:, :H], ws[0]), turned(x[:, H:H + KV], ws[1]), x[:, H + KV:]
        outs = []
        for i, m in enumerate(self.lens):
            r = slice(self.first[i], self.first[i + 1])
            at = torch.arange(m, device="cuda")
            ke, ve = (y[r].repeat_interleave(H // KV, 1).transpose(0, 1) for y in (k, v))
            sc = (q[r].transpose(0, 1) @ ke.transpose(1, 2) * self.scale).masked_fill(
                ~sees(at, at, self.window, self.sinks), -math.inf)
            outs.append((torch.softmax(sc, 2) @ ve).transpose(0, 1))
        out = torch.cat(outs)
        g = torch.autograd.grad(out, [x] + ws, self.do.double())
        return dict(out=out.detach(), dqkv=g[0], dw=torch.stack(g[1:]))


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm())


# Relative L2 over whole tensors.  fp32: the longest sums have under 1 500 terms; with random signs their errors stay
# below sqrt(1500) u = 2.3e-6, four operators in a row below 1e-5.  bf16: q and k after the norm, P, dS, out and every
# gradient between two operators are each rounded by up to 2^-8 (uniformly, so by 2^-8 / sqrt 3 in L2); at most seven
# such roundings are behind any output, each passed on with a factor of about one: sqrt(7 / 3) 2^-8 = 6e-3, held to twice.
TOL = {torch.float32: 1e-5, torch.bfloat16: 1.2e-2}

SHAPES = [
    dict(lens=[97, 40, 200, 1], H=4, KV=4, dh=64, rot=64, inter=False, bf16=False, window=32, sinks=1),
    dict(lens=[300, 129, 700], H=8, KV=2, dh=128, rot=64, inter=True, bf16=True, window=100, sinks=4),
    dict(lens=[300, 129], H=4, KV=2, dh=64, rot=32, inter=False, bf16=True, window=0, sinks=0),
]


@pytest.mark.parametrize("kw", SHAPES, ids=str)
def test_a_training_step(cuda, kw):
    layer = Layer(**kw)
    step, got = layer.train()
    step(None)
    torch.cuda.synchronize()
    want = layer.exact()
    for name in want:
        assert _rel(got[name], want[name]) < TOL[layer.t], name


def test_a_training_step_captured_while_an_eager_graph_lives(cuda):
    layer = Layer(**SHAPES[1])
    step, got = layer.train()
    leaf = torch.ones(4, device="cuda", requires_grad=True)
    eager = (leaf * 2).sum()          # an autograd graph that outlives the capture
    step(None)
    torch.cuda.synchronize()
    first = {m: x.clone() for m, x in got.items()}
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        step(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for x in got.values():
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        for m, x in got.items():
            assert torch.equal(x, first[m]), m
    eager.backward()
    assert torch.equal(leaf.grad, torch.full_like(leaf, 2.0))


@pytest.mark.parametrize("kw", SHAPES, ids=str)
def test_acting_token_by_token_equals_the_whole_sequence(cuda, kw):
    """Each sequence's first half goes into the cache in two chunks, the rest token by token, all sequences at once."""
    layer = Layer(**kw)
    L, H, KV, dh, lens = native.lib(), layer.H, layer.KV, layer.dh, layer.lens
    n, page = len(lens), 16
    per = -(-max(lens) // page)
    pages = n * per
    kp, vp = (torch.full((pages, page, KV, dh), float("nan"), dtype=layer.t, device="cuda") for _ in range(2))
    table = torch.randperm(pages, device="cuda").int().view(n, per)
    lay = LAY(sn=page * KV * dh, sl=KV * dh, sh=dh)
    cache = native.CPtcgPages(pages=pages, page=page, per_seq=per, k=lay, v=lay, kp=kp.data_ptr(), vp=vp.data_ptr(),
                              table=table.data_ptr(), table_sn=per)
    out = torch.empty(layer.T, H, dh, dtype=layer.t, device="cuda")

    def pieces():
        half = [(m + 1) // 2 for m in lens]
        quarter = [(m + 1) // 2 for m in half]
        yield [0] * n, quarter
        yield quarter, half
        for j in range(max(m - h for m, h in zip(lens, half))):
            yield [min(h + j, m) for h, m in zip(half, lens)], [min(h + j + 1, m) for h, m in zip(half, lens)]

    for lo, hi in pieces():
        new = [b - a for a, b in zip(lo, hi)]
        rows = torch.cat([torch.arange(layer.first[i] + lo[i], layer.first[i] + hi[i]) for i in range(n)]).cuda()
        x = layer.qkv[rows].contiguous()
        q_off = torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda")
        length = torch.tensor(hi, dtype=torch.int32, device="cuda")
        l, T = max(new), len(rows)
        w = layer.lay(H + 2 * KV, l)
        qo, o = (torch.empty(T, H, dh, dtype=layer.t, device="cuda") for _ in range(2))
        ap = native.CPtcgPagedAppend(n=n, lq=l, rows=T, heads=H, kv_heads=KV, dh=dh, bf16=layer.bf16, eps=1e-6, q=w, k=w,
                                     v=w, qo=layer.lay(H, l), q_off=q_off.data_ptr(), len=length.data_ptr(),
                                     wq=layer.wq.data_ptr(), wk=layer.wk.data_ptr(), rope=layer.rope(None), cache=cache)
        at = native.CPtcgPagedAttn(n=n, lq=l, rows=T, heads=H, kv_heads=KV, dh=dh, bf16=layer.bf16, scale=layer.scale,
                                   window=layer.window, sinks=layer.sinks, q=layer.lay(H, l), o=layer.lay(H, l),
                                   q_off=q_off.data_ptr(), len=length.data_ptr(), cache=cache)
        nb = L.ptcg_kernel_paged_attention_ws_bytes(ctypes.byref(at))
        ws = torch.empty(max(nb, 16), dtype=torch.uint8, device="cuda")
        native.check(L.ptcg_kernel_paged_append(ctypes.byref(ap), *layer.ptrs(x), qo.data_ptr(), None))
        native.check(L.ptcg_kernel_paged_attention(ctypes.byref(at), qo.data_ptr(), o.data_ptr(), None, ws.data_ptr(),
                                                   ws.numel(), None))
        out[rows] = o
    torch.cuda.synchronize()
    assert _rel(out, layer.exact()["out"]) < TOL[layer.t]
    step, got = layer.train()
    step(None)
    torch.cuda.synchronize()
    assert _rel(out, got["out"].double()) < TOL[layer.t]
