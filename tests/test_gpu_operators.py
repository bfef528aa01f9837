"""Embedding, cross attention and 8-bit checkpoints as they are used together,
and calls of theirs that share a device: streams, graphs, workspaces, tensors
past 2^31 elements."""
import ctypes
import math

import pytest
import torch

from ptcg_amd import native
from refxattn import reference, within
from test_gpu_ckpt8 import test_weight_gradient as check_weight_gradient, values64
from test_gpu_cross_attention import GUARD, Op

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Decoder:
    """Query tokens attend to a padded batch of encoder tokens; a GELU layer and a
    linear head follow, the layer's input and pre-activation kept in 8 bits:
      xe = s_e Te[ids_e], xq = s_q Tq[ids_q],  k, v = xe Wk^T, xe Wv^T
      o = attend(xq, k, v),  z = o W1^T + b1,  y = gelu(z) W2^T
    and, from dy, the gradients of every weight and of both tables."""

    def __init__(self, n=5, lq=7, lk=23, H=4, KV=2, dh=16, f=72, vocab=50):
        g = torch.Generator(device="cuda").manual_seed(11)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
        ids = lambda *s: torch.randint(0, vocab, s, generator=g, device="cuda", dtype=torch.int32)
        self.n, self.lq, self.lk, self.H, self.KV, self.dh, self.f, self.vocab = n, lq, lk, H, KV, dh, f, vocab
        self.d, self.dk_ = H * dh, KV * dh
        d, e, R, S = self.d, self.dk_, n * lq, n * lk
        self.lens = [lk, 0, 1, 9, lk - 2]            # encoder tokens of each sample, padding behind them
        self.k_len = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.ids_e, self.ids_q = ids(n, lk), ids(n, lq)
        self.ids_e[torch.arange(lk, device="cuda") >= self.k_len[:, None]] = -1
        self.s_e, self.s_q = 1.5, 0.5
        self.p = {"Te": rnd(vocab, d), "Tq": rnd(vocab, d), "Wk": rnd(e, d) / math.sqrt(d), "Wv": rnd(e, d) / math.sqrt(d),
                  "W1": rnd(f, d) / math.sqrt(d), "b1": rnd(f), "W2": rnd(d, f) / math.sqrt(f)}
        self.dy = rnd(R, d)
        z = lambda *s: torch.full(s, GUARD, device="cuda")
        u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")
        self.t = {"xe": z(S, d), "xq": z(R, d), "k": z(S, e), "v": z(S, e), "o": z(R, d), "lse": z(n, H, lq), "z": z(R, f),
                  "a": z(R, f), "y": z(R, d), "o8": u8(R, d), "o8s": u8(R, -(-d // 32)), "z8": u8(R, f),
                  "z8s": u8(R, -(-f // 32)), "da": z(R, f), "dz": z(R, f), "do": z(R, d), "dq": z(R, d), "dk": z(S, e),
                  "dv": z(S, e), "dxe": z(S, d), "act": z(R, f)}
        self.g = {"Te": z(vocab, d), "Tq": z(vocab, d), "W1": z(f, d), "b1": z(f)}
        lay = lambda l, h: native.CPtcgHeadLayout(l * h * dh, h * dh, dh)
        self.a = native.CPtcgCrossAttn(n=n, lq=lq, lk=lk, heads=H, kv_heads=KV, dh=dh, bf16=0, scale=1 / math.sqrt(dh),
                                       q=lay(lq, H), k=lay(lk, KV), v=lay(lk, KV), o=lay(lq, H),
                                       k_len=self.k_len.data_ptr())
        L = native.lib()
        need = [L.ptcg_kernel_cross_attention_ws_bytes(ctypes.byref(self.a), b) for b in (0, 1)]
        need += [L.ptcg_kernel_embedding_bwd_ws_bytes(x, vocab, d) for x in (R, S)]
        need += [L.ptcg_kernel_ckpt8_dw_ws_bytes(R, d, f, 0)]
        assert min(need) >= 0
        self.ws = torch.full((max(need) + 16,), 0xff, dtype=torch.uint8, device="cuda")     # one scratch for all, in turn

    def run(self, stream=None):
        L, c, t, p, g = native.lib(), native.check, self.t, self.p, self.g
        n, R, S, d, e, f = self.n, self.n * self.lq, self.n * self.lk, self.d, self.dk_, self.f
        P = lambda x: x.data_ptr()

        def gemm(M, N, K, A, B, C, b_t=0, epi=0, bias=None, C2=None):
            c(L.ptcg_kernel_gemm(M, N, K, P(A), K, 0, P(B), N if b_t else K, b_t, P(C), N, epi, bias and P(bias), None, 0,
                                 P(C2) if C2 is not None else None, N, None, 0, stream))

        ws, nb = P(self.ws), self.ws.numel()
        c(L.ptcg_kernel_embedding_fwd(P(self.ids_e), S, P(p["Te"]), d, 0, self.vocab, d, self.s_e, P(t["xe"]), d, 0, stream))
        c(L.ptcg_kernel_embedding_fwd(P(self.ids_q), R, P(p["Tq"]), d, 0, self.vocab, d, self.s_q, P(t["xq"]), d, 0, stream))
        gemm(S, e, d, t["xe"], p["Wk"], t["k"])
        gemm(S, e, d, t["xe"], p["Wv"], t["v"])
        c(L.ptcg_kernel_cross_attention_fwd(ctypes.byref(self.a), P(t["xq"]), P(t["k"]), P(t["v"]), P(t["o"]), P(t["lse"]),
                                            ws, nb, stream))
        c(L.ptcg_kernel_gemm(R, f, d, P(t["o"]), d, 0, P(p["W1"]), d, 0, P(t["z"]), f, 2, P(p["b1"]), None, 0, P(t["a"]), f,
                             None, 0, stream))
        c(L.ptcg_kernel_ckpt8_pack(P(t["o"]), d, 0, R, d, P(t["o8"]), d, P(t["o8s"]), t["o8s"].stride(0), stream))
        c(L.ptcg_kernel_ckpt8_pack(P(t["z"]), f, 0, R, f, P(t["z8"]), f, P(t["z8s"]), t["z8s"].stride(0), stream))
        gemm(R, d, f, t["a"], p["W2"], t["y"])
        # backward
        gemm(R, f, d, self.dy, p["W2"], t["da"], b_t=1)
        c(L.ptcg_kernel_ckpt8_gelu_bwd(P(t["z8"]), f, P(t["z8s"]), t["z8s"].stride(0), R, f, P(t["da"]), f, P(t["dz"]), f,
                                       P(t["act"]), f, 0, stream))
        c(L.ptcg_kernel_ckpt8_dw(R, d, f, P(t["dz"]), f, 0, P(t["o8"]), d, P(t["o8s"]), t["o8s"].stride(0), P(g["W1"]),
                                 P(g["b1"]), ws, nb, stream))
        gemm(R, d, f, t["dz"], p["W1"], t["do"], b_t=1)
        c(L.ptcg_kernel_cross_attention_bwd(ctypes.byref(self.a), P(t["xq"]), P(t["k"]), P(t["v"]), P(t["o"]), P(t["lse"]),
                                            P(t["do"]), P(t["dq"]), P(t["dk"]), P(t["dv"]), ws, nb, stream))
        gemm(S, d, e, t["dk"], p["Wk"], t["dxe"], b_t=1)
        gemm(S, d, e, t["dv"], p["Wv"], t["dxe"], b_t=1, epi=5)
        c(L.ptcg_kernel_embedding_bwd(P(self.ids_q), R, P(t["dq"]), d, 0, self.vocab, d, self.s_q, P(g["Tq"]), d, ws, nb,
                                      stream))
        c(L.ptcg_kernel_embedding_bwd(P(self.ids_e), S, P(t["dxe"]), d, 0, self.vocab, d, self.s_e, P(g["Te"]), d, ws, nb,
                                      stream))

    def results(self):
        torch.cuda.synchronize()
        return {k: x.clone() for k, x in list(self.t.items()) + [("d" + k, x) for k, x in self.g.items()]}


def _close(name, got, want, err):
    over = (got.double() - want).abs() / err
    assert float(over.max()) <= 1.0, f"{name}: {float(over.max()):.3g} times its bound"


def _product(name, got, a, b, extra=0.0):
    """got = a b in fp32: K terms and their sums, (2 K + 16) u of sum |a||b|."""
    a, b = a.double(), b.double()
    _close(name, got, a @ b + extra, (2 * a.shape[1] + 16) * U * (a.abs() @ b.abs() + abs(extra)) + 1e-37)


def _scatter(name, got, ids, x, scale, vocab):
    """Sums of m terms: (m + 8) u of their absolute sum."""
    at = torch.where(ids >= 0, ids, vocab).reshape(-1).long()
    add = lambda y: torch.zeros(vocab + 1, y.shape[1], dtype=torch.float64, device="cuda").index_add_(0, at, y)[:vocab]
    m = torch.bincount(at, minlength=vocab + 1)[:vocab, None]
    x = x.double() * scale
    _close(name, got, add(x), (m + 8) * U * add(x.abs()) + 1e-37)


def test_a_decoder_block_from_tokens_to_table_gradients(cuda):
    """Every operator on what the one before it left, each against 64 bits on the
    same inputs; what 8 bits cost against the unrounded pre-activation."""
    m = Decoder()
    m.run()
    r, p = m.results(), m.p
    S, R = m.n * m.lk, m.n * m.lq
    live = (m.ids_e >= 0).reshape(-1)
    xe = torch.where(live[:, None], p["Te"][m.ids_e.reshape(-1).clamp(min=0).long()], 0.0).double() * m.s_e
    _close("xe", r["xe"], xe, U * xe.abs() + 1e-37)
    xq = p["Tq"][m.ids_q.reshape(-1).long()].double() * m.s_q
    _close("xq", r["xq"], xq, U * xq.abs() + 1e-37)
    _product("k", r["k"], r["xe"], p["Wk"].t())
    _product("v", r["v"], r["xe"], p["Wv"].t())
    rows = lambda x, i, l, h: x.view(m.n, l, h, m.dh)[i]
    for i in range(m.n):
        keep = torch.arange(m.lk, device="cuda") < m.lens[i]
        ref = reference(rows(r["xq"], i, m.lq, m.H), rows(r["k"], i, m.lk, m.KV), rows(r["v"], i, m.lk, m.KV), keep,
                        m.a.scale, rows(r["do"], i, m.lq, m.H))
        within(f"o[{i}]", rows(r["o"], i, m.lq, m.H), *ref["out"])
        within(f"dq[{i}]", rows(r["dq"], i, m.lq, m.H), *ref["dq"])
        within(f"dk[{i}]", rows(r["dk"], i, m.lk, m.KV), *ref["dk"])
        within(f"dv[{i}]", rows(r["dv"], i, m.lk, m.KV), *ref["dv"])
    _product("z", r["z"], r["o"], p["W1"].t(), p["b1"].double())
    z8, o8 = values64(r["z8"], r["z8s"]), values64(r["o8"], r["o8s"])
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the group's scale for small ones
    for x, x8, sc in ((r["z"], z8, r["z8s"]), (r["o"], o8, r["o8s"])):
        unit = torch.exp2(sc.double() - 127).repeat_interleave(32, 1)[:, :x.shape[1]]
        assert ((x8 - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * unit).all()
    _product("y", r["y"], r["a"], p["W2"].t())
    _product("da", r["da"], m.dy, p["W2"])
    # gelu' in fp32 is off by 0.75e-7 (its erf) and some u of values to 1 + |z|; it
    # moves by at most 0.8 |z8 - z| (|gelu''| <= 2 phi(0) = 0.798)
    dgelu = lambda z: 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    own = r["da"].double().abs() * (0.75e-7 + 16 * U) * (1 + z8.abs()) + 1e-37
    _close("dz", r["dz"], r["da"].double() * dgelu(z8), own + 8 * U * (r["da"].double() * dgelu(z8)).abs())
    _close("dz of 8 bits", r["dz"], r["da"].double() * dgelu(r["z"].double()),
           own + r["da"].double().abs() * (0.8 * (z8 - r["z"].double()).abs() + 8 * U))
    dz = r["dz"].double()
    _close("dW1", r["dW1"], dz.t() @ o8, (3 * R + 8) * U * (dz.abs().t() @ o8.abs()) + 1e-37)
    _close("db1", r["db1"], dz.sum(0), (R + 8) * U * dz.abs().sum(0) + 1e-37)
    _product("do", r["do"], r["dz"], p["W1"])
    both = lambda x: x.double()
    dxe = both(r["dk"]) @ both(p["Wk"]) + both(r["dv"]) @ both(p["Wv"])
    mag = both(r["dk"]).abs() @ both(p["Wk"]).abs() + both(r["dv"]).abs() @ both(p["Wv"]).abs()
    _close("dxe", r["dxe"], dxe, (4 * m.dk_ + 32) * U * mag + 1e-37)
    _scatter("dTq", r["dTq"], m.ids_q, r["dq"], m.s_q, m.vocab)
    _scatter("dTe", r["dTe"], m.ids_e, r["dxe"], m.s_e, m.vocab)


def test_the_decoder_block_captured_beside_an_eager_one(cuda):
    """The whole run in a graph, replayed between eager runs of a block of its own
    tensors: the same bits every time."""
    m, other = Decoder(), Decoder(n=5, lq=9, lk=40)
    m.run()
    want = m.results()
    other.run()
    want2 = other.results()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        m.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for x in list(m.t.values()) + list(m.g.values()) + [m.ws]:
            x.fill_(7)
        graph.replay()
        other.run()
        got, got2 = m.results(), other.results()
        assert all(torch.equal(got[k], want[k]) for k in want)
        assert all(torch.equal(got2[k], want2[k]) for k in want2)


def test_two_graphs_over_one_workspace_replayed_in_turn(cuda):
    a, b = Op(2, 1, 5000, 4, 4, 64, 1, seed=1), Op(2, 40, 1200, 4, 4, 96, 0, seed=2)
    b.ws = a.ws = torch.full((max(a.ws.numel(), b.ws.numel()),), 0xff, dtype=torch.uint8, device="cuda")
    graphs, want = [], []
    for op in (a, b):
        op.fwd()
        op.bwd()
        op.check()
        want.append([x.clone() for x in (op.out, op.lse, op.dq, op.dk, op.dv)])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            op.fwd(torch.cuda.current_stream().cuda_stream)
            op.bwd(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for op in (a, b):
            for x in (op.out, op.lse, op.dq, op.dk, op.dv):
                x.fill_(GUARD)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for op, w in zip((a, b), want):
            assert all(torch.equal(x, y) for x, y in zip((op.out, op.lse, op.dq, op.dk, op.dv), w))


def test_calls_on_two_streams_at_once(cuda):
    ops = [Op(3, 64, 97, 4, 2, 64, 0, seed=1), Op(3, 1, 9000, 8, 2, 128, 1, seed=2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    for _ in range(8):
        for op, st in zip(ops, streams):
            op.fwd(st.cuda_stream)
            op.bwd(st.cuda_stream)
    for op in ops:
        op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("n,dh", [(60, 64), (70, 32), (60, 128)])
def test_many_packed_samples(n, dh, bf16, cuda):
    """More workgroups than run at once: up to 64 samples go longest first, more in
    index order; some hold no row or no key."""
    g = torch.Generator().manual_seed(n + dh)
    ql = torch.randint(0, 41, (n,), generator=g).tolist()
    kl = torch.randint(0, 91, (n,), generator=g).tolist()
    ql[3], kl[5], ql[7], kl[9] = 0, 0, 40, 90
    op = Op(n, 40, 90, 10, 10, dh, bf16, q_len=ql, k_off_len=kl, slack=1)
    op.fwd()
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
def test_rows_of_one_time_step_side_by_side(bf16, cuda):
    """Time-major tensors (row, sample, head): the sample's stride is the smaller."""
    n, lq, lk, H, KV, dh = 3, 34, 70, 4, 2, 32
    op = Op(n, lq, lk, H, KV, dh, bf16)
    swap = lambda x, l, h: x.view(n, l, h, dh).transpose(0, 1).contiguous()
    tm = {k: swap(getattr(op, k), lq, H) for k in ("q", "out", "do", "dq")}
    tm.update({k: swap(getattr(op, k), lk, KV) for k in ("k", "v", "dk", "dv")})
    for name, h in (("q", H), ("o", H), ("k", KV), ("v", KV)):
        setattr(op.a, name, native.CPtcgHeadLayout(h * dh, n * h * dh, dh))
    kept = {k: getattr(op, k) for k in tm}
    for k, x in tm.items():
        setattr(op, k, x)
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    for k, x in kept.items():
        x.copy_(tm[k].transpose(0, 1).reshape(x.shape))
        setattr(op, k, x)
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
def test_a_single_key_row_of_any_stride(bf16, cuda):
    """One key a sample: its row stride says nothing."""
    op = Op(3, 5, 1, 2, 1, 64, bf16)
    for l in (op.a.k, op.a.v):
        l.sl = 8
    op.v[1, 0, 40] = math.nan
    op.fwd()
    torch.cuda.synchronize()
    bad = op.out[5:10].isnan()
    assert bad[:, :, 40].all() and int(bad.sum()) == 5 * 2
    op.v[1, 0, 40] = 0.0
    op.fwd()
    op.bwd()
    op.check()


def test_a_long_cache_past_2_to_31_elements(cuda):
    """One sample's key rows 2^15 elements apart: the last ones lie past 2^31."""
    lk, ld, H, dh = 65600, 1 << 15, 2, 64
    cache = torch.empty(lk * ld, dtype=torch.bfloat16, device="cuda").view(lk, ld)
    grads = torch.empty_like(cache)
    op = Op(1, 1, lk, H, 1, dh, 1)
    k, v = cache[:, :dh], cache[:, dh:2 * dh]
    k.copy_(op.k[:, 0])
    v.copy_(op.v[:, 0])
    lay = native.CPtcgHeadLayout(0, ld, dh)
    op.a.k = op.a.v = lay
    op.k, op.v, op.dk, op.dv = (x.unsqueeze(1) for x in (k, v, grads[:, :dh], grads[:, dh:2 * dh]))
    op.fwd()
    op.bwd()
    op.check()


def test_a_table_past_2_to_31_elements(cuda):
    vocab, d, rows = (1 << 21) + 8, 1024, 700
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.empty(vocab, d, dtype=torch.bfloat16, device="cuda")
    ids = torch.randint(vocab - 300, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    ids[::9] = 5
    used = ids.long().unique()
    table[used] = torch.randn(used.numel(), d, generator=g, device="cuda").bfloat16()
    out = torch.empty(rows, d, device="cuda")
    L = native.lib()
    native.check(L.ptcg_kernel_embedding_fwd(ids.data_ptr(), rows, table.data_ptr(), d, 1, vocab, d, 2.0, out.data_ptr(),
                                             d, 0, None))
    torch.cuda.synchronize()
    assert torch.equal(out, table[ids.long()].float() * 2)
    del table
    dt = torch.full((vocab, d), GUARD, device="cuda")
    ws = torch.empty(L.ptcg_kernel_embedding_bwd_ws_bytes(rows, vocab, d), dtype=torch.uint8, device="cuda")
    native.check(L.ptcg_kernel_embedding_bwd(ids.data_ptr(), rows, out.data_ptr(), d, 0, vocab, d, 0.5, dt.data_ptr(), d,
                                             ws.data_ptr(), ws.numel(), None))
    torch.cuda.synchronize()
    at = torch.searchsorted(used, ids.long())
    _scatter("dtable", dt[used], at, out, 0.5, used.numel())
    dt[used] = 0
    assert int(torch.count_nonzero(dt)) == 0


def test_checkpoints_past_2_to_31_bytes(cuda):
    rows, ld, d, n = 65600, 1 << 15, 40, 24
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, d, generator=g, device="cuda")
    q = torch.empty(rows * ld, dtype=torch.uint8, device="cuda").view(rows, ld)
    sc = torch.empty(rows, 2, dtype=torch.uint8, device="cuda")
    L = native.lib()
    native.check(L.ptcg_kernel_ckpt8_pack(x.data_ptr(), d, 0, rows, d, q.data_ptr(), ld, sc.data_ptr(), 2, None))
    back = torch.empty_like(x)
    native.check(L.ptcg_kernel_ckpt8_unpack(q.data_ptr(), ld, sc.data_ptr(), 2, rows, d, back.data_ptr(), d, 0, None))
    dy = torch.randn(rows, n, generator=g, device="cuda")
    dW = torch.empty(n, d, device="cuda")
    ws = torch.empty(max(16, L.ptcg_kernel_ckpt8_dw_ws_bytes(rows, d, n, 0)), dtype=torch.uint8, device="cuda")
    native.check(L.ptcg_kernel_ckpt8_dw(rows, d, n, dy.data_ptr(), n, 0, q.data_ptr(), ld, sc.data_ptr(), 2, dW.data_ptr(),
                                        None, ws.data_ptr(), ws.numel(), None))
    torch.cuda.synchronize()
    x8 = values64(q[:, :d], sc)
    assert torch.equal(back.double(), x8)
    assert ((x8 - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * 0.5).all()
    y = dy.double()
    _close("dW", dW, y.t() @ x8, (3 * rows + 8) * U * (y.abs().t() @ x8.abs()))


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("dh", [32, 64, 96])
@pytest.mark.parametrize("lq,H,KV,lk,mask", [(3, 8, 8, 60, "keep"), (1, 16, 8, 150, "len"), (7, 32, 8, 33, "keep"),
                                             (20, 8, 8, 540, "len"), (50, 8, 8, 70, "keep"), (9, 8, 8, 1, None)])
def test_many_samples_of_few_rows(lq, H, KV, lk, mask, dh, bf16, cuda):
    """More workgroups than run at once, with up to 64 rows a kv head: waves with no
    partners along the keys, or for dk and dv along the rows."""
    n = 70
    kw = {}
    if mask == "keep":
        g = torch.Generator(device="cuda").manual_seed(lk)
        kw["keep"] = (torch.rand(n, lk, generator=g, device="cuda") < 0.7).float()
        kw["keep"][5] = 0.0
    elif mask == "len":
        kw["k_len"] = [(37 * i) % (lk + 1) for i in range(n)]
    op = Op(n, lq, lk, H, KV, dh, bf16, seed=lk, **kw)
    if mask == "keep":
        dead = (kw["keep"] == 0).reshape(-1)
        ref = [x.clone() for x in (op.k, op.v)]
        op.k[dead] = math.nan
        op.v[dead] = math.inf
    op.fwd()
    op.bwd()
    if mask == "keep":
        op.k, op.v = ref
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk,H,KV,dh,mask", [(1, 1024, 8, 2, 128, "len"), (1, 1024, 8, 2, 64, "keep"),
                                                (30, 1500, 2, 2, 32, "keep"), (50, 1100, 2, 2, 96, "len"),
                                                (4, 2049, 8, 1, 64, "empty")])
def test_long_keys_split_over_lone_waves(lq, lk, H, KV, dh, mask, bf16, cuda):
    kw = {}
    if mask == "len":
        kw["k_len"] = [lk, 40]
    else:
        g = torch.Generator(device="cuda").manual_seed(lk)
        kw["keep"] = (torch.rand(2, lk, generator=g, device="cuda") < 0.6).float()
        kw["keep"][1, lk // 3:] = 0.0
        if mask == "empty":
            kw["keep"][0] = 0.0
    op = Op(2, lq, lk, H, KV, dh, bf16, seed=4, **kw)
    assert native.lib().ptcg_kernel_cross_attention_ws_bytes(ctypes.byref(op.a), 0) > 0     # the split form
    op.fwd()
    op.bwd()
    op.check()
    first = op.out.clone()
    op.ws.fill_(0xff)
    op.fwd(lse=False)
    torch.cuda.synchronize()
    assert torch.equal(op.out, first)


@pytest.mark.parametrize("bf16", [0, 1])
def test_packed_rows_fewer_than_the_bound(bf16, cuda):
    """The bounds lq and lk of packed samples may pass all rows there are, in
    matrices of one head after the other too."""
    op = Op(2, 90, 200, 4, 2, 32, bf16, q_len=[3, 20], k_off_len=[30, 11], order="hld")
    op.fwd()
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("dh", [32, 64, 88, 128])
@pytest.mark.parametrize("lq,lk", [(2, 161), (33, 97), (2, 65), (5, 100), (61, 190)])
def test_wave_halves_without_rows_against_several_tiles(lq, lk, dh, bf16, cuda):
    """Lanes without a query row still carry their share of every key tile."""
    op = Op(3, lq, lk, 2, 2, dh, bf16, seed=30)
    op.fwd()
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("rows", [32, 33, 34, 35, 36, 65, 3000])
@pytest.mark.parametrize("k,n,pad", [(1, 4, 0), (1, 4, 1), (2, 1, 0), (3, 3, 0), (5, 1, 1), (9, 7, 0)])
def test_weight_gradient_of_the_narrowest_rows(k, n, pad, rows, bf16, cuda):
    """Rows of 1 to 9 bytes, whose last dword ends rows later."""
    check_weight_gradient(rows, k, n, pad, bf16, cuda)
