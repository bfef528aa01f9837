"""Cross attention (ptcg_kernel_cross_attention_*) against 64 bits: types, head
layouts, lengths, masks, packed samples, gradients, single tokens, graphs."""
import ctypes
import math

import pytest
import torch

from ptcg_amd import native
from refxattn import reference, within

pytestmark = pytest.mark.gpu

GUARD = 7.25   # what untouched memory holds


class Op:
    """Descriptor, outputs and workspace of one call.  order: 'lhd' rows of
    heads, 'hld' heads of rows, 'kv' k and v interleaved in one matrix."""

    def __init__(self, n, lq, lk, H, KV, dh, bf16, q_len=None, k_off_len=None, k_len=None, keep=None, order="lhd",
                 share_kv=False, seed=0, scale=None, slack=0):
        self.t = torch.bfloat16 if bf16 else torch.float32
        self.n, self.lq, self.lk, self.H, self.KV, self.dh, self.bf16 = n, lq, lk, H, KV, dh, bf16
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(self.t)
        self.scale = scale or 1 / math.sqrt(dh)
        a = native.CPtcgCrossAttn(n=n, lq=lq, lk=lk, heads=H, kv_heads=KV, dh=dh, bf16=int(bf16), scale=self.scale)
        self.q_off = self.k_off = None

        def offsets(lens):
            return torch.tensor([3 * slack + sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda")

        qr, kr = n * lq, n * lk
        if q_len is not None:
            self.q_off = offsets(q_len)
            qr = int(self.q_off[-1]) + slack
        if k_off_len is not None:
            self.k_off = offsets(k_off_len)
            kr = int(self.k_off[-1]) + slack
        self.qr, self.kr = qr, kr

        def make(rows, heads, per):
            """(rows, heads, dh) view with the order's memory layout, and its strides."""
            if order == "hld":
                if per is not None:   # padded: sample, head, row
                    m = rnd(rows // per, heads, per, dh)
                    return m, (heads * per * dh, dh, per * dh), lambda x: x.transpose(1, 2).reshape(rows, heads, dh)
                m = rnd(heads, rows, dh)
                return m, (0, dh, rows * dh), lambda x: x.transpose(0, 1)
            m = rnd(rows, heads, dh)
            return m, ((per or 0) * heads * dh, heads * dh, dh), lambda x: x

        qper = lq if q_len is None else None
        kper = lk if k_off_len is None else None
        self.q, ql, self.qv = make(qr, H, qper)
        self.out = torch.full_like(self.q, GUARD)
        self.do = rnd(*self.q.shape)
        self.dq = torch.full_like(self.q, GUARD)
        if order == "kv":
            m = rnd(kr, 2, KV, dh)
            kl = ((kper or 0) * 2 * KV * dh, 2 * KV * dh, dh)
            self.kv, self.dkv = m, torch.full_like(m, GUARD)
            self.k, self.v, self.dk, self.dv = m[:, 0], m[:, 1], self.dkv[:, 0], self.dkv[:, 1]
            self.kview = lambda x: x
        else:
            self.k, kl, self.kview = make(kr if not share_kv else lk, KV, kper)
            self.v = rnd(*self.k.shape)
            self.dk, self.dv = torch.full_like(self.k, GUARD), torch.full_like(self.k, GUARD)
            if share_kv:
                kl = (0,) + kl[1:]
        self.share_kv = share_kv
        for name, l in (("q", ql), ("o", ql), ("k", kl), ("v", kl)):
            setattr(a, name, native.CPtcgHeadLayout(*l))
        self.k_len = None if k_len is None else torch.tensor(k_len, dtype=torch.int32, device="cuda")
        self.keep = keep
        for name in ("q_off", "k_off", "k_len", "keep"):
            t = getattr(self, name)
            setattr(a, name, None if t is None else t.data_ptr())
        a.keep_sn = lk
        self.a = a
        self.lse = torch.full((n, H, lq), GUARD, device="cuda")
        L = native.lib()
        nb = [L.ptcg_kernel_cross_attention_ws_bytes(ctypes.byref(a), x) for x in (0, 1)]
        assert min(nb) >= 0
        self.ws = torch.full((max(16, *nb),), 0xff, dtype=torch.uint8, device="cuda")

    def fwd(self, stream=None, lse=True):
        native.check(native.lib().ptcg_kernel_cross_attention_fwd(
            ctypes.byref(self.a), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.out.data_ptr(),
            self.lse.data_ptr() if lse else None, self.ws.data_ptr(), self.ws.numel(), stream))

    def bwd(self, stream=None):
        native.check(native.lib().ptcg_kernel_cross_attention_bwd(
            ctypes.byref(self.a), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.out.data_ptr(),
            self.lse.data_ptr(), self.do.data_ptr(), self.dq.data_ptr(), self.dk.data_ptr(), self.dv.data_ptr(),
            self.ws.data_ptr(), self.ws.numel(), stream))

    def samples(self):
        """(i, query rows, key rows, keep) of each sample, over the (rows, heads, dh) views."""
        for i in range(self.n):
            qa, qb = (int(self.q_off[i]), int(self.q_off[i + 1])) if self.q_off is not None else \
                (i * self.lq, (i + 1) * self.lq)
            if self.k_off is not None:
                ka, kb = int(self.k_off[i]), int(self.k_off[i + 1])
                kp = self.keep[ka:kb] != 0 if self.keep is not None else None
            else:
                ka, kb = (0, self.lk) if self.share_kv else (i * self.lk, (i + 1) * self.lk)
                kp = self.keep[i] != 0 if self.keep is not None else None
            if kp is None:
                kp = torch.ones(kb - ka, dtype=torch.bool, device="cuda")
            if self.k_len is not None:
                kp = kp & (torch.arange(self.lk, device="cuda") < int(self.k_len[i]))
            yield i, slice(qa, qb), slice(ka, kb), kp

    def check(self, bwd=True, lse=True):
        torch.cuda.synchronize()
        q, o, do, dq = (self.qv(x) for x in (self.q, self.out, self.do, self.dq))
        k, v, dk, dv = (self.kview(x) for x in (self.k, self.v, self.dk, self.dv))
        qmask = torch.zeros(self.qr, dtype=torch.bool, device="cuda")
        kmask = torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
        for i, qs, ks, kp in self.samples():
            qmask[qs] = True
            kmask[ks] = True
            r = reference(q[qs], k[ks], v[ks], kp, self.scale, do[qs] if bwd else None, self.bf16)
            within(f"out[{i}]", o[qs], *r["out"])
            if lse:
                within(f"lse[{i}]", self.lse[i, :, :qs.stop - qs.start], *r["lse"])
            if bwd:
                within(f"dq[{i}]", dq[qs], *r["dq"])
                within(f"dk[{i}]", dk[ks], *r["dk"])
                within(f"dv[{i}]", dv[ks], *r["dv"])
        # rows of no sample stay as they were
        for x, m in ((o, qmask),) + (((dq, qmask), (dk, kmask), (dv, kmask)) if bwd else ()):
            assert (x[~m] == GUARD).all()


def _holes(n, lk, seed, share=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(n, lk, generator=g, device="cuda") < share).float()


SHAPES = [
    # n, lq, lk, H, KV, dh
    (1, 1, 1, 1, 1, 8), (2, 1, 33, 4, 4, 32), (3, 5, 7, 6, 2, 40), (2, 31, 64, 2, 1, 64), (2, 33, 65, 4, 4, 64),
    (1, 64, 97, 4, 4, 64), (2, 65, 129, 2, 2, 96), (1, 129, 31, 4, 1, 128), (1, 40, 300, 8, 2, 128),
    (3, 17, 200, 5, 5, 16), (1, 300, 33, 3, 1, 72), (2, 96, 32, 2, 2, 24),
]


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, bf16, cuda):
    print(f"cross attention {shape} bf16={bf16}", flush=True)
    op = Op(*shape, bf16)
    op.fwd()
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("order", ["hld", "kv"])
@pytest.mark.parametrize("packed", [False, True])
def test_layouts(order, packed, bf16, cuda):
    kw = dict(q_len=[5, 0, 40, 33], k_off_len=[70, 9, 0, 33], slack=2) if packed else {}
    n, lq, lk = (4, 40, 70) if packed else (2, 37, 70)
    op = Op(n, lq, lk, 4, 2, 64, bf16, order=order, **kw)
    op.fwd()
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("dh", [32, 64, 128])
def test_packed_rows_behind_the_last_sample_stay(dh, bf16, cuda):
    keep = None
    ql, kl = [1, 130, 17, 0, 64], [33, 1, 200, 64, 0]
    op = Op(5, 130, 200, 8, 2, dh, bf16, q_len=ql, k_off_len=kl, slack=5, seed=3)
    op.keep = (torch.rand(op.kr, generator=op.g, device="cuda") < 0.8).float()
    op.a.keep = op.keep.data_ptr()
    op.fwd()
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk", [(1, 50), (40, 50), (64, 97), (100, 200)])
def test_masks_with_empty_rows_and_nan_behind_them(lq, lk, bf16, cuda):
    keep = _holes(4, lk, 5)
    keep[1] = 0.0                      # a sample that keeps nothing
    keep[2] = 0.0
    keep[2, lk - 1] = -3.0             # only the last key, by any nonzero value
    keep[3, lk // 2:] = 0.0            # a prefix
    op = Op(4, lq, lk, 4, 2, 64, bf16, keep=keep, seed=1)
    dead = (keep == 0).reshape(-1)
    ref = [x.clone() for x in (op.k, op.v)]
    op.k[dead] = math.nan
    op.v[dead] = math.inf
    op.fwd()
    op.bwd()
    op.k, op.v = ref                   # the reference zeroes masked rows anyway
    op.check()
    assert (op.out[op.lq:2 * op.lq] == 0).all() and (op.dk[dead] == 0).all() and (op.dv[dead] == 0).all()


@pytest.mark.parametrize("bf16", [0, 1])
def test_nan_queries_of_an_empty_sample_and_of_a_live_one(bf16, cuda):
    keep = torch.ones(2, 40, device="cuda")
    keep[0] = 0.0
    op = Op(2, 9, 40, 2, 2, 32, bf16, keep=keep)
    op.q[:9] = math.nan
    op.q[9 + 4] = math.nan
    op.do[:9] = math.nan
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    assert (op.out[:9] == 0).all() and (op.dq[:9] == 0).all() and (op.lse[0] == -math.inf).all()
    assert (op.dk[:40] == 0).all() and (op.dv[:40] == 0).all()
    assert op.out[9 + 4].isnan().all() and op.lse[1, :, 4].isnan().all()
    rest = torch.cat([op.out[9:9 + 4], op.out[9 + 5:]])
    assert rest.isfinite().all()


@pytest.mark.parametrize("bf16", [0, 1])
def test_key_counts(bf16, cuda):
    op = Op(5, 20, 77, 4, 1, 64, bf16, k_len=[77, 0, 1, 33, 200], seed=2)   # a count past lk reads lk rows
    for i, n in enumerate([77, 0, 1, 33, 77]):
        op.k[i * 77 + n:(i + 1) * 77] = math.nan
    op.fwd()
    op.bwd()
    op.k.nan_to_num_(0.0)
    op.check()
    assert (op.dk[77:2 * 77] == 0).all() and (op.dv[2 * 77 + 1:3 * 77] == 0).all()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk,H,KV,dh,mask", [(1, 5000, 8, 2, 128, "len"), (1, 4097, 4, 4, 64, "keep"),
                                                (3, 3001, 8, 1, 32, None), (2, 1029, 3, 3, 40, "empty"),
                                                (70, 2100, 2, 2, 64, "keep")])
def test_few_rows_against_many_keys(lq, lk, H, KV, dh, mask, bf16, cuda):
    kw = {}
    if mask == "len":
        kw["k_len"] = [lk, 700]
    elif mask is not None:
        kw["keep"] = _holes(2, lk, 9)
        kw["keep"][1, lk // 3:] = 0.0
        if mask == "empty":
            kw["keep"][0] = 0.0
    op = Op(2, lq, lk, H, KV, dh, bf16, seed=4, **kw)
    assert native.lib().ptcg_kernel_cross_attention_ws_bytes(ctypes.byref(op.a), 0) > 0     # the split form
    op.fwd()
    op.check(bwd=False)
    op.out.fill_(GUARD)
    op.fwd(lse=False)
    op.check(bwd=False, lse=False)
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk,H,KV,dh,order,packed", [
    (700, 40, 4, 2, 64, "lhd", False), (600, 130, 6, 2, 128, "kv", True), (20, 900, 8, 2, 32, "hld", False),
    (513, 520, 2, 1, 40, "lhd", True), (40, 1200, 4, 4, 96, "kv", True)])
def test_backward_split_over_a_long_axis(lq, lk, H, KV, dh, order, packed, bf16, cuda):
    """Few workgroups along one axis: keys (for dq) or rows (for dk, dv) are split
    and added; masks and lengths cut through the splits."""
    if packed:
        op = Op(3, lq, lk, H, KV, dh, bf16, q_len=[lq, 0, lq // 3], k_off_len=[lk // 2, 7, lk], order=order, slack=3)
    else:
        op = Op(2, lq, lk, H, KV, dh, bf16, order=order, k_len=[lk, lk // 3])
        op.keep = _holes(2, lk, 2)
        op.a.keep = op.keep.data_ptr()
    n, R = op.n, op.n * H * lq
    assert native.lib().ptcg_kernel_cross_attention_ws_bytes(ctypes.byref(op.a), 1) > 4 * R + 16    # the split form
    op.fwd()
    op.bwd()
    op.check()
    a = [x.clone() for x in (op.dq, op.dk, op.dv)]
    op.ws.fill_(0xff)
    op.bwd()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, (op.dq, op.dk, op.dv)))


def test_broadcast_keys_and_queries_in_the_forward(cuda):
    op = Op(6, 10, 50, 4, 2, 32, 0, share_kv=True)
    op.fwd()
    op.check(bwd=False)
    with pytest.raises(native.PtcgError, match="overlap"):
        op.bwd()


@pytest.mark.parametrize("bf16", [0, 1])
def test_large_scores_keep_their_softmax(bf16, cuda):
    """Scores of several hundred, whose exponentials alone would overflow, in
    tiles that raise the running maximum late."""
    op = Op(1, 40, 260, 2, 2, 64, bf16, scale=1.0)
    op.q *= 8
    op.k *= torch.linspace(0.2, 4, 260, device="cuda")[:, None, None].to(op.t)
    op.fwd()
    op.bwd()
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk", [(1, 5000), (64, 97)])
def test_repeats_bit_for_bit(lq, lk, bf16, cuda):
    op = Op(3, lq, lk, 8, 2, 64, bf16)
    got = []
    for _ in range(2):
        for x in (op.out, op.dq, op.dk, op.dv):
            x.fill_(GUARD)
        op.fwd()
        op.bwd()
        torch.cuda.synchronize()
        got.append([x.clone() for x in (op.out, op.lse, op.dq, op.dk, op.dv)])
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("lq,lk", [(1, 5000), (64, 97)])
def test_captured_and_replayed_on_a_stream_of_its_own(lq, lk, cuda):
    op = Op(2, lq, lk, 4, 4, 64, 1)
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    want = [x.clone() for x in (op.out, op.lse, op.dq, op.dk, op.dv)]
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        op.fwd(torch.cuda.current_stream().cuda_stream)
        op.bwd(torch.cuda.current_stream().cuda_stream)
    q0 = op.q.clone()
    for k in range(3):
        for x in (op.out, op.lse, op.dq, op.dk, op.dv):
            x.fill_(GUARD)
        op.q.copy_(q0 * 2)             # other inputs in between, run eagerly
        op.fwd()
        op.q.copy_(q0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((op.out, op.lse, op.dq, op.dk, op.dv), want):
            assert torch.equal(x, y), f"replay {k}"


def test_gradients_against_differences(cuda):
    """Central differences of sum(out . do) along random directions, fp32
    kernel, at two steps: the tolerance is their disagreement (the h^2 term)
    plus the forward's own error bound over the step."""
    op = Op(2, 9, 21, 4, 2, 16, 0, keep=_holes(2, 21, 3))
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    noise = sum(float((reference(op.q[qs], op.k[ks], op.v[ks], kp, op.scale)["out"][1] * op.do[qs].double().abs()).sum())
                for _, qs, ks, kp in op.samples())
    for name in ("q", "k", "v"):
        x = getattr(op, name)
        grad = getattr(op, "d" + name).double()
        d = torch.randn(x.shape, generator=op.g, device="cuda")
        x0, diff = x.clone(), {}
        for h in (2.0 ** -5, 2.0 ** -6):
            loss = []
            for sgn in (1, -1):
                x.copy_(x0 + sgn * h * d)
                op.fwd()
                torch.cuda.synchronize()
                loss.append(float((op.out.double() * op.do.double()).sum()))
            diff[h] = (loss[0] - loss[1]) / (2 * h)
        x.copy_(x0)
        want = float((grad * d.double()).sum())
        tol = abs(diff[2.0 ** -5] - diff[2.0 ** -6]) + 4 * noise / 2.0 ** -6
        assert abs(want - diff[2.0 ** -6]) <= tol, (name, want, diff, tol)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk,H,KV,dh", [(1, 2100, 4, 2, 64), (37, 70, 4, 2, 40), (150, 90, 6, 2, 128), (64, 97, 4, 4, 64),
                                           (20, 700, 8, 1, 96)])
@pytest.mark.parametrize("packed", ["", "q", "k", "qk"])
def test_every_tensor_in_a_layout_of_its_own(packed, lq, lk, H, KV, dh, bf16, cuda):
    """q and k as rows of heads, out (with dout) and v (with dv) as heads of rows
    with a gap between them, queries and keys packed or padded on their own."""
    n = 3
    kw = dict(q_len=[lq, lq // 2, 1]) if "q" in packed else {}
    if "k" in packed:
        kw["k_off_len"] = [lk // 3, lk, 2]
    op = Op(n, lq, lk, H, KV, dh, bf16, slack=2, seed=lq + lk, **kw)
    if "k" in packed:
        op.keep = (torch.rand(op.kr, generator=op.g, device="cuda") < 0.7).float()
    else:
        op.keep = _holes(n, lk, 7)
    op.a.keep = op.keep.data_ptr()

    def turned(x, per, heads):
        """x (rows, heads, dh) in a new memory of (sample, head, row, dh + 8); its strides, and the way back."""
        m = torch.full((x.shape[0] // per, heads, per, dh + 8), GUARD, dtype=x.dtype, device="cuda")
        m[..., :dh] = x.view(-1, per, heads, dh).transpose(1, 2)
        return m, native.CPtcgHeadLayout(heads * per * (dh + 8), dh + 8, per * (dh + 8)), \
            lambda: m[..., :dh].transpose(1, 2).reshape(x.shape)

    qper, kper = (op.qr if "q" in packed else lq), (op.kr if "k" in packed else lk)
    flat = dict(do=op.do, v=op.v)
    op.out, op.a.o, out = turned(op.out, qper, H)
    op.do = turned(op.do, qper, H)[0]
    op.v, op.a.v, _ = turned(op.v, kper, KV)
    op.dv, _, dv = turned(op.dv, kper, KV)
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    for m in (op.out, op.dv):
        assert (m[..., dh:] == GUARD).all()
    op.out, op.dv = out(), dv()
    op.do, op.v = flat["do"], flat["v"]
    op.check()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk", [(1, 3000), (5, 40), (70, 97), (130, 300)])
@pytest.mark.parametrize("name", ["k", "v"])
def test_one_row_for_all_keys_in_the_forward(name, lq, lk, bf16, cuda):
    """A row stride of 0: every key reads the same row, masked ones aside."""
    op = Op(2, lq, lk, 4, 2, 64, bf16, keep=_holes(2, lk, 11), seed=8)
    x = getattr(op, name)
    x.view(2, lk, -1)[:] = x.view(2, lk, -1)[:, :1].clone()
    lay = native.CPtcgHeadLayout(lk * 2 * 64, 0, 64)
    setattr(op.a, name, lay)
    op.fwd()
    op.check(bwd=False)


@pytest.mark.parametrize("lq,lk", [(1, 2000), (40, 97), (130, 300)])
def test_bf16_rows_whose_every_kept_score_is_minus_infinity(lq, lk, cuda):
    """They count as rows that keep no key; a finite score beside the infinite
    ones gets the whole weight."""
    op = Op(2, lq, lk, 2, 2, 32, 1, keep=_holes(2, lk, 12), seed=9)
    op.q.abs_()
    op.q += 0.125
    op.k[:, :, 5] = -math.inf
    j = int(op.keep[1].nonzero()[0, 0])
    op.k[lk + j] = 0.5
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    assert (op.out[:lq] == 0).all() and (op.lse[0] == -math.inf).all() and (op.dq[:lq] == 0).all()
    assert (op.dk[:lk] == 0).all() and (op.dv[:lk] == 0).all()
    assert torch.equal(op.out[lq:], op.v[lk + j].expand(lq, 2, 32)) and op.lse[1].isfinite().all()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("lq,lk", [(5, 0), (300, 0), (0, 70), (0, 1)])
def test_no_keys_and_no_queries(lq, lk, bf16, cuda):
    """Without keys: out and dq of zeros, lse = -inf; without queries: dk and dv of zeros."""
    op = Op(2, lq, lk, 4, 2, 40, bf16)
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    assert (op.out == 0).all() and (op.dq == 0).all() and (op.lse == -math.inf).all()
    assert (op.dk == 0).all() and (op.dv == 0).all()
