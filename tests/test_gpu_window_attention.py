"""Causal attention with a window and first tokens over whole sequences
(ptcg_kernel_window_attention_*) against 64 bits, both directions."""
import ctypes
import math

import pytest
import torch

from ptcg_amd import native
from refseq import attention, sees, within

pytestmark = pytest.mark.gpu

GUARD = 7.25
LAY = native.CPtcgHeadLayout


class Op:
    """lens: live rows of each sequence; packed, or padded to l rows.  order: 'lhd' rows of heads, 'hld' heads of
    rows, 'qkv' q, k, v and their gradients in one matrix each."""

    def __init__(self, lens, l, H, KV, dh, bf16, window=0, sinks=0, packed=False, order="lhd", slack=0, seed=0,
                 scale=None, dead=float("nan")):
        self.t = torch.bfloat16 if bf16 else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed + 11 * dh + l)
        n = len(lens)
        self.lens, self.n, self.l, self.H, self.KV, self.dh, self.bf16 = lens, n, l, H, KV, dh, bf16
        self.window, self.sinks, self.packed = window, sinks, packed
        self.first = [slack + sum(lens[:i]) for i in range(n + 1)] if packed else [i * l for i in range(n + 1)]
        rows = self.first[-1] + (slack if packed else 0)
        self.rows = rows
        live = torch.zeros(rows, dtype=torch.bool, device="cuda")
        for i in range(n):
            live[self.first[i]:self.first[i] + lens[i]] = True
        self.live = live

        def rnd(h):
            x = torch.randn(rows, h, dh, generator=g, device="cuda").to(self.t)
            x[~live] = dead
            return x

        def make(h, values=None):
            """(rows, h, dh) view in the order's memory, and its layout."""
            if order == "hld":
                buf = torch.full((h, rows, dh), GUARD, dtype=self.t, device="cuda")
                view, lay = buf.transpose(0, 1), LAY(sn=l * dh, sl=dh, sh=rows * dh)
            else:
                buf = torch.full((rows, h, dh), GUARD, dtype=self.t, device="cuda")
                view, lay = buf, LAY(sn=l * h * dh, sl=h * dh, sh=dh)
            if values is not None:
                view.copy_(values)
            return view, lay

        if order == "qkv":
            w = (H + 2 * KV) * dh
            lay = LAY(sn=l * w, sl=w, sh=dh)
            both = []
            for fill in (lambda: rnd(H + 2 * KV), lambda: torch.full((rows, H + 2 * KV, dh), GUARD, dtype=self.t,
                                                                     device="cuda")):
                m = fill()
                both.append((m[:, :H], m[:, H:H + KV], m[:, H + KV:]))
            (self.q, self.k, self.v), (self.dq, self.dk, self.dv) = both
            lq = lk = lv = lay
        else:
            self.q, lq = make(H, rnd(H))
            self.k, lk = make(KV, rnd(KV))
            self.v, lv = make(KV, rnd(KV))
            self.dq, self.dk, self.dv = make(H)[0], make(KV)[0], make(KV)[0]
        self.out, lo = make(H)
        self.do, _ = make(H, rnd(H))
        self.lse = torch.full((n, H, l), GUARD, device="cuda")
        self.off = torch.tensor(self.first, dtype=torch.int32, device="cuda") if packed else None
        self.len = torch.tensor(lens, dtype=torch.int32, device="cuda") if not packed and min(lens) < l else None
        self.scale = scale or 1 / math.sqrt(dh)
        p = lambda t: None if t is None else t.data_ptr()
        self.a = native.CPtcgWindowAttn(n=n, l=l, heads=H, kv_heads=KV, dh=dh, bf16=int(bf16), scale=self.scale,
                                        window=window, sinks=sinks, q=lq, k=lk, v=lv, o=lo, off=p(self.off),
                                        len=p(self.len))
        nb = [native.lib().ptcg_kernel_window_attention_ws_bytes(ctypes.byref(self.a), x) for x in (0, 1)]
        assert min(nb) >= 0
        self.ws = torch.full((max(16, *nb),), 0xff, dtype=torch.uint8, device="cuda")

    def fwd(self, stream=None, lse=True):
        native.check(native.lib().ptcg_kernel_window_attention_fwd(
            ctypes.byref(self.a), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.out.data_ptr(),
            self.lse.data_ptr() if lse else None, self.ws.data_ptr(), self.ws.numel(), stream))
        return self

    def bwd(self, stream=None):
        native.check(native.lib().ptcg_kernel_window_attention_bwd(
            ctypes.byref(self.a), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.out.data_ptr(),
            self.lse.data_ptr(), self.do.data_ptr(), self.dq.data_ptr(), self.dk.data_ptr(), self.dv.data_ptr(),
            self.ws.data_ptr(), self.ws.numel(), stream))
        return self

    def check(self, bwd=True, lse=True):
        torch.cuda.synchronize()
        for i in range(self.n):
            m = self.lens[i]
            if m == 0:
                continue
            x = slice(self.first[i], self.first[i] + m)
            at = torch.arange(m, device="cuda")
            ref = attention(self.q[x], self.k[x], self.v[x], sees(at, at, self.window, self.sinks), self.scale,
                            self.do[x] if bwd else None, self.bf16)
            within(f"out[{i}]", self.out[x], *ref["out"])
            if lse:
                within(f"lse[{i}]", self.lse[i, :, :m], *ref["lse"])
            if bwd:
                for name in ("dq", "dk", "dv"):
                    within(f"{name}[{i}]", getattr(self, name)[x], *ref[name])
        dead = GUARD if self.packed else 0.0
        for name in ("out", "dq", "dk", "dv") if bwd else ("out",):
            assert (getattr(self, name)[~self.live] == dead).all(), name
        if not self.packed and lse:
            for i in range(self.n):
                assert (self.lse[i, :, self.lens[i]:] == -math.inf).all()
        return self


CASES = [
    dict(lens=[97, 40, 1, 0], l=97, H=4, KV=4, dh=64, bf16=False, window=32, sinks=1),
    dict(lens=[97, 40, 1, 0], l=97, H=4, KV=4, dh=64, bf16=True, window=32, sinks=1),
    dict(lens=[97] * 3, l=97, H=4, KV=2, dh=32, bf16=False),
    dict(lens=[1, 1], l=1, H=4, KV=2, dh=64, bf16=True),
    dict(lens=[7, 8, 3], l=8, H=4, KV=1, dh=64, bf16=True, window=3),
    dict(lens=[31, 32, 30], l=32, H=1, KV=1, dh=128, bf16=False, window=5, sinks=2),
    dict(lens=[50, 64, 33], l=64, H=2, KV=2, dh=128, bf16=True, order="qkv"),
    dict(lens=[50, 64, 33], l=64, H=2, KV=2, dh=128, bf16=False, order="hld"),
    dict(lens=[300, 129, 5], l=300, H=6, KV=3, dh=40, bf16=True, window=100, sinks=7, packed=True, slack=3),
    dict(lens=[300, 129, 5, 0, 64], l=300, H=6, KV=2, dh=96, bf16=False, window=100, packed=True, slack=2, order="qkv"),
    dict(lens=[300, 129, 5, 0, 64], l=300, H=8, KV=2, dh=128, bf16=True, packed=True, order="hld"),
    # rows that see first tokens alone, cut into chunks
    dict(lens=[700, 400, 160], l=700, H=4, KV=2, dh=64, bf16=True, window=20, sinks=3, packed=True, slack=1),
    dict(lens=[1300, 400, 160], l=1300, H=4, KV=2, dh=128, bf16=True, window=20, sinks=200),
    dict(lens=[900, 64], l=900, H=4, KV=2, dh=128, bf16=False, window=1, sinks=256, packed=True),
    dict(lens=[900, 64], l=900, H=2, KV=2, dh=64, bf16=True, window=64, sinks=300),
    dict(lens=[900, 64], l=900, H=2, KV=2, dh=64, bf16=True, window=64, sinks=2000, packed=True),
    dict(lens=[700], l=700, H=4, KV=1, dh=64, bf16=False, window=700, sinks=5),
    dict(lens=[1000], l=1000, H=2, KV=1, dh=128, bf16=True, window=1),
    dict(lens=[2050], l=2050, H=2, KV=1, dh=128, bf16=True),          # keys split
    dict(lens=[2050], l=2050, H=1, KV=1, dh=64, bf16=False, window=1500, sinks=4),
    dict(lens=[20 + 3 * i for i in range(80)], l=260, H=2, KV=1, dh=32, bf16=True, window=50, sinks=2, packed=True),
    dict(lens=[5] * 300, l=5, H=4, KV=4, dh=8, bf16=False, window=2, sinks=1),
    # few key tiles, cut along their rows; sequences without rows among them
    dict(lens=[900, 0, 300, 1], l=900, H=8, KV=1, dh=64, bf16=True),
    dict(lens=[900, 0, 300, 1], l=900, H=8, KV=1, dh=128, bf16=False, window=200, sinks=3),
    dict(lens=[0, 900, 257, 64], l=900, H=8, KV=1, dh=96, bf16=True, window=90, sinks=150, packed=True, slack=2),
]


@pytest.mark.parametrize("kw", CASES, ids=str)
def test_both_directions(cuda, kw):
    Op(**kw).fwd().bwd().check()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("l", [33, 64, 65, 96, 127, 128, 129, 192, 193])
def test_lengths_around_tiles(cuda, l, bf16):
    Op(lens=[l, l - 1, l - 31], l=l, H=3, KV=1, dh=64, bf16=bf16, window=l // 2, sinks=1).fwd().bwd().check()


@pytest.mark.parametrize("window", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 199, 200, 201, 2 ** 31 - 1])
def test_windows_around_tiles(cuda, window):
    Op(lens=[200], l=200, H=2, KV=1, dh=64, bf16=True, window=window, sinks=2).fwd().bwd().check()
    Op(lens=[200, 77], l=200, H=3, KV=1, dh=64, bf16=True, window=window, packed=True).fwd().bwd().check()


@pytest.mark.parametrize("l, dh", [(33, 64), (35, 128), (65, 32), (97, 128)])
def test_rows_so_far_apart_that_a_sequence_passes_31_bits(cuda, l, dh):
    """The queries' rows 2^31 bytes apart in all (bf16), the outputs' beside each other, and the other way round."""
    g = torch.Generator(device="cuda").manual_seed(l)
    H, KV, st = 2, 1, (2 ** 31 // 2 // l // 64 + 1) * 64
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    near, apart = LAY(sn=0, sl=H * dh, sh=dh), LAY(sn=0, sl=st, sh=dh)
    at = torch.arange(l, device="cuda")
    k, v, vals, grads = rnd(l, KV, dh), rnd(l, KV, dh), rnd(l, H, dh), rnd(l, H, dh)
    ref = attention(vals, k, v, sees(at, at, 20, 2), dh ** -0.5, grads, True)
    wide = lambda: torch.empty(l * st, dtype=torch.bfloat16, device="cuda").as_strided((l, H, dh), (st, dh, 1))
    dense = lambda: torch.empty(l, H, dh, dtype=torch.bfloat16, device="cuda")
    for lq, lo in ((apart, near), (near, apart)):
        q, dq = (wide() if lq is apart else dense() for _ in range(2))
        out, do = (wide() if lo is apart else dense() for _ in range(2))
        dk, dv = torch.empty_like(k), torch.empty_like(v)
        q.copy_(vals)
        do.copy_(grads)
        lse = torch.empty(H, l, device="cuda")
        lk = LAY(sn=0, sl=KV * dh, sh=dh)
        a = native.CPtcgWindowAttn(n=1, l=l, heads=H, kv_heads=KV, dh=dh, bf16=1, scale=dh ** -0.5, window=20, sinks=2,
                                   q=lq, k=lk, v=lk, o=lo)
        lib = native.lib()
        nb = max(lib.ptcg_kernel_window_attention_ws_bytes(ctypes.byref(a), x) for x in (0, 1))
        ws = torch.full((nb,), 0xff, dtype=torch.uint8, device="cuda")
        native.check(lib.ptcg_kernel_window_attention_fwd(
            ctypes.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), ws.data_ptr(), nb,
            None))
        native.check(lib.ptcg_kernel_window_attention_bwd(
            ctypes.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), do.data_ptr(),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), nb, None))
        torch.cuda.synchronize()
        for name, x in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
            within(name, x, *ref[name])
        within("lse", lse, *ref["lse"])


def test_forward_alone_and_large_scores(cuda):
    Op(lens=[500, 130], l=500, H=4, KV=2, dh=64, bf16=True, packed=True).fwd(lse=False).check(bwd=False, lse=False)
    Op(lens=[150, 130], l=150, H=4, KV=2, dh=64, bf16=False, scale=6.0, window=40).fwd().bwd().check()


@pytest.mark.parametrize("kw", [CASES[0], CASES[11], CASES[18]], ids=str)
def test_repeats_bit_for_bit_and_replays(cuda, kw):
    op = Op(**kw).fwd().bwd().check()
    names = ("out", "lse", "dq", "dk", "dv")
    first = {m: getattr(op, m).clone() for m in names}
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        st = torch.cuda.current_stream().cuda_stream
        op.fwd(st).bwd(st)
    for _ in range(3):
        for m in names:
            getattr(op, m).fill_(GUARD)
        op.ws.fill_(0xff)
        g.replay()
        torch.cuda.synchronize()
        for m in names:
            assert torch.equal(getattr(op, m)[op.live] if m != "lse" else op.lse.nan_to_num(),
                               first[m][op.live] if m != "lse" else first[m].nan_to_num()), m


def test_gradients_against_differences(cuda):
    """Central differences of the kernel's forward in fp32, of the sum of outputs times do: a step of 2^-6 leaves the
    third derivative's share, the forward's rounding 2^-24 / 2^-6 per output, both below 1e-2 of the largest gradient."""
    op = Op(lens=[40, 23], l=40, H=4, KV=2, dh=16, bf16=False, window=9, sinks=2, packed=True).fwd().bwd()
    h = 2.0 ** -6

    def loss():
        op.fwd()
        torch.cuda.synchronize()
        return float((op.out.double() * op.do.double()).sum())

    for x, dx in ((op.q, op.dq), (op.k, op.dk), (op.v, op.dv)):
        size = float(dx.double().abs().max())
        for row, head, e in ((0, 0, 3), (5, 1, 0), (39, 1, 15), (40, 0, 7), (62, 1, 2)):
            keep, at = float(x[row, head, e]), []
            for step in (h, -h):
                x[row, head, e] = keep + step
                at.append(loss())
            x[row, head, e] = keep
            assert abs((at[0] - at[1]) / (2 * h) - float(dx[row, head, e])) <= 1e-2 * size


@pytest.mark.parametrize("l", [3, 9, 18, 64, 200])
def test_bf16_gradients_are_off_by_two_roundings(cuda, l):
    """A rounding to bf16 is off by at most 2^-8 / m of a value of mantissa m in [1, 2), evenly: 2^-8 / sqrt(3) sqrt(mean
    1 / m^2) = 1.66e-3 in relative L2, with m logarithmically spread (mean 1 / m^2 = 3 / (8 ln 2)).  dq and dk are
    rounded themselves and made from one rounded factor, dS: 2.35e-3, and a tenth for chance.  (dq of keys
    past one tile has the rounding of the output in it as well.)"""
    n = max(4, 2000 // l)
    op = Op(lens=[l] * n, l=l, H=2, KV=2, dh=64, bf16=True, packed=True).fwd().bwd()
    torch.cuda.synchronize()
    at = torch.arange(l, device="cuda")
    got, want = {"dq": [], "dk": []}, {"dq": [], "dk": []}
    for i in range(n):
        x = slice(i * l, (i + 1) * l)
        ref = attention(op.q[x], op.k[x], op.v[x], sees(at, at, 0, 0), op.scale, op.do[x], True)
        for name in got:
            got[name].append(getattr(op, name)[x].double())
            want[name].append(ref[name][0].double())
    for name in ("dq", "dk") if l <= 64 else ("dk",):
        a, b = torch.cat(got[name]), torch.cat(want[name])
        off = float((a - b).norm() / b.norm())
        assert off < 1.1 * 2.35e-3, (name, off)


def test_broadcast_keys_in_the_forward(cuda):
    """One sequence's keys for all (stride 0)."""
    op = Op(lens=[90, 90, 90], l=90, H=4, KV=2, dh=64, bf16=True, window=30, sinks=1)
    op.a.k.sn = op.a.v.sn = 0
    op.fwd()
    for i in (1, 2):
        op.k[90 * i:90 * (i + 1)] = op.k[:90]
        op.v[90 * i:90 * (i + 1)] = op.v[:90]
    op.check(bwd=False)


def test_two_calls_on_streams_with_scratch_of_their_own(cuda):
    ops = [Op(lens=[900, 300], l=900, H=4, KV=2, dh=64, bf16=True, window=50, sinks=3, packed=True, seed=i)
           for i in range(2)]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    for op, s in zip(ops, streams):
        op.fwd(s.cuda_stream).bwd(s.cuda_stream)
    for op in ops:
        op.check()


def test_many_sequences_whose_parts_pass_one_round_of_the_sum(cuda):
    """16 800 (sequence, kv head) pairs with two cut key tiles of 128: 2^24.04 threads' worth of sums, of which a
    launch has 2^24; the long sequences are the last ones."""
    Op(lens=[3] * 2060 + [400, 300, 0, 150] * 10, l=400, H=8, KV=8, dh=8, bf16=True, window=1, sinks=200,
       packed=True).fwd().bwd().check()


def test_packed_sequences_of_as_many_rows_as_a_launch_takes(cuda):
    """4 096 sequences that might have 8 192 rows each, 8 kv heads: over 2^31 threads of 2^32."""
    Op(lens=[0] * 4000 + [3] * 60 + [200, 0, 97, 1] * 9, l=8192, H=8, KV=8, dh=8, bf16=True, packed=True,
       slack=1).fwd().bwd().check()
