"""Norms of queries and keys with the rotation (ptcg_kernel_qk_norm_rope_*) and the
way into a paged cache (ptcg_kernel_paged_append) against 64 bits."""
import ctypes

import pytest
import torch

from ptcg_amd import native
from refseq import frequencies, norm_rope, within

pytestmark = pytest.mark.gpu

GUARD = 7.25
LAY = native.CPtcgHeadLayout


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rope(rot, inter, scaling, pos):
    """CPtcgRope from the library's frequencies, and what it has to keep alive."""
    f, mag = (ctypes.c_double * max(1, rot // 2))(), ctypes.c_float()
    native.check(native.lib().ptcg_rope_frequencies(rot, 10000.0, scaling, 8.0, 4096.0, 32.0, 1.0, f, ctypes.byref(mag)))
    freq = torch.tensor(list(f)[:rot // 2], dtype=torch.float64, device="cuda")
    return native.CPtcgRope(rot=rot, interleaved=int(inter), mag=mag.value, freq=_ptr(freq) if rot else None,
                            pos=_ptr(pos)), freq


def _weight(g, dh, on):
    return 1 + 0.3 * torch.randn(dh, generator=g, device="cuda") if on else None


# n, l, H, KV, dh, rot, inter, bf16, norm, pos, order, off (elements the buffers start late)
CASES = [
    (3, 5, 4, 4, 64, 64, False, False, "qk", None, "lhd", 0),
    (1, 1, 1, 1, 128, 128, True, True, "qk", None, "lhd", 0),
    (2, 97, 4, 2, 64, 64, False, True, "qk", None, "lhd", 0),
    (1, 300, 8, 2, 128, 64, True, True, "qk", "far", "lhd", 0),
    (1, 300, 8, 2, 128, 32, False, False, "q", "far", "hld", 0),
    (2, 33, 6, 3, 40, 10, False, True, "k", "neg", "lhd", 0),
    (2, 33, 6, 3, 96, 24, True, True, "", "far", "lhd", 0),
    (1, 7, 3, 1, 2, 2, False, False, "qk", None, "lhd", 0),
    (1, 19, 2, 2, 6, 4, True, True, "qk", "far", "lhd", 1),
    (2, 21, 5, 1, 64, 64, False, True, "qk", None, "lhd", 3),
    (2, 21, 5, 1, 72, 36, True, False, "qk", None, "lhd", 2),
    (1, 40, 9, 0, 64, 0, False, True, "qk", None, "lhd", 0),
    (1, 1201, 16, 4, 128, 128, False, True, "qk", None, "lhd", 0),
    (40, 97, 4, 4, 64, 64, False, False, "qk", None, "lhd", 0),
    (1, 9000, 2, 1, 32, 16, True, True, "qk", "far", "lhd", 0),
]


class Op:
    def __init__(self, n, l, H, KV, dh, rot, inter, bf16, norm, pos, order, off, scaling=0, seed=0):
        self.t = torch.bfloat16 if bf16 else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed + 100 * dh + l)
        rows = n * l
        rnd = lambda h: (torch.randn(rows, h, dh, generator=g, device="cuda") *
                         torch.exp(torch.randn(rows, 1, 1, generator=g, device="cuda"))).to(self.t)
        self.hold = []

        def place(values, h):
            """A copy of (rows, h, dh) values in the order's memory, starting `off` elements late."""
            buf = torch.full((rows * h * dh + off + 8,), GUARD, dtype=self.t, device="cuda")
            self.hold.append(buf)
            body = buf[off:off + rows * h * dh]
            view = body.view(rows, h, dh) if order == "lhd" else body.view(h, rows, dh).transpose(0, 1)
            view.copy_(values)
            return view

        blank = lambda h: torch.full((rows, h, dh), GUARD, dtype=self.t, device="cuda")
        self.q, self.k = place(rnd(H), H), place(rnd(KV), KV)
        self.dqo, self.dko = place(rnd(H), H), place(rnd(KV), KV)
        self.qo, self.ko = place(blank(H), H), place(blank(KV), KV)
        self.dq, self.dk = place(blank(H), H), place(blank(KV), KV)
        self.wq, self.wk = _weight(g, dh, "q" in norm), _weight(g, dh, "k" in norm and KV)
        self.pos = None
        if pos == "far":
            self.pos = torch.randint(0, 2 ** 31 - 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if pos == "neg":
            self.pos = torch.randint(-5000, 5000, (rows,), generator=g, device="cuda", dtype=torch.int32)
        rope, self.freq = _rope(rot, inter, scaling, self.pos)
        self.ref_freq, self.mag = frequencies(rot, scaling=scaling) if rot else ([], 1.0)
        lay = lambda h: LAY(sn=l * h * dh, sl=h * dh, sh=dh) if order == "lhd" else LAY(sn=l * dh, sl=dh, sh=rows * dh)
        self.a = native.CPtcgQkRope(n=n, l=l, heads=H, kv_heads=KV, dh=dh, bf16=int(bf16), eps=1e-6, q=lay(H),
                                    k=lay(KV), qo=lay(H), ko=lay(KV), wq=_ptr(self.wq), wk=_ptr(self.wk), rope=rope)
        self.dwq = torch.full((dh,), GUARD, device="cuda") if self.wq is not None else None
        self.dwk = torch.full((dh,), GUARD, device="cuda") if self.wk is not None else None
        nb = native.lib().ptcg_kernel_qk_norm_rope_bwd_ws_bytes(ctypes.byref(self.a))
        assert nb >= 0
        self.ws = torch.full((max(16, nb),), 0xff, dtype=torch.uint8, device="cuda")
        self.at = self.pos if self.pos is not None else torch.arange(l, device="cuda").repeat(n)
        self.inter, self.KV = inter, KV

    def fwd(self, stream=None, inplace=False):
        qo, ko = (self.q, self.k) if inplace else (self.qo, self.ko)
        native.check(native.lib().ptcg_kernel_qk_norm_rope_fwd(ctypes.byref(self.a), _ptr(self.q), _ptr(self.k), _ptr(qo),
                                                               _ptr(ko), stream))

    def bwd(self, stream=None):
        native.check(native.lib().ptcg_kernel_qk_norm_rope_bwd(
            ctypes.byref(self.a), _ptr(self.q), _ptr(self.k), _ptr(self.dqo), _ptr(self.dko), _ptr(self.dq), _ptr(self.dk),
            _ptr(self.dwq), _ptr(self.dwk), _ptr(self.ws), self.ws.numel(), stream))

    def check(self, q, k, qo, ko, bwd=True):
        torch.cuda.synchronize()
        for name, x, y, w, dy, dx, dw in (("q", q, qo, self.wq, self.dqo, self.dq, self.dwq),
                                          ("k", k, ko, self.wk, self.dko, self.dk, self.dwk)):
            if not x.numel():
                continue
            ref = norm_rope(x, w, 1e-6, self.at, self.ref_freq, self.mag, self.inter, self.t, dy)
            within(name + "o", y, *ref["y"])
            if bwd:
                within("d" + name, dx, *ref["dx"])
                if dw is not None:
                    within("dw" + name, dw, *ref["dw"])
        for buf in self.hold:      # before and behind the tensors
            assert (buf[-8:] == GUARD).all()


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("scaling", [0, 3])
def test_both_directions(cuda, case, scaling):
    op = Op(*case, scaling=scaling)
    op.fwd()
    op.bwd()
    op.check(op.q, op.k, op.qo, op.ko)


@pytest.mark.parametrize("case", [CASES[2], CASES[5], CASES[8]], ids=str)
def test_in_place(cuda, case):
    op = Op(*case)
    q, k = op.q.clone(), op.k.clone()
    op.fwd()
    op.fwd(inplace=True)
    torch.cuda.synchronize()
    assert torch.equal(op.q, op.qo) and torch.equal(op.k, op.ko)
    op.check(q, k, op.q, op.k, bwd=False)


def test_gradients_against_differences(cuda):
    """Central differences of the kernel's own forward in fp32, of the sum of output times dqo: steps of 2^-6 leave
    the third derivative's share below 1e-3 of the gradient's size."""
    op = Op(1, 3, 2, 1, 16, 8, False, False, "qk", "neg", "lhd", 0)
    op.bwd()
    h = 2.0 ** -6

    def loss():
        op.fwd()
        torch.cuda.synchronize()
        return float((op.qo.double() * op.dqo.double()).sum() + (op.ko.double() * op.dko.double()).sum())

    size = float(op.dq.double().abs().max())
    for x, dx in ((op.q, op.dq), (op.k, op.dk), (op.wq, op.dwq), (op.wk, op.dwk)):
        flat, grad = x.view(-1), dx.reshape(-1)
        for e in (0, 5, flat.numel() - 1):
            keep, at = float(flat[e]), []
            for step in (h, -h):
                flat[e] = keep + step
                at.append(loss())
            flat[e] = keep
            assert abs((at[0] - at[1]) / (2 * h) - float(grad[e])) <= 2e-2 * max(size, abs(float(grad[e])))


def test_every_call_repeats_bit_for_bit_and_replays(cuda):
    op = Op(*CASES[12])
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    names = ("qo", "ko", "dq", "dk", "dwq", "dwk")
    first = {m: getattr(op, m).clone() for m in names}
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        op.fwd(torch.cuda.current_stream().cuda_stream)
        op.bwd(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for m in names:
            getattr(op, m).fill_(GUARD)
        g.replay()
        torch.cuda.synchronize()
        for m in names:
            assert torch.equal(getattr(op, m), first[m]), m


def test_broadcast_inputs_and_a_weightless_side(cuda):
    """One row for every head (stride 0) forward; gradients without either weight need no scratch and no inputs."""
    op = Op(2, 9, 4, 2, 32, 32, False, False, "", None, "lhd", 0)
    op.a.q.sh = 0
    op.fwd()
    op.check(op.q[:, :1].expand_as(op.q), op.k, op.qo, op.ko, bwd=False)
    op = Op(2, 9, 4, 2, 32, 32, False, False, "", None, "lhd", 0)
    native.check(native.lib().ptcg_kernel_qk_norm_rope_bwd(ctypes.byref(op.a), None, None, _ptr(op.dqo), _ptr(op.dko),
                                                           _ptr(op.dq), _ptr(op.dk), None, None, None, 0, None))
    op.fwd()
    op.check(op.q, op.k, op.qo, op.ko)


def test_no_rows_leave_gradients_of_zero(cuda):
    op = Op(1, 1, 2, 1, 32, 32, False, False, "qk", None, "lhd", 0)
    op.a.n = 0
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    assert (op.qo == GUARD).all() and (op.dwq == 0).all() and (op.dwk == 0).all()


# ------------------------------------------------------------------ the cache
class Append:
    """lens: lengths with the new rows; new: new rows of each sequence (packed), or one number for all."""

    def __init__(self, lens, new, H, KV, dh, rot, inter, bf16, page, order="rows", norm=True, pos=False, slack=0,
                 per_seq=None, with_q=True, seed=0):
        self.t = torch.bfloat16 if bf16 else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed + 17 * dh + page)
        n = len(lens)
        packed = isinstance(new, list)
        self.new = new if packed else [new] * n
        self.first = [slack + sum(self.new[:i]) for i in range(n + 1)]
        rows = self.first[-1] + slack
        self.rows, self.lens, self.page, self.n, self.dh, self.H, self.KV = rows, lens, page, n, dh, H, KV
        per = per_seq or max(1, -(-max(max(lens), 1) // page))
        pages = n * per + 5
        self.table = torch.randperm(pages, generator=g, device="cuda")[:n * per].int().view(n, per)
        shape = (pages, page, KV, dh) if order == "rows" else (pages, KV, page, dh)
        self.kp, self.vp = (torch.full(shape, GUARD, dtype=self.t, device="cuda") for _ in range(2))
        self.view = (lambda x: x) if order == "rows" else (lambda x: x.transpose(1, 2))
        self.qkv = torch.randn(rows, H + 2 * KV, dh, generator=g, device="cuda").to(self.t)
        self.qo = torch.full((rows, H, dh), GUARD, dtype=self.t, device="cuda")
        self.wq, self.wk = _weight(g, dh, norm), _weight(g, dh, norm)
        self.pos = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32) if pos else None
        self.len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.q_off = torch.tensor(self.first, dtype=torch.int32, device="cuda") if packed else None
        rope, self.freq = _rope(rot, inter, 0, self.pos)
        self.ref_freq, self.mag, self.inter = (frequencies(rot)[0] if rot else []), 1.0, inter
        w, l = (H + 2 * KV) * dh, max(max(self.new), 1)
        sl, sh = (KV * dh, dh) if order == "rows" else (dh, page * dh)
        lay, pl = LAY(sn=l * w, sl=w, sh=dh), LAY(sn=page * KV * dh, sl=sl, sh=sh)
        self.a = native.CPtcgPagedAppend(
            n=n, lq=l, rows=rows, heads=H, kv_heads=KV, dh=dh, bf16=int(bf16), eps=1e-6, q=lay, k=lay, v=lay,
            qo=LAY(sn=l * H * dh, sl=H * dh, sh=dh), q_off=_ptr(self.q_off), len=_ptr(self.len), wq=_ptr(self.wq),
            wk=_ptr(self.wk), rope=rope,
            cache=native.CPtcgPages(pages=pages, page=page, per_seq=per, k=pl, v=pl, kp=_ptr(self.kp), vp=_ptr(self.vp),
                                    table=_ptr(self.table), table_sn=per))
        self.with_q = with_q

    def run(self, stream=None):
        e = self.qkv.element_size() * self.dh
        p = _ptr(self.qkv)
        native.check(native.lib().ptcg_kernel_paged_append(
            ctypes.byref(self.a), p if self.with_q else None, p + self.H * e, p + (self.H + self.KV) * e,
            _ptr(self.qo) if self.with_q else None, stream))

    def check(self):
        torch.cuda.synchronize()
        want = {m: torch.full(x.shape, GUARD, dtype=torch.float64, device="cuda")
                for m, x in (("kp", self.kp), ("vp", self.vp), ("qo", self.qo))}
        err = {m: torch.full_like(x, 1e-30) for m, x in want.items()}
        H, KV = self.H, self.KV
        for i in range(self.n):
            rows = torch.arange(self.first[i], self.first[i + 1], device="cuda")
            if not len(rows):
                continue
            place = self.lens[i] - self.new[i] + torch.arange(self.new[i], device="cuda")
            at = self.pos[rows].long() if self.pos is not None else place
            x = self.qkv[rows]
            turned = lambda lo, hi, w: norm_rope(x[:, lo:hi], w, 1e-6, at, self.ref_freq, self.mag, self.inter,
                                                 self.t)["y"]
            if self.with_q:
                want["qo"][rows], err["qo"][rows] = turned(0, H, self.wq)
            k, kerr = turned(H, H + KV, self.wk)
            ok = (place >= 0) & (place // self.page < self.table.shape[1])
            pg = self.table[i].long()[(place // self.page).clamp(0, self.table.shape[1] - 1)]
            ok &= (pg >= 0) & (pg < self.kp.shape[0])
            pg, row = pg[ok], place[ok] % self.page
            self.view(want["kp"])[pg, row], self.view(err["kp"])[pg, row] = k[ok], kerr[ok]
            self.view(want["vp"])[pg, row] = x[ok][:, H + KV:].double()
        for m in want:
            within(m, getattr(self, m), want[m], err[m])


@pytest.mark.parametrize("kw", [
    dict(lens=[1, 17, 64, 100], new=1, H=4, KV=4, dh=64, rot=64, inter=False, bf16=False, page=16),
    dict(lens=[1, 17, 64, 100], new=1, H=8, KV=2, dh=128, rot=64, inter=True, bf16=True, page=16, order="heads"),
    dict(lens=[40, 5, 300, 33], new=[40, 0, 17, 1], H=8, KV=2, dh=128, rot=128, inter=False, bf16=True, page=64, slack=3),
    dict(lens=[40, 5, 300, 33], new=[40, 0, 17, 1], H=6, KV=3, dh=40, rot=10, inter=False, bf16=True, page=1),
    dict(lens=[90, 31], new=[7, 31], H=2, KV=1, dh=96, rot=96, inter=True, bf16=False, page=24, order="heads", slack=2),
    dict(lens=[90, 31], new=[7, 31], H=2, KV=1, dh=64, rot=0, inter=False, bf16=True, page=7, norm=False),
    dict(lens=[90, 31], new=9, H=2, KV=1, dh=64, rot=64, inter=False, bf16=True, page=32, pos=True, with_q=False),
    dict(lens=[3000], new=[2900], H=8, KV=8, dh=128, rot=128, inter=False, bf16=True, page=64),
    dict(lens=list(range(1, 258)), new=1, H=4, KV=4, dh=32, rot=32, inter=False, bf16=True, page=16),
    dict(lens=[2, 1, 40], new=[5, 4, 12], H=2, KV=1, dh=32, rot=32, inter=False, bf16=False, page=4),   # places below 0
    dict(lens=[50, 9], new=[8, 9], H=2, KV=1, dh=32, rot=32, inter=False, bf16=False, page=4, per_seq=11),   # past the table
], ids=str)
def test_append(cuda, kw):
    op = Append(**kw)
    op.run()
    op.check()
    op.run()      # the same again: nothing else moves
    op.check()


def test_append_to_entries_that_are_no_page(cuda):
    op = Append(lens=[64, 64], new=[40, 40], H=2, KV=1, dh=64, rot=64, inter=False, bf16=True, page=16)
    op.table[0, 2], op.table[1, 3], op.table[1, 2] = -1, op.kp.shape[0], 2 ** 31 - 1
    op.run()
    op.check()


def test_append_in_place_and_on_another_stream(cuda):
    op = Append(lens=[64, 20], new=[40, 9], H=4, KV=2, dh=64, rot=64, inter=False, bf16=True, page=16)
    op.run()
    torch.cuda.synchronize()
    qo = op.qo.clone()
    op.a.qo = op.a.q
    s = torch.cuda.Stream()
    p, e = _ptr(op.qkv), op.dh * 2
    native.check(native.lib().ptcg_kernel_paged_append(ctypes.byref(op.a), p, p + 4 * e, p + 6 * e, p, s.cuda_stream))
    s.synchronize()
    assert torch.equal(op.qkv[:, :4], qo)


def test_a_cache_past_32_bit_offsets(cuda):
    """Pages far into a pool of more than 2^32 bytes and 2^31 elements."""
    pages, page, KV, dh = 17000, 1024, 1, 128     # 2.2e9 elements
    kp = torch.empty(pages, page, KV, dh, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    op = Append(lens=[1500, 3], new=[8, 3], H=2, KV=1, dh=128, rot=128, inter=False, bf16=True, page=1024)
    op.table[0, 1], op.table[1, 0] = pages - 1, pages - 3
    small_k, small_v = op.kp, op.vp
    c = op.a.cache
    c.pages, c.kp, c.vp = pages, _ptr(kp), _ptr(vp)
    op.run()
    torch.cuda.synchronize()
    k = norm_rope(op.qkv[:8, 2:3], op.wk, 1e-6, torch.arange(1492, 1500, device="cuda"), op.ref_freq, 1.0, False, op.t)
    within("k", kp[pages - 1, 1492 - 1024:1500 - 1024], *k["y"])
    assert torch.equal(vp[pages - 3, :3], op.qkv[8:11, 3:4]) and torch.equal(vp[pages - 1, 468:476], op.qkv[:8, 3:4])
    assert (small_k == GUARD).all() and (small_v == GUARD).all()
