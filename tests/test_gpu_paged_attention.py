"""Attention over a paged cache (ptcg_kernel_paged_attention) against 64 bits:
tokens and chunks, pages of every size, windows, first tokens, masked entries."""
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
    """lens: lengths with the new rows; new: rows of each sequence (packed), or one number for all."""

    def __init__(self, lens, new, H, KV, dh, bf16, page, window=0, sinks=0, order="rows", slack=0, per_seq=None, seed=0,
                 scale=None, q_order="lhd", garbage=float("nan")):
        self.t = torch.bfloat16 if bf16 else torch.float32
        g = torch.Generator(device="cuda").manual_seed(seed + 7 * dh + page)
        n = len(lens)
        packed = isinstance(new, list)
        self.new = new if packed else [new] * n
        self.first = [slack + sum(self.new[:i]) for i in range(n + 1)]
        rows = self.first[-1] + slack
        self.lens, self.page, self.n, self.H, self.KV, self.dh = lens, page, n, H, KV, dh
        self.window, self.sinks, self.bf16, self.rows = window, sinks, bf16, rows
        per = per_seq if per_seq is not None else max(1, -(-max(max(lens), 1) // page))
        self.per = per
        pages = n * per + 3
        self.table = torch.randperm(pages, generator=g, device="cuda")[:n * per].int().view(n, per)
        shape = (pages, page, KV, dh) if order == "rows" else (pages, KV, page, dh)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(self.t)
        # places that no sequence has reached hold garbage
        self.kp, self.vp = (torch.full(shape, garbage, dtype=self.t, device="cuda") for _ in range(2))
        self.view = (lambda x: x) if order == "rows" else (lambda x: x.transpose(1, 2))
        for i, m in enumerate(lens):
            m = min(m, per * page)
            if m > 0:
                p = torch.arange(m, device="cuda")
                for pool in (self.kp, self.vp):
                    self.view(pool)[self.table[i].long()[p // page], p % page] = rnd(m, KV, dh)
        l = max(max(self.new), 1)
        if q_order == "lhd":
            self.q, lay, self.qv = rnd(rows, H, dh), LAY(sn=l * H * dh, sl=H * dh, sh=dh), lambda x: x
        else:
            self.q, lay, self.qv = rnd(H, rows, dh), LAY(sn=l * dh, sl=dh, sh=rows * dh), lambda x: x.transpose(0, 1)
        self.out = torch.full_like(self.q, GUARD)
        self.lse = torch.full((n, H, l), GUARD, device="cuda")
        self.len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.q_off = torch.tensor(self.first, dtype=torch.int32, device="cuda") if packed else None
        sl, sh = (KV * dh, dh) if order == "rows" else (dh, page * dh)
        pl = LAY(sn=page * KV * dh, sl=sl, sh=sh)
        self.scale = scale or 1 / math.sqrt(dh)
        self.a = native.CPtcgPagedAttn(
            n=n, lq=l, rows=rows, heads=H, kv_heads=KV, dh=dh, bf16=int(bf16), scale=self.scale, window=window, sinks=sinks,
            q=lay, o=lay, q_off=self.q_off.data_ptr() if packed else None, len=self.len.data_ptr(),
            cache=native.CPtcgPages(pages=pages, page=page, per_seq=per, k=pl, v=pl, kp=self.kp.data_ptr(),
                                    vp=self.vp.data_ptr(), table=self.table.data_ptr(), table_sn=per))
        nb = native.lib().ptcg_kernel_paged_attention_ws_bytes(ctypes.byref(self.a))
        assert nb >= 0
        self.ws = torch.full((max(16, nb),), 0xff, dtype=torch.uint8, device="cuda")

    def run(self, stream=None, lse=True):
        native.check(native.lib().ptcg_kernel_paged_attention(
            ctypes.byref(self.a), self.q.data_ptr(), self.out.data_ptr(), self.lse.data_ptr() if lse else None,
            self.ws.data_ptr(), self.ws.numel(), stream))
        return self

    def check(self, lse=True):
        torch.cuda.synchronize()
        q, out = self.qv(self.q), self.qv(self.out)
        seen = torch.zeros(self.rows, dtype=torch.bool, device="cuda")
        for i in range(self.n):
            lo, hi = self.first[i], self.first[i + 1]
            seen[lo:hi] = True
            if hi == lo:
                continue
            m = max(0, min(self.lens[i], self.per * self.page))
            p = torch.arange(m, device="cuda")
            pg = self.table[i].long()[p // self.page] if self.per else p
            ok = (pg >= 0) & (pg < self.kp.shape[0])
            pg = pg.clamp(0, self.kp.shape[0] - 1)
            k, v = (self.view(x)[pg, p % self.page] for x in (self.kp, self.vp))
            at = self.lens[i] - self.new[i] + torch.arange(self.new[i], device="cuda")
            see = sees(at, p, self.window, self.sinks) & ok[None]
            ref = attention(q[lo:hi], k, v, see, self.scale, bf16=self.bf16)
            within(f"out[{i}]", out[lo:hi], *ref["out"])
            if lse:
                within(f"lse[{i}]", self.lse[i, :, :hi - lo], *ref["lse"])
        assert (out[~seen] == GUARD).all()
        return self


TOKENS = [
    dict(lens=[1, 17, 64, 100], H=4, KV=4, dh=64, bf16=False, page=16),
    dict(lens=[1, 17, 64, 100, 0, 3], H=8, KV=2, dh=128, bf16=True, page=16, order="heads"),
    dict(lens=[5000, 33, 1, 700], H=8, KV=2, dh=128, bf16=True, page=64),
    dict(lens=[5000, 33, 1, 700], H=8, KV=2, dh=128, bf16=False, page=64),
    dict(lens=[3001], H=8, KV=1, dh=64, bf16=True, page=1),
    dict(lens=[3001, 2000], H=6, KV=3, dh=40, bf16=True, page=24),
    dict(lens=[3001, 2000], H=6, KV=3, dh=96, bf16=False, page=7, order="heads"),
    dict(lens=[3001, 2000, 90], H=4, KV=4, dh=32, bf16=True, page=128, window=100),
    dict(lens=[3001, 2000, 90, 103, 104, 105], H=4, KV=2, dh=64, bf16=True, page=16, window=100, sinks=4),
    dict(lens=[9000, 2000, 90], H=32, KV=1, dh=128, bf16=True, page=64, window=3000, sinks=37),
    dict(lens=[9000, 2000, 90], H=4, KV=4, dh=64, bf16=True, page=32, window=1, sinks=1),
    dict(lens=[9000, 12], H=4, KV=4, dh=8, bf16=False, page=32, window=5, sinks=10000),
    dict(lens=list(range(1, 300)), H=4, KV=1, dh=64, bf16=True, page=16),
    dict(lens=[20000] * 3, H=16, KV=1, dh=128, bf16=True, page=256),
    dict(lens=[1500] * 70, H=8, KV=4, dh=64, bf16=True, page=16, q_order="hld"),
]


@pytest.mark.parametrize("kw", TOKENS, ids=str)
def test_tokens(cuda, kw):
    Op(new=1, **kw).run().check()


CHUNKS = [
    dict(lens=[40, 5, 300, 33], new=[40, 0, 17, 1], H=8, KV=2, dh=128, bf16=True, page=64, slack=3),
    dict(lens=[40, 5, 300, 33], new=[40, 0, 17, 1], H=8, KV=2, dh=128, bf16=False, page=16, slack=3),
    dict(lens=[1000, 700, 64], new=[500, 130, 64], H=4, KV=4, dh=64, bf16=True, page=16),
    dict(lens=[1000, 700, 64], new=[500, 130, 64], H=4, KV=4, dh=64, bf16=False, page=24),
    dict(lens=[1000, 700, 64], new=[500, 130, 64], H=6, KV=2, dh=96, bf16=True, page=1),
    dict(lens=[1000, 700, 64], new=[500, 130, 64], H=6, KV=2, dh=96, bf16=True, page=5, order="heads"),
    dict(lens=[1000, 700, 64], new=[500, 130, 64], H=6, KV=3, dh=40, bf16=True, page=32, window=77, sinks=3),
    dict(lens=[3000, 700, 64], new=[1500, 130, 64], H=8, KV=2, dh=128, bf16=True, page=64, window=200, sinks=4),
    dict(lens=[3000, 700, 64], new=[1500, 130, 64], H=8, KV=2, dh=128, bf16=True, page=48, window=200, sinks=70),
    dict(lens=[3000, 700, 64], new=[1500, 130, 64], H=2, KV=2, dh=32, bf16=True, page=16, window=1),
    dict(lens=[9000, 700], new=[100, 65], H=4, KV=2, dh=128, bf16=True, page=64),              # split
    dict(lens=[9000, 700], new=[100, 65], H=4, KV=2, dh=64, bf16=False, page=16, window=4000, sinks=9),
    dict(lens=[6000, 900, 300], new=8, H=4, KV=1, dh=128, bf16=True, page=16),                # 32 rows
    dict(lens=[6000, 900, 300], new=9, H=5, KV=1, dh=128, bf16=True, page=16, window=2500, sinks=4),   # 45 rows
    dict(lens=[6000, 900, 300], new=3, H=7, KV=1, dh=64, bf16=False, page=64),
    dict(lens=[2, 1, 40, 70], new=[5, 4, 12, 66], H=4, KV=1, dh=32, bf16=False, page=4),       # places below 0
    dict(lens=[2, 1, 40, 70], new=[50, 40, 12, 66], H=4, KV=1, dh=64, bf16=True, page=16),
    dict(lens=[50, 9], new=[8, 9], H=2, KV=1, dh=32, bf16=False, page=4, per_seq=11),          # past the table
    dict(lens=[400, 90], new=[80, 90], H=4, KV=1, dh=64, bf16=True, page=16, per_seq=11, window=33, sinks=2),
    dict(lens=[700, 300, 33], new=[700, 200, 33], H=4, KV=4, dh=64, bf16=True, page=16, q_order="hld"),
]


@pytest.mark.parametrize("kw", CHUNKS, ids=str)
def test_chunks(cuda, kw):
    Op(**kw).run().check()


@pytest.mark.parametrize("kw", [
    # more sequences than lanes, whose tiles are cut by keys
    dict(lens=[2000 - 13 * i for i in range(100)], new=[1 + i % 50 for i in range(100)], H=2, KV=1, dh=64, page=16),
    dict(lens=[2000 - 13 * i for i in range(100)], new=40, H=1, KV=1, dh=32, page=64, window=900, sinks=5),
    dict(lens=[2000 - 13 * i for i in range(100)], new=1, H=2, KV=1, dh=64, page=16),
    # up to 64 rows, in pages of one and two waves' rows
    dict(lens=[6000, 900, 300], new=9, H=5, KV=1, dh=128, page=32),
    dict(lens=[6000, 900, 300], new=[9, 0, 3], H=5, KV=1, dh=64, page=64, window=700, sinks=40),
    dict(lens=[600, 900, 300], new=33, H=1, KV=1, dh=32, page=96, order="heads"),
    dict(lens=[600, 900, 300], new=12, H=4, KV=1, dh=48, page=8),
], ids=str)
@pytest.mark.parametrize("bf16", [True, False])
def test_plans_over_lanes_and_waves(cuda, kw, bf16):
    Op(bf16=bf16, **kw).run().check()


@pytest.mark.parametrize("bf16", [True, False])
def test_a_window_of_every_int(cuda, bf16):
    for window in (2 ** 31 - 1, 2 ** 31 - 200, 2 ** 30):
        Op(lens=[2100, 300], new=[70, 300], H=2, KV=1, dh=64, bf16=bf16, page=16, window=window, sinks=2 ** 31 - 1).run().check()


@pytest.mark.parametrize("new", [1, 70])
def test_no_page_in_a_pool_of_nan(cuda, new):
    """Rows that no page is left for, next to places that hold NaN: zeros and -inf."""
    op = Op(lens=[900, 400, 77], new=new, H=4, KV=2, dh=64, bf16=True, page=32)
    op.table[1] = -1
    op.table[2] = op.kp.shape[0]
    op.kp[op.table[0, -1].long(), 900 % 32:] = float("nan")
    op.run().check()
    assert (op.qv(op.out)[new:] == 0).all() and (op.lse[1:] == -math.inf).all()


def test_many_sequences_of_one_chunk_size(cuda):
    Op(lens=[130 + 3 * i for i in range(90)], new=33, H=4, KV=2, dh=64, bf16=True, page=16).run().check()
    Op(lens=[130 + 3 * i for i in range(90)], new=[1 + i % 40 for i in range(90)], H=4, KV=2, dh=64, bf16=True,
       page=16).run().check()


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("bf16", [True, False])
def test_entries_that_are_no_page(cuda, new, bf16):
    op = Op(lens=[900, 700, 100], new=new, H=4, KV=2, dh=64, bf16=bf16, page=16)
    op.table[0, 3], op.table[0, 40], op.table[1, 0], op.table[1, 43] = -1, op.kp.shape[0], 2 ** 31 - 1, -2 ** 31
    op.table[2] = -1          # no page at all
    op.run().check()
    assert torch.isinf(op.lse[2]).all()


@pytest.mark.parametrize("new", [1, 40])
def test_pages_behind_a_window_may_be_given_back(cuda, new):
    op = Op(lens=[2000, 1000], new=new, H=4, KV=2, dh=128, bf16=True, page=16, window=128, sinks=4)
    gone = [(2000 - new - 128) // 16, (1000 - new - 128) // 16]
    for i in range(2):
        op.table[i, 1:gone[i]] = -1
    op.run().check()


def test_pages_that_sequences_share(cuda):
    op = Op(lens=[600, 650, 620], new=1, H=8, KV=2, dh=128, bf16=True, page=16)
    op.table[1, :20] = op.table[0, :20]
    op.table[2, :20] = op.table[0, :20]
    op.run().check()


def test_no_table_and_no_rows(cuda):
    op = Op(lens=[5, 9], new=[2, 3], H=4, KV=2, dh=64, bf16=True, page=16, per_seq=0)
    op.run().check()
    op = Op(lens=[0, 0], new=[0, 0], H=4, KV=2, dh=64, bf16=True, page=16, slack=2)
    op.run().check()


@pytest.mark.parametrize("kw", [dict(lens=[3000, 700], new=1), dict(lens=[3000, 700], new=[300, 65]),
                                dict(lens=[9000, 700], new=[100, 65])], ids=str)
def test_graph_replays_equal_the_eager_call(cuda, kw):
    op = Op(H=8, KV=2, dh=128, bf16=True, page=16, window=2500, sinks=4, **kw).run().check()
    first, lse = op.out.clone(), op.lse.clone()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        op.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        op.out.fill_(GUARD)
        op.lse.fill_(GUARD)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(op.out, first) and torch.equal(op.lse, lse)
    # longer sequences, the same graph: lengths are the device's
    op.lens[1] = 690
    op.len[1] = 690
    g.replay()
    op.check()


def test_two_calls_at_once_with_scratch_of_their_own(cuda):
    ops = [Op(lens=[5000, 800], new=1, H=8, KV=2, dh=128, bf16=True, page=64, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    for op, s in zip(ops, streams):
        op.run(s.cuda_stream)
    for op in ops:
        op.check()


def test_without_lse_and_with_large_scores(cuda):
    Op(lens=[900], new=1, H=4, KV=2, dh=64, bf16=True, page=16).run(lse=False).check(lse=False)
    Op(lens=[900], new=[70], H=4, KV=2, dh=64, bf16=False, page=16, scale=6.0).run().check()


def test_a_cache_past_32_bit_offsets(cuda):
    pages, page, dh = 17000, 1024, 128        # 2.2e9 elements
    op = Op(lens=[1500, 1030], new=1, H=2, KV=1, dh=dh, bf16=True, page=page)
    big = torch.empty(2, pages, page, 1, dh, dtype=torch.bfloat16, device="cuda")
    for pool, small in ((big[0], op.kp), (big[1], op.vp)):
        for i in range(2):
            for e in range(2):
                pool[pages - 1 - 2 * i - e] = small[op.table[i, e].long()]
    for i in range(2):
        for e in range(2):
            op.table[i, e] = pages - 1 - 2 * i - e
    op.kp, op.vp = big[0], big[1]
    c = op.a.cache
    c.pages, c.kp, c.vp = pages, op.kp.data_ptr(), op.vp.data_ptr()
    op.run().check()
    op2 = Op(lens=[1500, 1030], new=[200, 90], H=2, KV=1, dh=dh, bf16=True, page=page)
    op2.table, op2.kp, op2.vp = op.table, op.kp, op.vp
    op2.a.cache = c
    op2.run().check()


def test_packed_rows_of_sequences_that_could_be_long(cuda):
    """600 sequences of up to 2^17 new rows of 8 heads on one: only the rows that there are count as launched."""
    new = [0] * 590 + [1, 40, 0, 300, 7, 0, 65, 2, 129, 33]
    op = Op(lens=[x + 50 for x in new], new=new, H=8, KV=1, dh=64, bf16=True, page=16, slack=2)
    op.a.lq = 1 << 17
    nb = native.lib().ptcg_kernel_paged_attention_ws_bytes(ctypes.byref(op.a))
    assert nb >= 0
    op.ws = torch.full((max(16, nb),), 0xff, dtype=torch.uint8, device="cuda")
    op.run(lse=False).check(lse=False)
