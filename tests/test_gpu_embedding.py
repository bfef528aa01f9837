"""Embedding lookup with scaling and its gradient by sorted tokens
(ptcg_kernel_embedding_*) against 64 bits."""
import math

import pytest
import torch

from ptcg_amd import native

pytestmark = pytest.mark.gpu

GUARD = 7.25
T = {0: torch.float32, 1: torch.bfloat16}


def _ids(rows, vocab, kind, g):
    if kind == "one":
        return torch.full((rows,), vocab - 1, dtype=torch.int32, device="cuda")
    if kind == "padding":
        return torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    if kind == "ascending":
        return (torch.arange(rows, device="cuda") % vocab).int()
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    ids = ((vocab ** u - 1) if kind == "skewed" else vocab * u).long().clamp(0, vocab - 1).int()
    pad = torch.rand(rows, generator=g, device="cuda")
    ids[pad < 0.1] = -1
    ids[pad > 0.95] = vocab + 3
    return ids


def _fwd(ids, table, vocab, d, scale, out, ldo, stream=None):
    native.check(native.lib().ptcg_kernel_embedding_fwd(
        ids.data_ptr(), ids.numel(), table.data_ptr(), table.stride(0), int(table.dtype == torch.bfloat16), vocab, d,
        scale, out.data_ptr(), ldo, int(out.dtype == torch.bfloat16), stream))


def _bwd(ids, dout, vocab, d, scale, dtable, ws, stream=None):
    native.check(native.lib().ptcg_kernel_embedding_bwd(
        ids.data_ptr(), ids.numel(), dout.data_ptr(), dout.stride(0), int(dout.dtype == torch.bfloat16), vocab, d,
        scale, dtable.data_ptr(), dtable.stride(0), ws.data_ptr(), ws.numel(), stream))


def _ws(rows, vocab, d):
    nb = native.lib().ptcg_kernel_embedding_bwd_ws_bytes(rows, vocab, d)
    assert nb > 0
    return torch.full((nb,), 0xff, dtype=torch.uint8, device="cuda")


def _padded(rows, d, pad, t, fill=None, g=None):
    """A (rows, d) view of wider rows, and the whole."""
    full = torch.randn(max(rows, 1), d + pad, generator=g, device="cuda").to(t) if fill is None else \
        torch.full((max(rows, 1), d + pad), fill, dtype=t, device="cuda")
    return full[:rows, :d], full


def _check_grad(ids, dout, vocab, scale, got):
    """fp32 sums of n terms in any order are off by at most (n + 8) u sum|x|."""
    d = dout.shape[1]
    live = (ids >= 0) & (ids < vocab)
    at = torch.where(live, ids, vocab).long()
    x = dout.double() * scale
    want = torch.zeros(vocab + 1, d, dtype=torch.float64, device="cuda").index_add_(0, at, x)[:vocab]
    mag = torch.zeros(vocab + 1, d, dtype=torch.float64, device="cuda").index_add_(0, at, x.abs())[:vocab]
    cnt = torch.bincount(at, minlength=vocab + 1)[:vocab, None]
    err = (cnt + 8) * 2.0 ** -24 * mag
    assert ((got.double() - want).abs() <= err).all()
    assert (got[cnt[:, 0] == 0] == 0).all()


CASES = [
    # rows, vocab, d, ids
    (1, 1, 1, "uniform"), (1, 5, 8, "padding"), (3, 2048, 256, "uniform"), (64, 7, 64, "one"), (65, 3, 32, "one"),
    (1000, 50, 77, "uniform"), (1024, 2048, 256, "skewed"), (1025, 2049, 256, "skewed"), (5000, 300, 300, "skewed"),
    (3000, 100003, 40, "uniform"), (20000, 2048, 128, "one"), (30011, 9000, 136, "skewed"), (4096, 16, 1024, "uniform"),
    (777, 513, 1500, "ascending"), (5003, 1 << 20, 12, "skewed"), (270000, 700, 16, "skewed"),
    (300000, 5000, 8, "uniform"), (4095, 3000, 20, "skewed"), (4097, 3000, 20, "skewed"), (63, 64, 4, "ascending"),
    (2000, (1 << 31) - 1 >> 9, 4, "uniform"),
]


@pytest.mark.parametrize("tb,ob", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("case", CASES)
def test_lookup_and_gradient(case, tb, ob, cuda):
    rows, vocab, d, kind = case
    print(f"embedding {case} table bf16={tb} out bf16={ob}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    scale = 0.375 if d % 3 else math.sqrt(d)
    ids = _ids(rows, vocab, kind, g)
    table = torch.randn(vocab, d, generator=g, device="cuda").to(T[tb])
    out = torch.full((rows, d), GUARD, dtype=T[ob], device="cuda")
    _fwd(ids, table, vocab, d, scale, out, d)
    # one product and one rounding: the same bits as torch
    live = (ids >= 0) & (ids < vocab)
    s32 = torch.tensor(scale, dtype=torch.float32, device="cuda")
    want = (table.float()[ids.clamp(0, vocab - 1).long()] * s32 * live[:, None]).to(T[ob])
    assert torch.equal(out, want + 0.0) or torch.equal(out.abs(), want.abs())
    dout = torch.randn(rows, d, generator=g, device="cuda").to(T[ob])
    dtable = torch.full((vocab, d), GUARD, device="cuda")
    _bwd(ids, dout, vocab, d, scale, dtable, _ws(rows, vocab, d))
    torch.cuda.synchronize()
    _check_grad(ids, dout, vocab, float(s32), dtable)


@pytest.mark.parametrize("ob", [0, 1])
@pytest.mark.parametrize("d,pad,off", [(64, 8, 0), (64, 3, 0), (64, 8, 1), (20, 4, 4), (33, 0, 0)])
def test_strides_and_alignment(d, pad, off, ob, cuda):
    """Rows of wider matrices, from bases that break the vector forms; what lies
    between the rows stays."""
    g = torch.Generator(device="cuda").manual_seed(d + pad)
    rows, vocab = 700, 90
    ids = _ids(rows, vocab, "skewed", g)
    table = torch.randn(vocab, d + pad + off, generator=g, device="cuda")[:, off:off + d]
    full = torch.full((rows, d + pad + off), GUARD, dtype=T[ob], device="cuda")
    out = full[:, off:off + d]
    _fwd(ids, table, vocab, d, 2.0, out, full.stride(0))
    live = (ids >= 0) & (ids < vocab)
    want = (table[ids.clamp(0, vocab - 1).long()] * 2.0 * live[:, None]).to(T[ob])
    assert torch.equal(out.abs(), want.abs())
    assert (full[:, :off] == GUARD).all() and (full[:, off + d:] == GUARD).all()
    dout = torch.randn(rows, d + pad + off, generator=g, device="cuda").to(T[ob])[:, off:off + d]
    gfull = torch.full((vocab, d + pad + off), GUARD, device="cuda")
    _bwd(ids, dout, vocab, d, 2.0, gfull[:, off:off + d], _ws(rows, vocab, d))
    torch.cuda.synchronize()
    _check_grad(ids, dout, vocab, 2.0, gfull[:, off:off + d])
    assert (gfull[:, :off] == GUARD).all() and (gfull[:, off + d:] == GUARD).all()


def test_no_tokens_clear_the_gradient(cuda):
    dtable = torch.full((300, 24), GUARD, device="cuda")
    ws = _ws(0, 300, 24)
    native.check(native.lib().ptcg_kernel_embedding_bwd(None, 0, None, 24, 0, 300, 24, 1.0, dtable.data_ptr(), 24,
                                                        ws.data_ptr(), ws.numel(), None))
    torch.cuda.synchronize()
    assert (dtable == 0).all()


def test_nan_of_padding_tokens_and_of_one_id(cuda):
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 40, (500,), generator=g, device="cuda").int()
    ids[10:20] = -1
    ids[100] = 7
    dout = torch.randn(500, 64, generator=g, device="cuda")
    dout[10:20] = math.nan
    dout[100, 3] = math.inf
    dtable = torch.empty(40, 64, device="cuda")
    _bwd(ids, dout, 40, 64, 1.0, dtable, _ws(500, 40, 64))
    torch.cuda.synchronize()
    assert dtable[7, 3] == math.inf
    dtable[7, 3] = 0.0
    assert dtable.isfinite().all()


@pytest.mark.parametrize("rows,vocab,kind", [(50000, 2048, "skewed"), (40000, 30000, "skewed"), (3000, 5, "uniform")])
def test_repeats_bit_for_bit(rows, vocab, kind, cuda):
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = _ids(rows, vocab, kind, g)
    dout = torch.randn(rows, 64, generator=g, device="cuda")
    got = []
    for _ in range(3):
        dtable = torch.empty(vocab, 64, device="cuda")
        _bwd(ids, dout, vocab, 64, 1.5, dtable, _ws(rows, vocab, 64))
        got.append(dtable)
    torch.cuda.synchronize()
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_captured_and_replayed(cuda):
    g = torch.Generator(device="cuda").manual_seed(6)
    rows, vocab, d = 9000, 5000, 96
    ids = _ids(rows, vocab, "skewed", g)
    table, dout = torch.randn(vocab, d, generator=g, device="cuda"), torch.randn(rows, d, generator=g, device="cuda")
    out, dtable, ws = torch.empty(rows, d, device="cuda"), torch.empty(vocab, d, device="cuda"), _ws(rows, vocab, d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        _fwd(ids, table, vocab, d, 1.0, out, d, st)
        _bwd(ids, dout, vocab, d, 1.0, dtable, ws, st)
    for k in range(3):
        ids.copy_(_ids(rows, vocab, "uniform" if k == 1 else "skewed", g))     # other tokens, other runs
        graph.replay()
        torch.cuda.synchronize()
        got = (out.clone(), dtable.clone())
        _fwd(ids, table, vocab, d, 1.0, out, d)
        _bwd(ids, dout, vocab, d, 1.0, dtable, ws)
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], dtable), f"replay {k}"
        _check_grad(ids, dout, vocab, 1.0, dtable)


def test_gradient_against_differences(cuda):
    """The lookup is linear in the table: a difference along a direction is the
    gradient's product with it but for rounding (each fp32 output and the sums:
    u (|L+| + |L-|) / h per term)."""
    g = torch.Generator(device="cuda").manual_seed(8)
    rows, vocab, d, h = 400, 60, 32, 0.5
    ids = _ids(rows, vocab, "skewed", g)
    table, dout = torch.randn(vocab, d, generator=g, device="cuda"), torch.randn(rows, d, generator=g, device="cuda")
    dirn = torch.randn(vocab, d, generator=g, device="cuda")
    dtable, out = torch.empty(vocab, d, device="cuda"), torch.empty(rows, d, device="cuda")
    _bwd(ids, dout, vocab, d, 3.0, dtable, _ws(rows, vocab, d))
    loss, mag = [], 0.0
    for sgn in (1, -1):
        _fwd(ids, table + sgn * h * dirn, vocab, d, 3.0, out, d)
        torch.cuda.synchronize()
        loss.append(float((out.double() * dout.double()).sum()))
        mag += float((out.double() * dout.double()).abs().sum())
    want = float((dtable.double() * dirn.double()).sum())
    slack = float((dtable.double() * dirn.double()).abs().sum())
    assert abs((loss[0] - loss[1]) / (2 * h) - want) <= 2.0 ** -24 * (3 * mag / (2 * h) + rows * slack)


def _check_lookup(ids, table, vocab, scale, out):
    """One product and one rounding: torch's bits, signs among them (zeros of either sign are equal)."""
    live = (ids >= 0) & (ids < vocab)
    rows = table.float()[ids.clamp(0, vocab - 1).long()]
    assert torch.equal(out, torch.where(live[:, None], rows * scale, 0.0).to(out.dtype))


@pytest.mark.parametrize("tb,ob", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("d,pad,off", [(1, 0, 0), (64, 0, 0), (64, 3, 0), (77, 0, 0), (256, 8, 1), (1500, 4, 4)])
def test_lookup_keeps_signs(d, pad, off, tb, ob, cuda):
    g = torch.Generator(device="cuda").manual_seed(d + pad)
    rows, vocab = 333, 50
    ids = _ids(rows, vocab, "uniform", g)
    table = torch.randn(vocab, d + pad + off, generator=g, device="cuda").to(T[tb])[:, off:off + d]
    full = torch.full((rows, d + pad + off), GUARD, dtype=T[ob], device="cuda")
    for scale in (1.5, -0.375):
        _fwd(ids, table, vocab, d, scale, full[:, off:off + d], full.stride(0))
        torch.cuda.synchronize()
        _check_lookup(ids, table, vocab, scale, full[:, off:off + d])


@pytest.mark.parametrize("ob", [0, 1])
@pytest.mark.parametrize("rows,vocab,d,kind", [
    # few counts, scanned within the placement, with two and with four batches a wave in flight
    (99999, 40, 16, "skewed"), (100000, 60, 4, "uniform"), (100001, 40, 16, "skewed"), (120001, 3000, 8, "uniform"),
    (131000, 4096, 4, "skewed"),
    # tiles of more than 1 024 tokens, whose waves load their keys anew
    (1048576, 700, 4, "skewed"), (1048577, 700, 4, "skewed"), (1200007, 5, 4, "uniform"), (1200007, 5000, 4, "skewed"),
    (2100001, 60, 4, "skewed"), (1200007, 100003, 4, "uniform"),
])
def test_gradient_of_every_sort_shape(rows, vocab, d, kind, ob, cuda):
    print(f"embedding gradient {rows} x {d} of {vocab} {kind} bf16={ob}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    ids = _ids(rows, vocab, kind, g)
    dout = torch.randn(rows, d, generator=g, device="cuda").to(T[ob])
    dtable = torch.full((vocab, d), GUARD, device="cuda")
    _bwd(ids, dout, vocab, d, 0.5, dtable, _ws(rows, vocab, d))
    torch.cuda.synchronize()
    # as _check_grad, on the host, where a million tokens of few ids do not queue
    ids, x, got = ids.cpu().long(), dout.double().cpu() * 0.5, dtable.double().cpu()
    at = torch.where((ids >= 0) & (ids < vocab), ids, vocab)
    zeros = torch.zeros(vocab + 1, d, dtype=torch.float64)
    want, mag = zeros.index_add(0, at, x)[:vocab], zeros.index_add(0, at, x.abs())[:vocab]
    cnt = torch.bincount(at, minlength=vocab + 1)[:vocab, None]
    assert ((got - want).abs() <= (cnt + 8) * 2.0 ** -24 * mag).all()
    assert (got[cnt[:, 0] == 0] == 0).all()


def _in_token_order(ids, dout, vocab, scale, most):
    """scale * (((0 + dout[t0]) + dout[t1]) + ...) in fp32 over the first `most` of each id's tokens."""
    live = torch.nonzero((ids >= 0) & (ids < vocab))[:, 0]
    order = live[torch.argsort(ids[live].long(), stable=True)]
    key = ids[order].long()
    first = torch.searchsorted(key, torch.arange(vocab, device="cuda"))
    nth = torch.arange(order.numel(), device="cuda") - first[key]
    s = torch.zeros(vocab, dout.shape[1], device="cuda")
    for k in range(most):
        sel = nth == k
        s[key[sel]] += dout[order[sel]].float()
    return s * scale


COUNTS = [1, 2, 31, 32, 33, 39, 40, 41, 42, 63, 64, 65, 40, 96, 97, 41, 7, 128, 40, 0, 41, 300, 40, 129]


@pytest.mark.parametrize("ob", [0, 1])
@pytest.mark.parametrize("d", [12, 136, 520])
@pytest.mark.parametrize("stride,fill", [(1, 0), (1, 4500), (4001, 0), (4001, 4500)])   # ids apart; tokens of the last id
def test_runs_around_the_lengths_that_are_cut(stride, fill, d, ob, cuda):
    """Ids of 1 to 300 tokens, around 40 (the longest added in line) and multiples
    of 32 (the pieces of longer ones), at every start within a piece: up to 40
    tokens the sum is in token order, to the bit, wherever the run lies."""
    n = len(COUNTS)
    vocab = (n + 1) * stride + 1
    for lead in (0, 1, 8, 23, 31, 32):
        g = torch.Generator(device="cuda").manual_seed(lead + d)
        counts = [lead] + COUNTS + [fill]
        ids = torch.cat([torch.full((c,), min(i * stride, vocab - 1), dtype=torch.int32) for i, c in enumerate(counts)])
        ids = torch.cat([ids, torch.tensor([-1, vocab], dtype=torch.int32)]).cuda()
        ids = ids[torch.randperm(ids.numel(), generator=g, device="cuda")].contiguous()
        dout = torch.randn(ids.numel(), d, generator=g, device="cuda").to(T[ob])
        dtable = torch.full((vocab, d), GUARD, device="cuda")
        _bwd(ids, dout, vocab, d, 1.25, dtable, _ws(ids.numel(), vocab, d))
        torch.cuda.synchronize()
        _check_grad(ids, dout, vocab, 1.25, dtable)
        short = torch.bincount(ids[(ids >= 0) & (ids < vocab)].long(), minlength=vocab) <= 40
        assert torch.equal(dtable[short], _in_token_order(ids, dout, vocab, 1.25, 40)[short]), f"lead {lead}"
