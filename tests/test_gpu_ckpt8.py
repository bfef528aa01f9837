"""Activation checkpoints in 8 bits (ptcg_kernel_ckpt8_*): the stored form bit
for bit, the GELU backward and the weight gradient against 64 bits."""
import math

import pytest
import torch

from ptcg_amd import native

pytestmark = pytest.mark.gpu

GUARD = 7.25
T = {0: torch.float32, 1: torch.bfloat16}
U = 2.0 ** -24


def _groups(d):
    return -(-d // 32)


def store64(x):
    """Scales and kept values by the definition, in 64 bits (finite x)."""
    rows, d = x.shape
    y = torch.zeros(rows, _groups(d) * 32, dtype=torch.float64, device=x.device)
    y[:, :d] = x.double()
    y = y.view(rows, -1, 32)
    top = y.abs().amax(2)
    e = torch.full_like(top, -110.0)
    for k in range(-110, 120):     # the least e with top <= 448 2^e
        e = torch.where((top > 448.0 * 2.0 ** (k - 1)) & (k > -110), float(k), e)
    v = (y * torch.exp2(-e)[..., None]).clamp(-448, 448)
    mant = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    mant = torch.where(torch.exp2(mant) > v.abs().clamp(min=2.0 ** -6), mant - 1, mant)
    step = torch.exp2(mant - 3)
    kept = torch.round(v / step) * step * torch.exp2(e)[..., None]
    return e.int(), kept.view(rows, -1)[:, :d]


def values64(q, sc):
    """What codes and scale bytes stand for."""
    d = q.shape[1]
    w = torch.exp2(sc.double() - 127).repeat_interleave(32, 1)[:, :d]
    return q.contiguous().view(torch.float8_e4m3fn).double() * w


def _pack(x, q, sc, d, stream=None):
    native.check(native.lib().ptcg_kernel_ckpt8_pack(x.data_ptr(), x.stride(0), int(x.dtype == torch.bfloat16),
                                                     x.shape[0], d, q.data_ptr(), q.stride(0), sc.data_ptr(),
                                                     sc.stride(0), stream))


def _unpack(q, sc, d, x, stream=None):
    native.check(native.lib().ptcg_kernel_ckpt8_unpack(q.data_ptr(), q.stride(0), sc.data_ptr(), sc.stride(0),
                                                       x.shape[0], d, x.data_ptr(), x.stride(0),
                                                       int(x.dtype == torch.bfloat16), stream))


def _new(rows, d, pad=0):
    return (torch.full((rows, d + pad), 0xaa, dtype=torch.uint8, device="cuda"),
            torch.full((rows, _groups(d) + pad), 0xaa, dtype=torch.uint8, device="cuda"))


def _random(rows, d, g, spread=1.0):
    return torch.randn(rows, d, generator=g, device="cuda") * torch.exp(spread * torch.randn(rows, 1, generator=g,
                                                                                              device="cuda"))


SIZES = [(1, 1), (1, 8), (3, 31), (5, 32), (7, 33), (300, 256), (65, 634), (17, 1024), (1000, 40), (2, 4100)]


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("pad", [0, 8, 5])
def test_store_and_restore(rows, d, pad, bf16, cuda):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + d)
    x = _random(rows, d + pad, g, 3.0).to(T[bf16])[:, :d]
    q, sc = _new(rows, d, pad)
    _pack(x, q[:, :d], sc[:, :_groups(d)], d)
    full = torch.full((rows, d + pad), GUARD, dtype=T[bf16], device="cuda")
    _unpack(q[:, :d], sc[:, :_groups(d)], d, full[:, :d])
    torch.cuda.synchronize()
    e, kept = store64(x)
    assert torch.equal(sc[:, :_groups(d)].int() - 127, e)
    assert torch.equal(values64(q[:, :d], sc[:, :_groups(d)]), kept)
    assert torch.equal(full[:, :d].double(), kept)
    assert (q[:, d:] == 0xaa).all() and (sc[:, _groups(d):] == 0xaa).all() and (full[:, d:] == GUARD).all()


def test_edges_of_the_stored_form(cuda):
    """Zeros, the borders of the scale rule, ties, the scale's two ends, and
    values that are not finite."""
    vals = [[0.0], [448.0], [math.nextafter(448.0, 1e9)], [449.0], [1.75], [1.7500001], [2.0 ** -149],
            [2.0 ** -110 * 3], [2.0 ** 127 * 1.99], [448 * 2.0 ** 119], [448 * 2.0 ** 119 * 1.1],
            [256.0, 17.0, 19.0, -17.0, -19.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9 * 1.5],
            [300.0, 0.0155, 0.0157, 2.0 ** -7, -0.0]]
    x = torch.zeros(len(vals), 32, device="cuda")
    for i, v in enumerate(vals):
        x[i, :len(v)] = torch.tensor(v, dtype=torch.float64).float()
    q, sc = _new(len(vals), 32)
    _pack(x, q, sc, 32)
    out = torch.empty_like(x)
    _unpack(q, sc, 32, out)
    torch.cuda.synchronize()
    e, kept = store64(x)
    assert torch.equal(sc.int() - 127, e)
    assert torch.equal(out.double(), kept) and torch.equal(values64(q, sc), kept)
    x = torch.randn(4, 64, device="cuda")
    want = store64(x.clone().index_fill_(0, torch.tensor([1, 2], device="cuda"), 0.0))
    x[1], x[2] = math.nan, -math.inf
    x[3, 5], x[3, 40] = math.nan, math.inf
    clean = x.nan_to_num(0.0, 0.0, 0.0)
    e, kept = store64(clean)
    q, sc = _new(4, 64)
    out = torch.empty_like(x)
    _pack(x, q, sc, 64)
    _unpack(q, sc, 64, out)
    torch.cuda.synchronize()
    bad = ~x.isfinite()
    assert out[bad].isnan().all() and torch.equal(out[~bad].double(), kept[~bad]) and torch.equal(sc.int() - 127, e)
    assert torch.equal(e[0], want[0][0])


def _gelu64(z):
    cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("pad,act", [(0, True), (3, True), (8, False)])
def test_gelu_backward(rows, d, pad, act, bf16, cuda):
    """The erf behind both is off by at most 1.5e-7 (Abramowitz & Stegun
    7.1.26), halved in the distribution; its fp32 evaluation adds a few units of
    2^-24 of values up to 1 + |z|; then one rounding to the stored type."""
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    x = _random(rows, d, g) * 2
    q, sc = _new(rows, d, pad)
    q, sc = q[:, :d], sc[:, :_groups(d)]
    _pack(x, q, sc, d)
    dy = torch.randn(rows, d + pad, generator=g, device="cuda").to(T[bf16])[:, :d]
    dz = torch.full((rows, d + pad), GUARD, dtype=T[bf16], device="cuda")
    a = torch.full((rows, d + pad), GUARD, dtype=T[bf16], device="cuda")
    native.check(native.lib().ptcg_kernel_ckpt8_gelu_bwd(
        q.data_ptr(), q.stride(0), sc.data_ptr(), sc.stride(0), rows, d, dy.data_ptr(), dy.stride(0), dz.data_ptr(),
        d + pad, a.data_ptr() if act else None, d + pad, bf16, None))
    torch.cuda.synchronize()
    z = values64(q, sc)
    want_a, grad = _gelu64(z)
    b = torch.finfo(T[bf16]).eps / 2
    tol = 0.75e-7 + 16 * U
    assert ((a[:, :d].double() - want_a).abs() <= tol * z.abs() + b * want_a.abs() + 1e-37).all() if act else \
        (a == GUARD).all()
    want = dy.double() * grad
    assert ((dz[:, :d].double() - want).abs() <= dy.double().abs() * tol * (1 + z.abs().clamp(max=15))
            + (b + 4 * U) * want.abs() + 1e-37).all()
    assert (dz[:, d:] == GUARD).all()


def test_gelu_backward_in_place(cuda):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(100, 256, generator=g, device="cuda")
    q, sc = _new(100, 256)
    _pack(x, q, sc, 256)
    dy = torch.randn(100, 256, generator=g, device="cuda")
    dz = torch.empty_like(dy)
    L = native.lib()
    for y, z in ((dy, dz), (dy, dy)):
        native.check(L.ptcg_kernel_ckpt8_gelu_bwd(q.data_ptr(), 256, sc.data_ptr(), 8, 100, 256, y.data_ptr(), 256,
                                                  z.data_ptr(), 256, None, 0, 0, None))
    torch.cuda.synchronize()
    assert torch.equal(dz, dy)


def _dw(rows, k, n, dy, q, sc, dW, db, ws, stream=None):
    native.check(native.lib().ptcg_kernel_ckpt8_dw(
        rows, k, n, dy.data_ptr() if rows else None, dy.stride(0) if rows else n, int(dy.dtype == torch.bfloat16),
        q.data_ptr() if rows else None, q.stride(0) if rows else k, sc.data_ptr() if rows else None,
        sc.stride(0) if rows else _groups(k), dW.data_ptr(), None if db is None else db.data_ptr(), ws.data_ptr(),
        ws.numel(), stream))


def _ws(rows, k, n, bf16):
    nb = native.lib().ptcg_kernel_ckpt8_dw_ws_bytes(rows, k, n, bf16)
    assert nb >= 0
    return torch.full((max(nb, 16),), 0xff, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("rows,k,n,pad", [
    (1, 1, 1, 0), (5, 33, 7, 0), (32, 128, 128, 0), (33, 130, 129, 3), (1000, 256, 64, 0), (700, 634, 136, 0),
    (2047, 200, 300, 8), (9000, 128, 128, 0), (513, 1024, 256, 0), (40, 256, 1024, 0), (4000, 40, 24, 16),
    (100003, 64, 32, 0), (300, 520, 264, 0), (36001, 1100, 1040, 0), (36001, 1088, 1032, 5),
])
def test_weight_gradient(rows, k, n, pad, bf16, cuda):
    """Each product is exact (bf16 terms) and sums of m of them are fp32: off by
    at most (m + 8) u sum|dy||x8|, m the row count (three terms each in fp32),
    whatever the order."""
    print(f"ckpt8_dw rows={rows} k={k} n={n} pad={pad} bf16={bf16}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    q, sc = _new(rows, k, pad)
    q, sc = q[:, :k], sc[:, :_groups(k)]
    _pack(_random(rows, k, g, 2.0), q, sc, k)
    dy = (torch.randn(rows, n + pad, generator=g, device="cuda") * 1e-3).to(T[bf16])[:, :n]
    dW, db = torch.full((n, k), GUARD, device="cuda"), torch.full((n,), GUARD, device="cuda")
    _dw(rows, k, n, dy, q, sc, dW, db, _ws(rows, k, n, bf16))
    torch.cuda.synchronize()
    x8, y = values64(q, sc), dy.double()
    m = (1 if bf16 else 3) * rows
    assert ((dW.double() - y.t() @ x8).abs() <= (m + 8) * U * (y.abs().t() @ x8.abs()) + 1e-37).all()
    assert ((db.double() - y.sum(0)).abs() <= (rows + 8) * U * y.abs().sum(0)).all()
    # without the bias gradient, and bit for bit again
    w2 = torch.empty_like(dW)
    _dw(rows, k, n, dy, q, sc, w2, None, _ws(rows, k, n, bf16))
    torch.cuda.synchronize()
    assert torch.equal(dW, w2)


@pytest.mark.parametrize("bf16", [0, 1])
def test_weight_gradient_is_tight_on_average(bf16, cuda):
    """Random signs: the error in the 2-norm stays within the random walk of the
    fp32 sums, sqrt(m) u (twice, for the accumulation order), not just the worst
    case."""
    g = torch.Generator(device="cuda").manual_seed(3)
    rows, k, n = 20000, 256, 256
    q, sc = _new(rows, k)
    _pack(torch.randn(rows, k, generator=g, device="cuda"), q, sc, k)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(T[bf16])
    dW, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    _dw(rows, k, n, dy, q, sc, dW, db, _ws(rows, k, n, bf16))
    torch.cuda.synchronize()
    want = dy.double().t() @ values64(q, sc)
    assert float((dW.double() - want).norm() / want.norm()) <= 2 * math.sqrt(rows) * U


def test_no_rows_clear_the_weight_gradient(cuda):
    dW, db = torch.full((64, 96), GUARD, device="cuda"), torch.full((64,), GUARD, device="cuda")
    e = torch.empty(0, 96, device="cuda")
    _dw(0, 96, 64, e, e, e, dW, db, _ws(0, 96, 64, 0))
    torch.cuda.synchronize()
    assert (dW == 0).all() and (db == 0).all()


def test_captured_and_replayed(cuda):
    g = torch.Generator(device="cuda").manual_seed(4)
    rows, k, n = 3000, 256, 200
    x, dy = torch.randn(rows, k, generator=g, device="cuda"), torch.randn(rows, n, generator=g, device="cuda")
    q, sc = _new(rows, k)
    dW, db, ws = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda"), _ws(rows, k, n, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        _pack(x, q, sc, k, st)
        _dw(rows, k, n, dy, q, sc, dW, db, ws, st)
    for i in range(3):
        x.copy_(torch.randn(rows, k, generator=g, device="cuda") * 2.0 ** i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, sc, dW, db)]
        _pack(x, q, sc, k)
        _dw(rows, k, n, dy, q, sc, dW, db, ws)
        torch.cuda.synchronize()
        for a, b in zip(got, (q, sc, dW, db)):
            assert torch.equal(a, b), f"replay {i}"
