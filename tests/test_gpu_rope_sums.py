"""Gradients of the norm's weights as exact sums: a row lost or taken twice shows.

x is 1 or -1 and dh a power of two, so the mean of x^2 is 1 without rounding, and with
eps = 0 the root is 1 (the forward in fp32 shows it: x itself comes out).  At position 0
nothing turns.  dy is x times 1, 2 or 4: every product is one of these, every sum of them
in whatever order a whole number, and below 2^24 exact in fp32.  Each row adds 1 or more
to each of its columns."""
import pytest
import torch

from test_gpu_rope import Op

pytestmark = pytest.mark.gpu

# n, l, H, KV, dh, bf16, order, off.  The backward launches four workgroups a CU at most (1 024), of 256 lanes over a row's
# (a power of two for each head) and its groups: the longer ones walk.
CASES = [
    (1, 1, 1, 1, 64, False, "lhd", 0),
    (40, 97, 4, 4, 64, False, "lhd", 0),
    (512, 97, 4, 4, 64, False, "lhd", 0),
    (1, 9000, 2, 1, 32, True, "lhd", 0),
    (1, 1201, 16, 4, 128, True, "lhd", 0),
    (1, 65539, 8, 2, 128, True, "hld", 0),
    (1, 5003, 1, 0, 128, False, "lhd", 1),
    (1, 2049, 33, 7, 64, True, "lhd", 3),
    (3, 30011, 1, 1, 8, False, "lhd", 0),
    (1, 100003, 3, 2, 2, True, "lhd", 0),
    (7, 4099, 5, 3, 16, False, "hld", 2),
]


@pytest.mark.parametrize("n,l,H,KV,dh,bf16,order,off", CASES)
def test_weight_gradients_are_exact_sums_of_whole_numbers(cuda, n, l, H, KV, dh, bf16, order, off):
    op = Op(n, l, H, KV, dh, dh, False, bf16, "qk", None, order, off)
    g = torch.Generator(device="cuda").manual_seed(n + l + dh)
    pos = torch.zeros(n * l, dtype=torch.int32, device="cuda")
    op.a.rope.pos, op.a.eps = pos.data_ptr(), 0.0
    want = {}
    for name, x, dy, h in (("q", op.q, op.dqo, H), ("k", op.k, op.dko, KV)):
        x.copy_(2.0 * torch.randint(0, 2, (n * l, h, dh), generator=g, device="cuda") - 1)
        times = 2.0 ** torch.randint(0, 3, (n * l, h, dh), generator=g, device="cuda")
        dy.copy_(x.float() * times)
        want[name] = times.double().sum((0, 1))
        assert want[name].numel() == 0 or float(want[name].max()) < 2 ** 24
    for w in (op.wq, op.wk):
        if w is not None:
            w.fill_(1.0)
    op.fwd()
    op.bwd()
    torch.cuda.synchronize()
    assert torch.equal(op.qo, op.q) and torch.equal(op.ko, op.k)
    assert torch.equal(op.dwq.double(), want["q"])
    if KV:
        assert torch.equal(op.dwk.double(), want["k"])
