"""What the cross-attention, embedding and 8-bit checkpoint entry points refuse
before anything reaches a device (the checks run on the host alone)."""
import ctypes

import pytest

from ptcg_amd import native

P = 4096          # a 16-byte aligned address nothing reads


def _desc(**kw):
    a = native.CPtcgCrossAttn(n=2, lq=8, lk=16, heads=4, kv_heads=2, dh=32, bf16=0, scale=0.5)
    for name, h, l in (("q", 4, 8), ("k", 2, 16), ("v", 2, 16), ("o", 4, 8)):
        setattr(a, name, native.CPtcgHeadLayout(sn=l * h * 32, sl=h * 32, sh=32))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _fwd(a, q=P, k=P, v=P, out=P, ws=None, nb=0):
    return native.check(native.lib().ptcg_kernel_cross_attention_fwd(ctypes.byref(a), q, k, v, out, None, ws, nb, None))


def _bwd(a, q=P, k=P, v=P, out=P, lse=P, dout=P, dq=P, dk=P, dv=P, ws=P, nb=1 << 20):
    return native.check(native.lib().ptcg_kernel_cross_attention_bwd(ctypes.byref(a), q, k, v, out, lse, dout, dq, dk,
                                                                     dv, ws, nb, None))


LAY = native.CPtcgHeadLayout


@pytest.mark.parametrize("kw,match", [
    (dict(n=-1), "negative size"), (dict(lk=-5), "negative size"),
    (dict(heads=3), "kv heads"), (dict(kv_heads=0), "kv heads"),
    (dict(dh=12), "head width"), (dict(dh=136), "head width"), (dict(dh=0), "head width"),
    (dict(bf16=2), "bf16"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(k=LAY(sn=-4, sl=64, sh=32)), "strides"), (dict(q=LAY(sn=1024, sl=130, sh=32)), "strides"),
    (dict(bf16=1, v=LAY(sn=1024, sl=68, sh=32)), "strides"),
    (dict(k_off=P, k_len=P), "k_len"),
    (dict(lq=1 << 30), "too long"), (dict(lk=1 << 30), "too long"), (dict(n=1 << 28, lk=1 << 20), "too many"),
    (dict(o=LAY(sn=0, sl=128, sh=32)), "overlap"), (dict(o=LAY(sn=1024, sl=64, sh=32)), "overlap"),
    (dict(o=LAY(sn=1024, sl=128, sh=16)), "overlap"),
])
def test_cross_attention_refuses(kw, match):
    with pytest.raises(native.PtcgError, match=match):
        _fwd(_desc(**kw))


def test_cross_attention_refuses_buffers():
    L = native.lib()
    assert L.ptcg_kernel_cross_attention_ws_bytes(ctypes.byref(_desc(dh=7)), 0) == -1
    with pytest.raises(native.PtcgError, match="null descriptor"):
        native.check(L.ptcg_kernel_cross_attention_fwd(None, P, P, P, P, None, None, 0, None))
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _fwd(_desc(), **kw)
    with pytest.raises(native.PtcgError, match="16 B aligned"):
        _fwd(_desc(), v=P + 8)
    # a single token against many keys splits them and needs scratch
    a = _desc(lq=1, lk=100000)
    need = L.ptcg_kernel_cross_attention_ws_bytes(ctypes.byref(a), 0)
    assert need > 0
    for ws, nb in ((None, need), (P, need - 1), (P + 8, need)):
        with pytest.raises(native.PtcgError, match="workspace"):
            _fwd(a, ws=ws, nb=nb)
    for kw in (dict(lse=None), dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(out=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _bwd(_desc(), **kw)
    with pytest.raises(native.PtcgError, match="workspace"):
        _bwd(_desc(), nb=4)
    with pytest.raises(native.PtcgError, match="dq overlap"):
        _bwd(_desc(q=LAY(sn=0, sl=128, sh=32)))
    for name in ("k", "v"):
        with pytest.raises(native.PtcgError, match="dk or dv overlap"):
            _bwd(_desc(**{name: LAY(sn=0, sl=64, sh=32)}))


def test_cross_attention_of_nothing_is_done():
    _fwd(_desc(n=0), q=None, k=None, v=None, out=None)
    _fwd(_desc(lq=0), q=None, k=None, v=None, out=None)
    _bwd(_desc(n=0), *[None] * 9, ws=None, nb=0)
