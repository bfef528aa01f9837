"""Frequencies of the position rotation (host), and what the rotation's entry points refuse (host alone)."""
import ctypes

import pytest

from ptcg_amd import native
from refseq import frequencies

P = 4096          # an aligned address nothing reads
LAY = native.CPtcgHeadLayout


def _freq(rot, base=10000.0, scaling=0, factor=8.0, length=4096.0, fast=32.0, slow=1.0):
    f, mag = (ctypes.c_double * max(1, rot // 2))(), ctypes.c_float(-1)
    native.check(native.lib().ptcg_rope_frequencies(rot, base, scaling, factor, length, fast, slow, f, ctypes.byref(mag)))
    return list(f)[:rot // 2], mag.value


@pytest.mark.parametrize("rot", [0, 2, 4, 64, 128])
@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
@pytest.mark.parametrize("factor", [1.0, 8.0, 40.5])
def test_frequencies(rot, scaling, factor):
    got, mag = _freq(rot, scaling=scaling, factor=factor)
    want, wmag = frequencies(rot, scaling=scaling, factor=factor) if rot else ([], None)
    assert len(got) == len(want) and all(abs(a - b) <= 1e-14 * b for a, b in zip(got, want))
    if rot:
        assert abs(mag - wmag) <= 2.0 ** -24 * wmag


def test_by_parts_keeps_fast_pairs_and_divides_slow_ones():
    base, _ = _freq(128)
    got, _ = _freq(128, scaling=3)
    assert got[0] == base[0] and abs(got[-1] - base[-1] / 8) < 1e-18


@pytest.mark.parametrize("kw,match", [
    (dict(rot=3), "turning"), (dict(rot=-2), "turning"), (dict(rot=4, base=1.0), "base"),
    (dict(rot=4, base=float("nan")), "base"), (dict(rot=4, scaling=4), "scaling"), (dict(rot=4, scaling=-1), "scaling"),
    (dict(rot=4, scaling=1, factor=0.5), "factor"), (dict(rot=4, scaling=2, factor=float("inf")), "factor"),
    (dict(rot=4, scaling=3, length=0.0), "by parts"), (dict(rot=4, scaling=3, fast=1.0), "by parts"),
    (dict(rot=4, scaling=3, slow=-1.0), "by parts"),
])
def test_frequencies_refuse(kw, match):
    with pytest.raises(native.PtcgError, match=match):
        _freq(**kw)


def _rope(**kw):
    return native.CPtcgRope(**{**dict(rot=32, interleaved=0, mag=1.0, freq=P, pos=None), **kw})


def _qk(**kw):
    lay = lambda h: LAY(sn=8 * h * 32, sl=h * 32, sh=32)
    a = native.CPtcgQkRope(n=2, l=8, heads=4, kv_heads=2, dh=32, bf16=0, eps=1e-6, q=lay(4), k=lay(2), qo=lay(4),
                           ko=lay(2), wq=P, wk=P, rope=_rope())
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _fwd(a, q=P, k=P, qo=2 * P, ko=2 * P):
    return native.check(native.lib().ptcg_kernel_qk_norm_rope_fwd(ctypes.byref(a), q, k, qo, ko, None))


def _bwd(a, q=P, k=P, dqo=P, dko=P, dq=P, dk=P, dwq=P, dwk=P, ws=P, nb=1 << 30):
    return native.check(native.lib().ptcg_kernel_qk_norm_rope_bwd(ctypes.byref(a), q, k, dqo, dko, dq, dk, dwq, dwk, ws, nb,
                                                                  None))


BAD = [
    (dict(n=-1), "negative size"), (dict(n=1 << 20, l=1 << 20), "too many rows"), (dict(heads=0), "heads"),
    (dict(kv_heads=-1), "heads"), (dict(dh=0), "head width"), (dict(dh=33), "head width"), (dict(dh=130), "head width"),
    (dict(bf16=2), "bf16"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(rope=_rope(rot=34)), "turning"), (dict(rope=_rope(rot=7)), "turning"), (dict(rope=_rope(rot=-2)), "turning"),
    (dict(rope=_rope(interleaved=2)), "interleaved"), (dict(rope=_rope(freq=None)), "frequencies"),
    (dict(rope=_rope(mag=float("inf"))), "mag"), (dict(q=LAY(sn=-1, sl=128, sh=32)), "negative stride"),
    (dict(ko=LAY(sn=512, sl=64, sh=-32)), "negative stride"),
]


@pytest.mark.parametrize("kw,match", BAD)
def test_norm_rope_refuses(kw, match):
    for call in (_fwd, _bwd):
        with pytest.raises(native.PtcgError, match=match):
            call(_qk(**kw))
    assert native.lib().ptcg_kernel_qk_norm_rope_bwd_ws_bytes(ctypes.byref(_qk(**kw))) == -1


def test_norm_rope_refuses_buffers():
    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _fwd(_qk(), **kw)
    with pytest.raises(native.PtcgError, match="alignment"):
        _fwd(_qk(), q=P + 2)
    for kw, match in ((dict(qo=LAY(sn=0, sl=128, sh=32)), "qo overlap"), (dict(ko=LAY(sn=512, sl=32, sh=32)), "ko overlap")):
        with pytest.raises(native.PtcgError, match=match):
            _fwd(_qk(**kw))
    with pytest.raises(native.PtcgError, match="in place"):
        _fwd(_qk(q=LAY(sn=2048, sl=256, sh=32)), qo=P)
    for kw in (dict(q=None), dict(k=None), dict(dqo=None), dict(dko=None), dict(dq=None), dict(dk=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _bwd(_qk(), **kw)
    for kw in (dict(ws=None), dict(nb=16), dict(ws=P + 8)):
        with pytest.raises(native.PtcgError, match="workspace"):
            _bwd(_qk(), **kw)
    with pytest.raises(native.PtcgError, match="without its weight"):
        _bwd(_qk(wq=None))
    with pytest.raises(native.PtcgError, match="dq overlap"):
        _bwd(_qk(q=LAY(sn=1024, sl=128, sh=0)))
    with pytest.raises(native.PtcgError, match="dk overlap"):
        _bwd(_qk(k=LAY(sn=0, sl=64, sh=32)))
    with pytest.raises(native.PtcgError, match="null descriptor"):
        native.check(native.lib().ptcg_kernel_qk_norm_rope_fwd(None, P, P, P, P, None))


def _pages(**kw):
    lay = LAY(sn=16 * 64, sl=64, sh=32)
    return native.CPtcgPages(**{**dict(pages=9, page=16, per_seq=4, k=lay, v=lay, kp=P, vp=P, table=P, table_sn=4), **kw})


def _append(a_kw=None, ptr=(P, P, P, 2 * P), **kw):
    lay = lambda h: LAY(sn=8 * h * 32, sl=h * 32, sh=32)
    a = native.CPtcgPagedAppend(n=2, lq=8, rows=16, heads=4, kv_heads=2, dh=32, bf16=0, eps=1e-6, q=lay(4), k=lay(2),
                                v=lay(2), qo=lay(4), q_off=None, len=P, wq=P, wk=P, rope=_rope(), cache=_pages(**kw))
    for name, x in (a_kw or {}).items():
        setattr(a, name, x)
    return native.check(native.lib().ptcg_kernel_paged_append(ctypes.byref(a), *ptr, None))


@pytest.mark.parametrize("kw,match", BAD[2:8] + BAD[10:16] + [
    (dict(n=-1), "negative size"), (dict(lq=-1), "negative size"), (dict(q_off=P, rows=-1), "negative size"),
    (dict(q_off=P, rows=1 << 30), "too many rows"), (dict(kv_heads=0), "kv heads"), (dict(len=None), "null buffer"),
    (dict(v=LAY(sn=512, sl=-64, sh=32)), "negative stride"), (dict(qo=LAY(sn=1024, sl=64, sh=32)), "qo overlap"),
    (dict(q_off=P, qo=LAY(sn=0, sl=64, sh=32)), "qo overlap"),
])
def test_append_refuses(kw, match):
    with pytest.raises(native.PtcgError, match=match):
        _append(kw)


@pytest.mark.parametrize("kw,match", [
    (dict(pages=-1), "pages"), (dict(page=0), "pages"), (dict(per_seq=-1), "pages"),
    (dict(page=1 << 20, per_seq=1 << 20, table_sn=1 << 20), "2\\^30"), (dict(table_sn=3), "tables overlap"),
    (dict(k=LAY(sn=1024, sl=-64, sh=32)), "page strides"), (dict(table=None), "page table"), (dict(vp=None), "no pool"),
    (dict(k=LAY(sn=512, sl=64, sh=32)), "pages overlap"), (dict(v=LAY(sn=1024, sl=64, sh=16)), "pages overlap"),
    (dict(kp=P + 2), "alignment"),
])
def test_append_refuses_pages(kw, match):
    with pytest.raises(native.PtcgError, match=match):
        _append(**kw)


def test_append_takes_q_and_qo_together():
    for ptr in ((None, P, P, P), (P, P, P, None)):
        with pytest.raises(native.PtcgError, match="together"):
            _append(ptr=ptr)
    with pytest.raises(native.PtcgError, match="in place"):
        _append(dict(q=LAY(sn=2048, sl=256, sh=32)), ptr=(P, P, P, P))
