"""What the cross-attention, embedding and 8-bit checkpoint entry points refuse
before anything reaches a device (the checks run on the host alone)."""
import ctypes
import os
import subprocess

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


def _emb_fwd(ids=P, rows=10, table=P, ldt=8, vocab=5, d=8, out=P, ldo=8):
    return native.check(native.lib().ptcg_kernel_embedding_fwd(ids, rows, table, ldt, 0, vocab, d, 1.0, out, ldo, 0,
                                                               None))


def _emb_bwd(ids=P, rows=10, dout=P, ldo=8, vocab=5, d=8, dtable=P, ldt=8, ws=P, nb=1 << 20):
    return native.check(native.lib().ptcg_kernel_embedding_bwd(ids, rows, dout, ldo, 0, vocab, d, 1.0, dtable, ldt, ws,
                                                               nb, None))


@pytest.mark.parametrize("call", [_emb_fwd, _emb_bwd])
@pytest.mark.parametrize("kw,match", [
    (dict(rows=-1), "rows"), (dict(rows=1 << 30), "rows"), (dict(vocab=0), "vocab"), (dict(d=0), "d=0"),
    (dict(d=65537, ldt=65537, ldo=65537), "d=65537"), (dict(ldt=7), "row strides"), (dict(ldo=4), "row strides"),
    (dict(ids=None), "null buffer"),
])
def test_embedding_refuses(call, kw, match):
    with pytest.raises(native.PtcgError, match=match):
        call(**kw)


def test_embedding_refuses_buffers():
    L = native.lib()
    for kw in (dict(table=None), dict(out=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _emb_fwd(**kw)
    for kw in (dict(dout=None), dict(dtable=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _emb_bwd(**kw)
    need = L.ptcg_kernel_embedding_bwd_ws_bytes(10, 5, 8)
    assert need > 0 and L.ptcg_kernel_embedding_bwd_ws_bytes(10, 0, 8) == -1
    for kw in (dict(ws=None), dict(nb=need - 1), dict(ws=P + 4)):
        with pytest.raises(native.PtcgError, match="workspace"):
            _emb_bwd(**kw)
    _emb_fwd(rows=0, ids=None, table=None, out=None)     # nothing to look up


def test_ckpt8_refuses():
    L, check = native.lib(), native.check
    bad = lambda match: pytest.raises(native.PtcgError, match=match)
    for rows, d, ldx, ldq, lds, match in ((-1, 8, 8, 8, 1, "rows"), (4, 0, 8, 8, 1, "d=0"), (4, 8, 7, 8, 1, "stride"),
                                          (4, 8, 8, 7, 1, "strides"), (4, 40, 40, 40, 1, "strides"),
                                          (2 ** 31 - 1, 2 ** 20, 2 ** 20, 2 ** 20, 2 ** 15, "too many")):
        with bad(match):
            check(L.ptcg_kernel_ckpt8_pack(P, ldx, 0, rows, d, P, ldq, P, lds, None))
        with bad(match):
            check(L.ptcg_kernel_ckpt8_unpack(P, ldq, P, lds, rows, d, P, ldx, 0, None))
        with bad(match):
            check(L.ptcg_kernel_ckpt8_gelu_bwd(P, ldq, P, lds, rows, d, P, ldx, P, ldx, None, 0, 0, None))
    with bad("stride"):
        check(L.ptcg_kernel_ckpt8_gelu_bwd(P, 8, P, 1, 4, 8, P, 8, P, 8, P, 4, 0, None))
    for k in range(3):
        a = [None if i == k else P for i in range(3)]
        with bad("null buffer"):
            check(L.ptcg_kernel_ckpt8_pack(a[0], 8, 0, 4, 8, a[1], 8, a[2], 1, None))
        with bad("null buffer"):
            check(L.ptcg_kernel_ckpt8_unpack(a[0], 8, a[1], 1, 4, 8, a[2], 8, 0, None))
    dw = lambda rows=4000, k=32, n=16, dy=P, lddy=16, q=P, ldq=32, sc=P, lds=1, dW=P, ws=P, nb=1 << 30: check(
        L.ptcg_kernel_ckpt8_dw(rows, k, n, dy, lddy, 0, q, ldq, sc, lds, dW, P, ws, nb, None))
    need = L.ptcg_kernel_ckpt8_dw_ws_bytes(4000, 32, 16, 0)
    assert need > 0 and L.ptcg_kernel_ckpt8_dw_ws_bytes(4000, 0, 16, 0) == -1
    for kw, match in ((dict(rows=-1), "rows"), (dict(k=0), "in=0"), (dict(n=0), "out=0"), (dict(lddy=15), "stride"),
                      (dict(ldq=31), "strides"), (dict(lds=0), "strides"), (dict(dy=None), "null"),
                      (dict(q=None), "null"), (dict(sc=None), "null"), (dict(dW=None), "null"),
                      (dict(ws=None), "workspace"), (dict(nb=need - 1), "workspace"), (dict(ws=P + 2), "workspace"),
                      (dict(k=1 << 20, n=1 << 20, ldq=1 << 20, lds=1 << 15, lddy=1 << 20), "too large")):
        with bad(match):
            dw(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(k=LAY(sn=1024, sl=16, sh=32)), "key rows overlap"), (dict(v=LAY(sn=1024, sl=24, sh=512)), "key rows overlap"),
    (dict(lk=1, k_off=P, v=LAY(sn=0, sl=16, sh=32)), "key rows overlap"),
    (dict(n=1 << 22, kv_heads=4), "too many"), (dict(n=1 << 16, lq=1 << 15, q=LAY(sl=128, sh=32)), "too many"),
    (dict(o=LAY(sn=1 << 60, sl=128, sh=32), n=100), "overlap"),
])
def test_cross_attention_refuses_what_a_launch_cannot_hold(kw, match):
    with pytest.raises(native.PtcgError, match=match):
        _fwd(_desc(**kw))


@pytest.mark.parametrize("kw", [dict(o=LAY(sn=0, sl=0, sh=32)), dict(o=LAY(sn=0, sl=128, sh=0)),
                                dict(o=LAY(sn=0, sl=16, sh=320))])
def test_packed_cross_attention_refuses_rows_upon_another(kw):
    with pytest.raises(native.PtcgError, match="overlap"):
        _fwd(_desc(q_off=P, k_off=P, **kw))


def test_operators_refuse_more_than_a_launch_holds():
    bad = lambda match: pytest.raises(native.PtcgError, match=match)
    L, check = native.lib(), native.check
    with bad("too many"):
        _emb_fwd(rows=(1 << 30) - 1, d=4096, ldt=4096, ldo=4096)
    with bad("too many"):
        _emb_bwd(rows=100, vocab=1 << 30, d=64, ldt=64, ldo=64, nb=1 << 60)
    with bad("too many"):
        _emb_bwd(rows=(1 << 30) - 1, d=1024, ldt=1024, ldo=1024, nb=1 << 60)
    with bad("too many"):
        check(L.ptcg_kernel_ckpt8_pack(P, 1024, 0, 1 << 26, 1024, P, 1024, P, 32, None))
    with bad("stride"):
        check(L.ptcg_kernel_ckpt8_gelu_bwd(P, 8, P, 1, 4, 8, P, 8, P, 16, None, 0, 0, None))
    for dz, act in ((P, P + 64), (P + 64, P + 64)):      # act over dy, over dz
        with bad("act is"):
            check(L.ptcg_kernel_ckpt8_gelu_bwd(P, 8, P, 1, 4, 8, P + 64, 8, dz, 8, act, 8, 0, None))


def test_cross_attention_struct_matches_the_header(tmp_path):
    """Sizes and field offsets from the C header (compiled with gcc) equal the
    ctypes declarations."""
    for name, ct in (("PtcgHeadLayout", native.CPtcgHeadLayout), ("PtcgCrossAttn", native.CPtcgCrossAttn)):
        fields = [f for f, _ in ct._fields_]
        src, exe = tmp_path / (name + ".c"), tmp_path / name
        src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ptcg_amd_kernels.h"\nint main(void) {\n'
                       f'  printf("size %zu\\n", sizeof({name}));\n'
                       + "".join(f'  printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f in fields)
                       + "  return 0;\n}\n")
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
        got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                     check=True).stdout.splitlines())
        assert int(got["size"]) == ctypes.sizeof(ct)
        for f in fields:
            assert int(got[f]) == getattr(ct, f).offset, f


@pytest.mark.parametrize("lay", [
    LAY(sn=0, sl=64, sh=32),      # row r + 1's head 0 on row r's head 2
    LAY(sn=0, sl=32, sh=32),      # rows and heads at one stride
    LAY(sn=0, sl=96, sh=32),      # one head too many for a row
    LAY(sn=0, sl=64, sh=64),
    LAY(sn=0, sl=128, sh=132),    # heads of rows: the second row reaches into the next head
    LAY(sn=0, sl=1 << 40, sh=1 << 39),
    LAY(sn=0, sl=1 << 62, sh=1 << 62),
])
def test_packed_outputs_refuse_rows_that_reach_into_heads(lay):
    """Whatever the packed row counts: from two rows on, two elements share an address."""
    with pytest.raises(native.PtcgError, match="output overlap"):
        _fwd(_desc(q_off=P, k_off=P, o=lay))
    with pytest.raises(native.PtcgError, match="dq overlap"):
        _bwd(_desc(q_off=P, k_off=P, q=lay))
    # 4 kv heads: the same layouts for the gradients of k and v
    for name in ("k", "v") if lay.sl < 1 << 22 else ():
        with pytest.raises(native.PtcgError, match="dk or dv overlap"):
            _bwd(_desc(q_off=P, k_off=P, kv_heads=4, **{name: lay}))


@pytest.mark.parametrize("lay", [
    LAY(sn=0, sl=128, sh=32), LAY(sn=0, sl=256, sh=32), LAY(sn=0, sl=512, sh=128), LAY(sn=0, sl=32, sh=64),
    LAY(sn=0, sl=32, sh=32 * 16), LAY(sn=0, sl=132, sh=164), LAY(sn=0, sl=1 << 40, sh=1 << 38)])
def test_packed_outputs_that_may_lie_apart_pass_the_layout_check(lay):
    """They get as far as the workspace (a long sample, whose keys are split)."""
    with pytest.raises(native.PtcgError, match="workspace"):
        _fwd(_desc(n=1, lq=3, lk=100000, q_off=P, k_off=P, o=lay))
    with pytest.raises(native.PtcgError, match="workspace"):
        _bwd(_desc(q_off=P, k_off=P, q=lay), nb=4)


def test_a_lone_row_takes_any_row_stride_and_a_lone_head_any_head_stride():
    with pytest.raises(native.PtcgError, match="workspace"):
        _fwd(_desc(n=1, lq=1, lk=100000, q_off=P, k_off=P, o=LAY(sn=0, sl=0, sh=32)))
    with pytest.raises(native.PtcgError, match="workspace"):
        _fwd(_desc(n=1, lq=3, lk=100000, heads=1, kv_heads=1, q_off=P, k_off=P, o=LAY(sn=0, sl=32, sh=0)))


@pytest.mark.parametrize("kw", [dict(lk=0, k=LAY(sn=0, sl=64, sh=32), v=LAY(sn=0, sl=64, sh=32)),
                                dict(lk=0, k_off=P, k=LAY(sn=0, sl=0, sh=0), v=LAY(sn=0, sl=0, sh=0))])
def test_gradients_of_no_rows_need_no_layout(kw):
    """Dense tensors of no keys have a sample stride of 0."""
    with pytest.raises(native.PtcgError, match="workspace"):
        _bwd(_desc(**kw), nb=4)
