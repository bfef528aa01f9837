"""What the paged and windowed attention refuse before anything reaches a device,
the decoder operators' structs against the header, and their assembly."""
import ctypes
import os
import re
import subprocess

import pytest

from ptcg_amd import build, native
from test_register_copies import stray_copies

P = 4096          # a 16-byte aligned address nothing reads
LAY = native.CPtcgHeadLayout


def _pages(**kw):
    lay = LAY(sn=16 * 64, sl=64, sh=32)
    return native.CPtcgPages(**{**dict(pages=9, page=16, per_seq=4, k=lay, v=lay, kp=P, vp=P, table=P, table_sn=4), **kw})


def _paged(a_kw=None, **kw):
    lay = LAY(sn=8 * 128, sl=128, sh=32)
    a = native.CPtcgPagedAttn(n=2, lq=8, rows=16, heads=4, kv_heads=2, dh=32, bf16=0, scale=0.5, window=0, sinks=0,
                              q=lay, o=lay, q_off=None, len=P, cache=_pages(**kw))
    for name, x in (a_kw or {}).items():
        setattr(a, name, x)
    return a


def _run_paged(a, q=P, out=P, ws=None, nb=0):
    return native.check(native.lib().ptcg_kernel_paged_attention(ctypes.byref(a), q, out, None, ws, nb, None))


def _window(**kw):
    lay = lambda h: LAY(sn=16 * h * 32, sl=h * 32, sh=32)
    a = native.CPtcgWindowAttn(n=2, l=16, heads=4, kv_heads=2, dh=32, bf16=0, scale=0.5, window=0, sinks=0, q=lay(4),
                               k=lay(2), v=lay(2), o=lay(4), off=None, len=None)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


def _fwd(a, q=P, k=P, v=P, out=P, ws=None, nb=0):
    return native.check(native.lib().ptcg_kernel_window_attention_fwd(ctypes.byref(a), q, k, v, out, None, ws, nb, None))


def _bwd(a, q=P, k=P, v=P, out=P, lse=P, dout=P, dq=P, dk=P, dv=P, ws=P, nb=1 << 40):
    return native.check(native.lib().ptcg_kernel_window_attention_bwd(ctypes.byref(a), q, k, v, out, lse, dout, dq, dk, dv,
                                                                      ws, nb, None))


COMMON = [
    (dict(n=-1), "negative size"), (dict(heads=3), "kv heads"), (dict(kv_heads=0), "kv heads"),
    (dict(dh=12), "head width"), (dict(dh=136), "head width"), (dict(dh=0), "head width"), (dict(bf16=2), "bf16"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(q=LAY(sn=1024, sl=130, sh=32)), "strides"),
    (dict(o=LAY(sn=1024, sl=-128, sh=32)), "strides"), (dict(bf16=1, q=LAY(sn=1024, sl=132, sh=32)), "strides"),
    (dict(n=1 << 22), "too many rows"),
]


@pytest.mark.parametrize("kw,match", COMMON + [
    (dict(lq=-1), "negative size"), (dict(lq=1 << 30), "too long"), (dict(q_off=P, rows=-1), "rows"),
    (dict(q_off=P, rows=1 << 30), "rows"),
])
def test_paged_attention_refuses(kw, match):
    with pytest.raises(native.PtcgError, match=match):
        _run_paged(_paged(kw))
    assert native.lib().ptcg_kernel_paged_attention_ws_bytes(ctypes.byref(_paged(kw))) == -1


@pytest.mark.parametrize("kw,match", [
    (dict(pages=-1), "pages"), (dict(page=0), "pages"), (dict(per_seq=-1), "pages"),
    (dict(page=1 << 20, per_seq=1 << 20, table_sn=1 << 20), "2\\^30"), (dict(table_sn=3), "tables overlap"),
    (dict(k=LAY(sn=1024, sl=-64, sh=32)), "page strides"), (dict(v=LAY(sn=1024, sl=66, sh=32)), "page strides"),
    (dict(table=None), "page table"), (dict(kp=None), "no pool"), (dict(vp=P + 8), "16 B aligned"),
])
def test_paged_attention_refuses_pages(kw, match):
    with pytest.raises(native.PtcgError, match=match):
        _run_paged(_paged(**kw))


def test_paged_attention_refuses_buffers():
    for kw in (dict(q=None), dict(out=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _run_paged(_paged(), **kw)
    with pytest.raises(native.PtcgError, match="null buffer"):
        _run_paged(_paged(dict(len=None)))
    with pytest.raises(native.PtcgError, match="16 B aligned"):
        _run_paged(_paged(), q=P + 8)
    for lay in (LAY(sn=0, sl=128, sh=32), LAY(sn=1024, sl=64, sh=32), LAY(sn=1024, sl=128, sh=16)):
        with pytest.raises(native.PtcgError, match="output overlap"):
            _run_paged(_paged(dict(o=lay)))
    with pytest.raises(native.PtcgError, match="output overlap"):
        _run_paged(_paged(dict(q_off=P, o=LAY(sn=0, sl=64, sh=32))))
    # a token against many keys splits them and needs scratch
    a = _paged(dict(lq=1), per_seq=4000, table_sn=4000)
    need = native.lib().ptcg_kernel_paged_attention_ws_bytes(ctypes.byref(a))
    assert need > 0
    for ws, nb in ((None, need), (P, need - 1), (P + 8, need)):
        with pytest.raises(native.PtcgError, match="workspace"):
            _run_paged(a, ws=ws, nb=nb)
    with pytest.raises(native.PtcgError, match="null descriptor"):
        native.check(native.lib().ptcg_kernel_paged_attention(None, P, P, None, None, 0, None))


@pytest.mark.parametrize("kw,match", COMMON + [
    (dict(l=-1), "negative size"), (dict(l=1 << 30), "too long"), (dict(off=P, len=P), "take no len"),
    (dict(k=LAY(sn=1024, sl=66, sh=32)), "strides"), (dict(v=LAY(sn=1024, sl=1 << 22, sh=32)), "2\\^22"),
    (dict(k=LAY(sn=1024, sl=16, sh=512)), "key rows overlap"),
])
def test_window_attention_refuses(kw, match):
    for call in (_fwd, _bwd):
        with pytest.raises(native.PtcgError, match=match):
            call(_window(**kw))
    for back in (0, 1):
        assert native.lib().ptcg_kernel_window_attention_ws_bytes(ctypes.byref(_window(**kw)), back) == -1


def test_window_attention_refuses_buffers():
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _fwd(_window(), **kw)
        with pytest.raises(native.PtcgError, match="null buffer"):
            _bwd(_window(), **kw)
    for kw in (dict(lse=None), dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None)):
        with pytest.raises(native.PtcgError, match="null buffer"):
            _bwd(_window(), **kw)
    with pytest.raises(native.PtcgError, match="16 B aligned"):
        _fwd(_window(), k=P + 4)
    with pytest.raises(native.PtcgError, match="16 B aligned"):
        _bwd(_window(), dv=P + 4)
    with pytest.raises(native.PtcgError, match="output overlap"):
        _fwd(_window(o=LAY(sn=0, sl=128, sh=32)))
    with pytest.raises(native.PtcgError, match="dq overlap"):
        _bwd(_window(q=LAY(sn=2048, sl=0, sh=32)))
    for name in ("k", "v"):
        with pytest.raises(native.PtcgError, match="dk or dv overlap"):
            _bwd(_window(**{name: LAY(sn=0, sl=64, sh=32)}))
    for kw in (dict(ws=None), dict(nb=16), dict(ws=P + 8)):
        with pytest.raises(native.PtcgError, match="workspace"):
            _bwd(_window(), **kw)


@pytest.mark.parametrize("name,ct", [
    ("PtcgRope", native.CPtcgRope), ("PtcgQkRope", native.CPtcgQkRope), ("PtcgPages", native.CPtcgPages),
    ("PtcgPagedAppend", native.CPtcgPagedAppend), ("PtcgPagedAttn", native.CPtcgPagedAttn),
    ("PtcgWindowAttn", native.CPtcgWindowAttn)])
def test_structs_match_the_header(tmp_path, name, ct):
    fields = [f for f, _ in ct._fields_]
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ptcg_amd_kernels.h"\nint main(void) {\n'
                   f'  printf("size %zu\\n", sizeof({name}));\n'
                   + "".join(f'  printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f in fields) + "  return 0;\n}\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(ct)
    for f in fields:
        assert int(got[f]) == getattr(ct, f).offset, f


def _stored_behind(lines, at, copy):
    """Whether a copy to an accumulation register belongs to the region's body: a store of registers that hold it stands
    between it and the lanes' return (line at)."""
    reg = re.match(r"v_accvgpr_\w+ a(\d+),", copy)
    first = max(n for n in range(at) if lines[n].split(";")[0].strip() == copy)
    for x in lines[first + 1:at] if reg else []:
        for lo, hi in re.findall(r"_store_\w+ .*a\[(\d+):(\d+)\]", x):
            if int(lo) <= int(reg.group(1)) <= int(hi):
                return True
    return False


@pytest.mark.parametrize("name", ["rope", "seqattn"])
def test_no_register_is_copied_before_the_lanes_return(name):
    src = os.path.join(build.CSRC, name + ".hip")
    r = subprocess.run([build._hipcc(), *build.CFLAGS, "-w", "--cuda-device-only", "-S", src, "-o", "-"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.count("s_or_b64 exec, exec") > 10
    lines = r.stdout.split("\n")
    # v_writelane writes its lane whatever the mask
    assert [x for x in stray_copies(r.stdout) if not x[2].startswith("v_writelane") and not _stored_behind(lines, int(x[1].split()[-1]) - 1, x[2])] == []
