"""How many rows the paged and windowed attention take (host alone: sizes of scratch)."""
import ctypes

import pytest

from ptcg_amd import native

P = 4096          # a 16-byte aligned address nothing reads
LAY = native.CPtcgHeadLayout


def _paged(n, lq, heads, kv, rows=None, dh=64):
    lay = LAY(sn=lq * heads * dh, sl=heads * dh, sh=dh)
    pool = LAY(sn=16 * kv * dh, sl=kv * dh, sh=dh)
    pages = native.CPtcgPages(pages=9, page=16, per_seq=4, k=pool, v=pool, kp=P, vp=P, table=P, table_sn=4)
    a = native.CPtcgPagedAttn(n=n, lq=lq, rows=rows or 0, heads=heads, kv_heads=kv, dh=dh, bf16=1, scale=0.5, q=lay,
                              o=lay, q_off=None if rows is None else P, len=P, cache=pages)
    return native.lib().ptcg_kernel_paged_attention_ws_bytes(ctypes.byref(a))


def _window(n, l, heads, kv, packed, back, dh=64, **kw):
    lay = lambda h: LAY(sn=l * h * dh, sl=h * dh, sh=dh)
    a = native.CPtcgWindowAttn(n=n, l=l, heads=heads, kv_heads=kv, dh=dh, bf16=1, scale=0.5, q=lay(heads), k=lay(kv),
                               v=lay(kv), o=lay(heads), off=P if packed else None, **kw)
    return native.lib().ptcg_kernel_window_attention_ws_bytes(ctypes.byref(a), back)


def test_packed_rows_count_as_many_as_there_are():
    # 4 096 sequences of up to 8 192 new rows, 8 heads and 64 on 8: however long one may be, 100 000 rows in all
    assert _paged(4096, 8192, 8, 8, rows=100_000) >= 0
    assert _paged(4096, 8192, 64, 8, rows=100_000) >= 0
    assert _paged(4096, 8192, 64, 8) == -1
    # (rows / 32 + 2 n) kv heads of one head each below 2^24: 2^20 sequences of 8 kv heads are too many alone, and of
    # 4 sequences rows from 2^26 - 256 on with 8 kv heads, from 2^27 - 256 on with 4
    assert _paged(1 << 20, 8, 8, 8, rows=9) == -1 and _paged((1 << 20) - 1, 8, 8, 8, rows=9) >= 0
    for kv, rows in ((8, (1 << 26) - 256), (4, (1 << 27) - 256)):
        assert _paged(4, 1 << 27, kv, kv, rows=rows) == -1 and _paged(4, 1 << 27, kv, kv, rows=rows - 1) >= 0

@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("back", [0, 1])
def test_windowed_sequences_up_to_the_threads_of_a_launch(packed, back):
    assert _window(4096, 8192, 8, 8, packed, back) >= 0           # 2^31 threads and a little
    assert _window(8128, 8192, 8, 8, packed, back) >= 0
    assert _window(8130, 8192, 8, 8, packed, back) == -1
    assert _window(1, (1 << 28) - 65, 1, 1, packed, back) >= 0
    assert _window(1, (1 << 28) - 64, 1, 1, packed, back) == -1
