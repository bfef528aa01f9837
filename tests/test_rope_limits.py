"""How many rows a launch of the rotation's entry points takes: more are refused by name, not by the launch."""
import ctypes

import pytest

from ptcg_amd import native

P = 4096          # an aligned address nothing reads
LAY = native.CPtcgHeadLayout

# (head width, bf16, its lanes): an access is one element where dh / 2 is odd, else as many as divide it, up to 16 bytes
WIDTHS = [(66, 1, 64), (34, 1, 32), (128, 1, 8), (128, 0, 16), (36, 0, 16)]


def _rows(lanes):
    """The fewest rows that make 2^32 lanes, or 2^30 - 1, the most that any call takes."""
    return (1 << 32) // lanes


@pytest.mark.parametrize("dh,bf16,lanes", [w for w in WIDTHS if _rows(w[2]) < 1 << 30])
def test_rows_past_a_launch_are_refused(dh, bf16, lanes):
    l = _rows(lanes)
    lay = LAY(sn=l * dh, sl=dh, sh=dh)
    rope = native.CPtcgRope(rot=dh, interleaved=0, mag=1.0, freq=P, pos=None)
    a = native.CPtcgQkRope(n=1, l=l, heads=1, kv_heads=0, dh=dh, bf16=bf16, eps=1e-6, q=lay, k=lay, qo=lay, ko=lay,
                           wq=P, wk=P, rope=rope)
    with pytest.raises(native.PtcgError, match="qk_norm_rope_fwd: too many rows"):
        native.check(native.lib().ptcg_kernel_qk_norm_rope_fwd(ctypes.byref(a), P, None, 2 * P, None, None))
    pool = LAY(sn=16 * dh, sl=dh, sh=dh)
    pages = native.CPtcgPages(pages=9, page=16, per_seq=4, k=pool, v=pool, kp=P, vp=P, table=P, table_sn=4)
    for off, n, lq in ((None, 1, l), (P, 4, 16)):
        a = native.CPtcgPagedAppend(n=n, lq=lq, rows=l, heads=1, kv_heads=1, dh=dh, bf16=bf16, eps=1e-6, q=lay, k=lay,
                                    v=lay, qo=lay, q_off=off, len=P, wq=P, wk=P, rope=rope, cache=pages)
        with pytest.raises(native.PtcgError, match="paged_append: too many rows"):
            native.check(native.lib().ptcg_kernel_paged_append(ctypes.byref(a), P, P, P, 2 * P, None))
