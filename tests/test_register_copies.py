"""The assembly of the kernels that fill the registers: nothing may touch a vector
register between a divergent region's end and the lanes' return.

A region that only some lanes run ends in a label with `s_or_b64 exec, exec, ...`
behind it; lanes that skip the region jump there by `s_cbranch_execz`.  Where
the register allocator puts copies of live registers (to accumulation registers
or to scratch) before the `s_or_b64`, the lanes outside the region keep stale
values: results are lost on some lanes only, with no error.  The compiler has
made such code for a kernel that is no longer built."""
import concurrent.futures as cf
import os
import re
import subprocess

import pytest

from ptcg_amd import build

SOURCES = ["xattn", "embed", "ckpt8"]

VECTOR = re.compile(r"(v_|ds_|scratch_|buffer_|global_|flat_)")
ENDS = re.compile(r"(\.LBB|s_c?branch|s_endpgm|s_setpc)")
COPY = re.compile(r"(v_accvgpr_write_b32 a\d+, v|v_accvgpr_mov|scratch_store)")


def stray_copies(asm):
    """(kernel, label or line, instruction) of each vector instruction on a region's
    end before the lanes return.  Where the end has no label of its own, its block
    holds the region's body too: there only copies to accumulation registers or
    scratch count."""
    lines = [x.split(";")[0].strip() if not x.startswith("; %bb") else "%bb" for x in asm.split("\n")]
    joins = {m.group(1) for x in lines for m in [re.match(r"s_cbranch_execz (\S+)", x)] if m}
    found, kernel, block, label = [], None, [], None
    for n, x in enumerate(lines):
        if re.match(r"_Z\w+:", x):
            kernel = x[:-1]
        if re.match(r"(\.LBB\w+:|%bb)", x):
            label, block = x.rstrip(":"), []
        elif x.startswith("s_or_b64 exec, exec") and block is not None:
            at = f"{label} line {n + 1}"
            found += [(kernel, at, i) for i in block if label in joins or COPY.match(i)]
            block = None
        elif re.match(r"s_\w+ (exec|\S+, exec)|s_\w*saveexec", x) or ENDS.match(x):
            block = None          # another mask from here on, or no end of a region
        elif block is not None and VECTOR.match(x) and not x.startswith("v_readlane"):   # reads whatever the mask
            block.append(x)
    return found


GOOD = """
_Z1kv:
	s_and_saveexec_b64 s[4:5], vcc
	s_cbranch_execz .LBB0_2
; %bb.1:
	v_accvgpr_write_b32 a3, 0
	global_load_dword v5, v[0:1], off
.LBB0_2:
	s_waitcnt vmcnt(0)
	v_readlane_b32 s4, v40, 2
	s_or_b64 exec, exec, s[4:5]
	v_accvgpr_write_b32 a4, v9
"""


@pytest.mark.parametrize("put", ["v_accvgpr_write_b32 a4, v9", "scratch_store_dword off, v9, off offset:16",
                                 "v_mov_b32_e32 v60, v9", "v_accvgpr_read_b32 v2, a9"])
def test_the_search_finds_a_copy_before_the_lanes_return(put):
    assert stray_copies(GOOD) == []
    bad = GOOD.replace("\ts_waitcnt vmcnt(0)\n", "\ts_waitcnt vmcnt(0)\n\t" + put + "\n")
    assert [(k, i) for k, _, i in stray_copies(bad)] == [("_Z1kv", put)]
    # the region's end in a block of its own without a label, or merged with its body
    merged = bad.replace(".LBB0_2:", "; %bb.2:")
    assert len(stray_copies(merged)) == ("accvgpr_write" in put or "scratch" in put)


@pytest.fixture(scope="module")
def assembly():
    def one(name):
        src = os.path.join(build.CSRC, name + ".hip")
        cmd = [build._hipcc(), *build.CFLAGS, "-w", "--cuda-device-only", "-S", src, "-o", "-"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-2000:]
        return r.stdout

    with cf.ThreadPoolExecutor(len(SOURCES)) as ex:
        return dict(zip(SOURCES, ex.map(one, SOURCES)))


@pytest.mark.parametrize("name", SOURCES)
def test_no_register_is_copied_before_the_lanes_return(name, assembly):
    asm = assembly[name]
    assert asm.count("s_or_b64 exec, exec") > 10      # the search has something to look at
    assert stray_copies(asm) == []
