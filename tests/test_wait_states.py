"""The assembly of the kernels that load straight into LDS from inline assembly: the
compiler puts no wait states into such a block, so the block has to hold its own.

Two rules of these processors' documentation are searched for, in wait states (an
instruction is one, `s_nop n` is n + 1) along every path:
  - five between a vector instruction's write of a scalar register (v_readfirstlane of a
    buffer descriptor's word) and a memory instruction that reads it, else it may read the
    old one: another bound than the rows have;
  - one between a write of M0 and a load into LDS, whose place M0 is."""
import concurrent.futures as cf
import os
import re
import subprocess

import pytest

from ptcg_amd import build

SOURCES = ["gemm", "seqattn"]
DESCRIPTOR, PLACE = 5, 1

MEMORY = re.compile(r"(buffer_|global_|flat_|scratch_)")
SREG = re.compile(r"\bs(\d+)\b|\bs\[(\d+):(\d+)\]|\b(vcc|m0)\b")


def _regs(text):
    out = set()
    for one, lo, hi, name in SREG.findall(text):
        out |= {name} if name else {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return out


def _written(op, rest):
    """Scalar registers that a vector instruction writes."""
    if not op.startswith("v_"):
        return set()
    dst = rest.split(",")
    n = 2 if "_co_" in op or op.startswith(("v_div_scale", "v_mad_u64", "v_mad_i64")) else 1
    return set().union(*(_regs(x) for x in dst[:n])) if op.startswith(("v_cmp", "v_read")) or n == 2 else set()


def _blocks(lines):
    """[(instructions by line, labels that it may jump to, whether it may fall through)], and labels' blocks."""
    blocks, labels, cur = [], {}, []

    def close(to=(), falls=True):
        nonlocal cur
        blocks.append((cur, to, falls))
        cur = []

    for n, raw in enumerate(lines):
        x = raw.split(";")[0].strip()
        m = re.match(r"([\w.$]+):", x)
        if m:
            close()
            labels[m.group(1)] = len(blocks)
            continue
        if not x or x.startswith((".", "#", "/")):
            continue
        op, _, rest = x.partition(" ")
        cur.append((n, op, rest))
        if op == "s_branch":
            close((rest.strip(),), False)
        elif op.startswith("s_cbranch"):
            close((rest.strip(),))
        elif op in ("s_endpgm", "s_setpc_b64"):
            close((), False)
    close((), False)
    return blocks, labels


def late_waits(asm):
    """(line, instruction, register) of each load that comes too soon after a write of what
    it reads."""
    blocks, labels = _blocks(asm.split("\n"))
    start, found = [{} for _ in blocks], {}
    todo = list(range(len(blocks)))
    while todo:
        b = todo.pop()
        ins, to, falls = blocks[b]
        # wait states since a register's last write that matters
        state = dict(start[b])
        for n, op, rest in ins:
            if MEMORY.match(op):
                for r in _regs(rest):
                    if state.get(r, DESCRIPTOR) < DESCRIPTOR:
                        found[n, r] = f"{op} {rest}"
                if re.search(r"\blds\b", rest) and state.get("place", PLACE) < PLACE:
                    found[n, "m0"] = f"{op} {rest}"
            more = int(rest.strip(), 0) + 1 if op == "s_nop" else 1
            state = {r: d + more for r, d in state.items() if d + more < DESCRIPTOR}
            for r in _written(op, rest):
                state[r] = 0
            if re.match(r"(s|v_read)\w* m0\b", f"{op} {rest}"):
                state["place"] = 0
            elif op.startswith("s_") and not op.startswith(("s_cmp", "s_bitcmp")):
                for r in _regs(rest.split(",")[0]):      # a scalar write in its place
                    state.pop(r, None)
        for nb in [labels[x] for x in to if x in labels] + ([b + 1] if falls and b + 1 < len(blocks) else []):
            old = start[nb]
            new = {r: min(old.get(r, DESCRIPTOR), state.get(r, DESCRIPTOR)) for r in set(old) | set(state)}
            if new != old:
                start[nb] = new
                todo.append(nb)
    return sorted((n + 1, i, str(r)) for (n, r), i in found.items())


GOOD = """
_Z1kv:
	v_readfirstlane_b32 s42, v18
	s_mov_b32 m0, s69
	s_nop 4
	buffer_load_dwordx4 v82, s[40:43], 0 offen lds
.LBB0_1:
	buffer_load_dwordx4 v82, s[40:43], 0 offen
	v_readlane_b32 s41, v3, 2
	s_nop 3
	s_cbranch_scc1 .LBB0_1
	s_endpgm
"""


@pytest.mark.parametrize("was,put,want", [
    ("s_nop 4", "s_nop 2", "42"),                       # four wait states of five
    ("s_nop 4", "", "m0"), ("s_nop 4", "", "42"),
    ("s_nop 3", "s_nop 2", "41"),                       # by way of the loop
    ("s_nop 3", "v_cmp_lt_i32_e64 s[42:43], v1, v2", "43"),
    ("s_nop 3", "v_mad_u64_u32 v[2:3], s[40:41], v4, v5, v[2:3]", "40"),
])
def test_the_search_finds_a_missing_wait(was, put, want):
    assert late_waits(GOOD) == []
    assert want in [r for _, _, r in late_waits(GOOD.replace(was, put))]


def test_the_search_counts_the_instructions_between():
    five = GOOD.replace("\ts_nop 4\n", "\ts_nop 0\n" + "\tv_add_u32_e32 v1, v1, v2\n" * 3)
    assert late_waits(five) == []
    assert late_waits(five.replace("\ts_nop 0\n", ""))
    # a scalar write in between takes the vector one's place
    scalar = GOOD.replace("\ts_nop 4\n", "\ts_mov_b32 s42, 64\n")
    assert late_waits(scalar) == []


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
def test_loads_into_lds_wait_for_what_they_read(name, assembly):
    asm = assembly[name]
    assert len(re.findall(r"offen lds$", asm, re.M)) > 100      # the search has something to look at
    assert late_waits(asm) == []


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(build.CSRC) if f.endswith((".hip", ".h"))))
def test_assembly_that_moves_m0_says_so(name):
    with open(os.path.join(build.CSRC, name)) as f:
        blocks = re.findall(r"asm volatile\((.*?)\);", f.read(), re.S)
    assert [b for b in blocks if "m0" in b.split("::")[0] and '"m0"' not in b.split(":")[-1]] == []
