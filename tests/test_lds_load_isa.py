"""The inline-asm loads that go straight to LDS against the wait states the
compiler does not count for them (CPU test: hipcc builds the translation units to
gfx950 assembly, nothing runs).

Such a load reads its LDS address from m0 and its buffer descriptor from SGPRs.
gfx950 asks for 1 wait state between a scalar write of m0 and the load, and for 5
between a VALU write of an SGPR (v_readlane, v_readfirstlane, v_cmp) and a vector
memory instruction that reads it; it checks neither.  The compiler keeps to both for its own
loads, but does not look into inline asm.  This test reads the built code, along every path that leads
to such a load, and fails where fewer states lie between.

The compiler does not take m0 as changed by the asm either (it is a reserved register, which no clobber names):
the test also fails where an instruction of the compiler's own reads m0 behind the asm's write of it.
"""
import concurrent.futures
import os
import re
import subprocess

import pytest

from tests.test_tall_isa import HIPCC, ROOT, _states

HIP = os.path.join(ROOT, "cuda_llm_ops_amd", "csrc", "hip")
VGPR_FORM = {"flash_gqa_forward_tall.hip", "flash_gqa_backward_dkdv.hip"}   # (as the Makefile builds them)

M0_STATES = 1
SGPR_STATES = 5


def _sgprs(spec):
    out = {r for r in ("vcc", "m0") if re.search(rf"\b{r}\b", spec)}
    for m in re.finditer(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", spec):
        out |= {f"s{m.group(3)}"} if m.group(3) else {f"s{i}" for i in range(int(m.group(1)), int(m.group(2)) + 1)}
    return out


def _code(asm):
    """[(text, inside inline asm)], and the indices that control may come from before each."""
    code, labels, in_asm = [], {}, False
    for line in asm.split("\n"):
        t = line.strip()
        if t.startswith((";;#ASMSTART", ";;#ASMEND")):
            in_asm = t.startswith(";;#ASMSTART")
        elif re.match(r"[.\w$]+:", t):
            labels[t.split(":")[0]] = len(code)
        elif t and not t.startswith((";", ".")):
            code.append((t.split(";")[0].strip(), in_asm))
    before = [[i - 1] if i and not re.match(r"s_branch|s_endpgm|s_setpc", code[i - 1][0]) else [] for i in range(len(code))]
    for i, (t, _) in enumerate(code):
        m = re.match(r"s_c?branch\w*\s+(\S+)", t)
        if m and labels.get(m.group(1), len(code)) < len(code):
            before[labels[m.group(1)]].append(i)
    return code, before


def _written_by(t):
    """(SGPRs that a VALU instruction writes, whether a scalar one writes m0)"""
    name, _, rest = t.partition(" ")
    if name.startswith("v_"):
        ops = rest.split(",")
        # (the destination; a carry or the mask of a comparison or division is the second one, and VOPC's plain form writes vcc)
        out = _sgprs(ops[0]) | (_sgprs(ops[1]) if re.match(r"v_(add|sub|subrev|addc|subb|subbrev)_co|v_div_scale|v_mad_[iu]64", name) else set())
        return out, False
    return set(), name.startswith("s_") and not name.startswith(("s_cmp", "s_bitcmp", "s_nop", "s_waitcnt")) and rest.split(",")[0].strip() == "m0"


def lds_load_hazards(asm):
    """(the loads to LDS inside inline asm, writes of m0 too near to them, writes of SGPRs too near)"""
    code, before = _code(asm)
    loads = [i for i, (t, a) in enumerate(code) if a and re.match(r"(buffer|global)_load\w*\s.*\blds\b", t)]
    near_m0, near_sgprs = [], []
    for k in loads:
        reads = _sgprs(code[k][0])
        seen = set()
        paths = [(i, 0) for i in before[k]]
        while paths:
            i, ws = paths.pop()
            if ws >= SGPR_STATES or (i, ws) in seen:
                continue
            seen.add((i, ws))
            t = code[i][0]
            sgprs, m0 = _written_by(t)
            if m0 and ws < M0_STATES:
                near_m0.append(f"{t}  ->  {code[k][0]} after {ws} wait states")
            if sgprs & reads:
                near_sgprs.append(f"{t}  ->  {code[k][0]} after {ws} wait states")
                continue
            paths += [(j, ws + _states(t)) for j in before[i]]
    return loads, near_m0, near_sgprs


def _writes_m0(t):
    return _written_by(t)[1]


def m0_reads(asm):
    """(instructions outside inline asm that read m0, those that the asm's m0 may reach)"""
    code, before = _code(asm)
    reads = [i for i, (t, a) in enumerate(code) if not a and "m0" in _sgprs(t) and not _writes_m0(t)]
    found = []
    for k in reads:
        seen, paths = {k}, list(before[k])
        while paths:
            i = paths.pop()
            if i in seen:
                continue
            seen.add(i)
            if _writes_m0(code[i][0]):
                if code[i][1]:
                    found.append(f"{code[i][0]}  ->  {code[k][0]}")
                continue
            paths += before[i]
    return reads, found


def _build(name, out):
    form = ["-mllvm", "-amdgpu-mfma-vgpr-form"] if name in VGPR_FORM else []
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "--cuda-device-only", "-S",
                    "-I" + os.path.join(ROOT, "include"), "-I" + HIP, "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", *form, os.path.join(HIP, name), "-o", out],
                   check=True, capture_output=True, timeout=600)
    with open(out) as f:
        return f.read()


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("needs hipcc")
    out = tmp_path_factory.mktemp("isa")
    names = sorted(n for n in os.listdir(HIP) if n.endswith(".hip"))
    with concurrent.futures.ThreadPoolExecutor(8) as pool:
        return dict(zip(names, pool.map(lambda n: _build(n, str(out / (n + ".s"))), names)))


def test_lds_load_wait_states(built):
    counts, found_m0, found_sgprs = {}, [], []
    for name, asm in built.items():
        loads, near_m0, near_sgprs = lds_load_hazards(asm)
        counts[name] = len(loads)
        found_m0 += [f"{name}: {x}" for x in near_m0 + m0_reads(asm)[1]]
        found_sgprs += [f"{name}: {x}" for x in near_sgprs]
    with_loads = {n for n, c in counts.items() if c}
    assert {"decode_shared.hip", "flash_gqa_forward.hip", "flash_gqa_forward_tall.hip", "flash_gqa_backward.hip",
            "flash_gqa_backward_dkdv.hip"} <= with_loads, f"no load to LDS found: the check would pass vacuously ({counts})"
    assert not found_m0, f"{len(found_m0)}\n" + "\n".join(found_m0[:20])
    assert not found_sgprs, f"{len(found_sgprs)}\n" + "\n".join(found_sgprs[:20])


def test_scan_finds_planted_cases():
    """The scan itself: an m0 written right before the load, a descriptor read from a lane 4 states before it, and one at
    the end of a loop that the load begins must be reported; the same with the states between must not."""
    bad = """
.LBB0_1:
    ;;#ASMSTART
    s_add_u32 m0, s4, 1024
    s_nop 4
    buffer_load_dwordx4 v1, s[8:11], 0 offen lds
    ;;#ASMEND
    v_readlane_b32 s12, v3, 0
    s_nop 1
    ;;#ASMSTART
    s_mov_b32 m0, s4
    buffer_load_dwordx4 v1, s[12:15], 0 offen lds
    ;;#ASMEND
    s_nop 7
.LBB0_2:
    ;;#ASMSTART
    buffer_load_dword v1, s[16:19], s20 offen lds
    ;;#ASMEND
    v_readfirstlane_b32 s20, v7
    s_cbranch_scc1 .LBB0_2
    s_endpgm
    """
    loads, near_m0, near_sgprs = lds_load_hazards(bad)
    assert len(loads) == 3 and [x.split(" ")[0] for x in near_m0] == ["s_mov_b32"]
    assert sorted(x.split(" ")[0] for x in near_sgprs) == ["v_readfirstlane_b32", "v_readlane_b32"]
    good = """
    v_readlane_b32 s8, v3, 0
    v_cmp_lt_i32_e64 s[20:21], v1, v2
    ;;#ASMSTART
    s_add_u32 m0, s4, 1024
    s_nop 4
    buffer_load_dwordx4 v1, s[8:11], s20 offen lds
    ;;#ASMEND
    v_readlane_b32 s8, v3, 0
    s_endpgm
    """
    loads, near_m0, near_sgprs = lds_load_hazards(good)
    assert len(loads) == 1 and near_m0 == [] and near_sgprs == []
    mixed = """
    s_mov_b32 m0, s1
    v_writelane_b32 v2, s0, m0
    ;;#ASMSTART
    s_mov_b32 m0, s4
    ;;#ASMEND
    s_cbranch_scc0 .LBB0_1
    s_mov_b32 m0, s1
.LBB0_1:
    v_writelane_b32 v2, s2, m0
    """
    reads, found = m0_reads(mixed)
    assert len(reads) == 2 and found == ["s_mov_b32 m0, s4  ->  v_writelane_b32 v2, s2, m0"]
