"""A compile-time check of the loads that paged_chunk_kernel issues from assembly (no GPU needed).

The compiler knows neither their hazards nor what they read: a scalar register that vector code wrote (v_readlane gives the
addresses of a block's rows) takes five wait states before a load may read it, and m0, which names the place in LDS, one after a scalar
move. A load that comes too early goes by what the register held before."""
import os
import re
import subprocess
import sys

import pytest

from helpers import ROOT

CSRC = os.path.join(ROOT, "itak-torch-rebuild_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
WAIT = 5


def scalars(text):
    regs = set()
    for m in re.finditer(r"\bs\[(\d+):(\d+)\]", text):
        regs |= set(range(int(m.group(1)), int(m.group(2)) + 1))
    for m in re.finditer(r"\bs(\d+)\b", text):
        regs.add(int(m.group(1)))
    return regs


def early(lines):
    """Loads to LDS whose scalar address, or m0, is fewer wait states old than it has to be, and how many loads there are."""
    age, m0_age, loads, bad = {}, 99, 0, []
    for n, raw in enumerate(lines, 1):
        line = raw.split(";")[0].strip()
        if not line or line.startswith(".") and not line.endswith(":"):
            continue
        if line.endswith(":"):
            continue  # (ages go on over labels: a register written before a branch is no younger behind it)
        op, _, rest = line.partition(" ")
        if op.startswith("global_load_lds"):
            loads += 1
            for reg in scalars(rest):
                if age.get(reg, 99) < WAIT:
                    bad.append((n, line, age[reg]))
            if m0_age < 1:
                bad.append((n, line, "m0"))
        states = int(rest, 0) + 1 if op == "s_nop" else 1
        age = {r: a + states for r, a in age.items() if a + states < WAIT}
        m0_age += states
        if op.startswith("v_"):
            for reg in scalars(rest.split(",")[0]):
                age[reg] = 0
        if op.startswith("s_mov") and rest.split(",")[0].strip() == "m0":
            m0_age = 0
    return bad, loads


def test_the_check_itself():
    load = "\tglobal_load_lds_dwordx4 v1, s[4:5]"
    assert early(["\tv_readlane_b32 s4, v0, 1", "\ts_mov_b32 m0, s9", "\ts_nop 0", load])[0]
    assert not early(["\tv_readlane_b32 s4, v0, 1", "\ts_mov_b32 m0, s9", "\ts_nop 3", load])[0]
    assert not early(["\tv_readlane_b32 s6, v0, 1", "\ts_mov_b32 m0, s9", "\ts_nop 0", load])[0]
    assert early(["\ts_mov_b32 m0, s9", load])[0]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is not installed")
def test_addresses_are_old_enough_for_the_loads_that_read_them(tmp_path):
    sys.path.insert(0, ROOT)
    from __graft_entry__ import _load_builder

    build = _load_builder()
    src, out = "paged_chunk_f16.hip", str(tmp_path / "kernel.s")
    flags = [f for f in build.FLAGS if not f.startswith("-Rpass")]
    subprocess.run([HIPCC, *flags, *build.source_flags(src), "--cuda-device-only", "-S", os.path.join(CSRC, src), "-o", out],
                   check=True, capture_output=True)
    bad, loads = early(open(out).read().split("\n"))
    assert loads > 100 and not bad, bad[:5]


def test_copies_under_lanes_that_are_off_are_found():
    from __graft_entry__ import _load_builder

    find = _load_builder().misplaced
    head = ["_ZN1k:", "\ts_and_saveexec_b64 s[6:7], vcc", ".LBB0_2:"]
    restore = "\ts_or_b64 exec, exec, s[6:7]"
    copy = "\tv_accvgpr_write_b32 a53, v71"
    assert find([*head, copy, restore]) == [("_ZN1k", 4)]
    assert find([*head, "\ts_nop 0 ; a comment", copy, restore])
    for fine in ([restore, copy], ["\ts_cbranch_execz .LBB0_3", copy, restore], ["\ts_and_saveexec_b64 s[8:9], vcc", copy, restore], [copy]):
        assert not find([*head, *fine])
