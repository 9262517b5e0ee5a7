"""CPU checks of the attention kernels' compiled code. Where registers are short, the compiler has put a copy that it made for that at
the end of a divergent branch in front of the instruction that brings the other lanes back (s_or_b64 exec): they lost the value, and
addresses formed from it faulted. The kernels avoid such branches; this looks for what is left of them."""
import os
import re
import subprocess

import pytest

from vib3_amd import build

COPY = re.compile(r"v_accvgpr_(write|read|mov)|v_mov_b(32|64)(_e32)? v[\[\d:\]]+, v|scratch_(load|store)")


def copies_before_joins(text):
    """(function, copies) of the blocks that begin with register copies and then restore exec."""
    found, function, seen = [], None, None
    for raw in text.splitlines():
        line = raw.split(";")[0].strip()
        if re.match(r"^_Z\w+:$", line):
            function, seen = line[:-1], None
        elif re.match(r"^\.LBB\w+:$", line):
            seen = []
        elif seen is None or not line or line.startswith("."):
            continue
        elif re.match(r"s_or_b64 exec, exec,", line):
            if seen:
                found.append((function, seen))
            seen = None
        elif "saveexec" in line or line.startswith(("s_cbranch", "s_branch", "s_endpgm")) or re.match(r"s_\w+ exec", line):
            seen = None
        elif line.startswith(("v_", "ds_", "global_", "scratch_", "buffer_", "flat_")):
            if not COPY.match(line):
                seen = None  # the branch's own work: its label lies within it
            else:
                seen.append(line)
    return found


def test_the_check_sees_a_copy():
    text = "_Zk:\n.LBB0_1:\n  v_accvgpr_write_b32 a210, v138\n  s_mov_b32 s15, s51\n  s_or_b64 exec, exec, s[6:7]\n"
    assert copies_before_joins(text) == [("_Zk", ["v_accvgpr_write_b32 a210, v138"])]
    assert copies_before_joins(text.replace("  v_acc", "  s_or_b64 exec, exec, s[6:7]\n  v_acc")) == []
    assert copies_before_joins(text.replace("v_accvgpr_write_b32 a210, v138", "v_add_u32_e32 v1, v2, v3")) == []


@pytest.mark.parametrize("source", ["gqa_append.hip", "gqa_decode.hip", "gqa_chunk.hip", "cache_pages.hip"])
def test_no_copy_before_a_join(source, tmp_path):
    out = str(tmp_path / "code.s")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *build.HIPCC_FLAGS, "-S", "--cuda-device-only", "-o", out,
                    os.path.join(build.CSRC, source)], check=True, capture_output=True)
    text = open(out).read()
    assert "s_or_b64 exec, exec," in text
    assert copies_before_joins(text) == []


def late_scalars(text, wait=5):
    """Loads to LDS (written in assembly, which the compiler keeps no distance for) whose scalar address a vector instruction
    wrote fewer than `wait` instructions before."""
    lines = [line.split(";")[0].strip() for line in text.splitlines()]
    lines = [line for line in lines if line and (not line.startswith(".") or line.startswith(".LBB"))]
    found, loads = [], 0
    for i, line in enumerate(lines):
        m = re.match(r"global_load_lds_dwordx4 v\d+, s\[(\d+):(\d+)\]", line)
        if not m:
            continue
        loads += 1
        address, steps = set(range(int(m[1]), int(m[2]) + 1)), 0
        for before in reversed(lines[:i]):
            if steps == wait:
                break
            n = re.match(r"s_nop (\d+)", before)
            steps += int(n[1]) + 1 if n else not before.startswith(".LBB")
            w = re.match(r"v_\w+ s(?:(\d+)|\[(\d+):(\d+)\])(?:,|$)", before)
            if w and address & set(range(int(w[1] or w[2]), int(w[1] or w[3]) + 1)):
                found.append((before, line))
    return found, loads


def test_scalar_addresses_of_loads_to_lds(tmp_path):
    load = "global_load_lds_dwordx4 v1, s[8:9]"
    assert late_scalars(f"v_readlane_b32 s9, v1, 3\ns_nop 2\n{load}") == ([("v_readlane_b32 s9, v1, 3", load)], 1)
    assert late_scalars(f"v_readlane_b32 s9, v1, 3\ns_nop 4\n{load}") == ([], 1)
    assert late_scalars(f"v_readlane_b32 s7, v1, 3\ns_cselect_b32 s9, s1, s2\n{load}") == ([], 1)
    out = str(tmp_path / "code.s")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *build.HIPCC_FLAGS, "-S", "--cuda-device-only", "-o", out,
                    os.path.join(build.CSRC, "gqa_chunk.hip")], check=True, capture_output=True)
    found, loads = late_scalars(open(out).read())
    assert loads > 100 and found == []
