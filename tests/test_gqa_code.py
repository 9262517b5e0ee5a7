"""CPU check of the attention kernels' compiled code. Where registers are short, the compiler has put a copy that it made for that at
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
