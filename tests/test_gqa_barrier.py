"""CPU check of the chunk kernels' compiled code: the flag for values that were cleared is set to 0 by one wave and to 1 by any, so a
barrier stands between the two. What sets it follows the loads to LDS: a barrier in front of the first of them is one in front of it."""
import os
import re
import subprocess

from vib3_amd import build


def without_barrier(text, kernel="k_gqa_tiles"):
    """The functions of this name that load to LDS before their first barrier, and how many there are."""
    late, count, name, barrier = [], 0, None, False
    for raw in text.splitlines():
        line = raw.split(";")[0].strip()
        if re.match(rf"^_Z\w*{kernel}\w*:$", line):
            name, barrier, count = line[:-1], False, count + 1
        elif re.match(r"^_Z\w+:$", line):
            name = None
        elif name and line.startswith("s_barrier"):
            barrier = True
        elif name and line.startswith("global_load_lds"):
            if not barrier:
                late.append(name)
            name = None
    return late, count


def test_the_check_sees_a_missing_barrier():
    text = "_Z11k_gqa_tilesIv:\n ds_write_b32 v0, v1\n s_barrier\n global_load_lds_dwordx4 v1, s[8:9]\n"
    assert without_barrier(text) == ([], 1)
    assert without_barrier(text.replace(" s_barrier\n", "")) == (["_Z11k_gqa_tilesIv"], 1)
    assert without_barrier(text.replace(" s_barrier\n", "") + " s_barrier\n_Z1av:\n s_endpgm\n") == (["_Z11k_gqa_tilesIv"], 1)


def test_flag_is_cleared_behind_a_barrier(tmp_path):
    out = str(tmp_path / "code.s")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *build.HIPCC_FLAGS, "-S", "--cuda-device-only", "-o", out,
                    os.path.join(build.CSRC, "gqa_chunk.hip")], check=True, capture_output=True)
    late, count = without_barrier(open(out).read())
    assert count == 24 and late == []  # two types, three heads, cut or whole, whole groups on a page or not
