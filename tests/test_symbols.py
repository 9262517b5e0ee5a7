"""CPU check of the compiled objects: of two functions of one name and signature in namespace vib3 the linker keeps one, and a file whose
own is dropped calls the other. What two objects define alike has to come from a header."""
import glob
import os
import re
import subprocess
from collections import defaultdict

from vib3_amd import build


def defined_twice(listing, headers):
    """Weak functions of vib3 (from {object: output of nm -C}) that two objects define and no header names."""
    where = defaultdict(set)
    for obj, text in listing.items():
        for line in text.splitlines():
            m = re.match(r"[0-9a-f]+ [WVu] (.*)", line)
            if m and "vib3::" in m[1]:
                where[m[1]].add(obj)
    found = []
    for symbol, objs in where.items():
        name = re.search(r"vib3::(?:\w+::)*(~?\w+)", symbol)
        if len(objs) > 1 and not (name and re.search(rf"\b{name[1]}\s*[(<]", headers)):
            found.append(symbol)
    return found


def test_the_check_sees_a_pair():
    line = "0000000000000000 W int vib3::launch<1>(vib3::Args const&)"
    assert defined_twice({"a": line, "b": line}, "inline int other(int);") == ["int vib3::launch<1>(vib3::Args const&)"]
    assert defined_twice({"a": line, "b": line}, "inline int launch(const Args&);") == []
    assert defined_twice({"a": line, "b": line.replace("launch", "other")}, "") == []


def test_no_function_is_defined_by_two_files(tmp_path):
    objs = {s: os.path.join(build.OBJ, os.path.splitext(s)[0] + ".o") for s in build.SOURCES}
    if not all(os.path.exists(o) for o in objs.values()):
        build.build(objdir=str(tmp_path), out=str(tmp_path / "lib.so"))
        objs = {s: os.path.join(str(tmp_path), os.path.basename(o)) for s, o in objs.items()}
    listing = {s: subprocess.run(["nm", "-C", o], check=True, capture_output=True, text=True).stdout for s, o in objs.items()}
    headers = "".join(open(h).read() for h in sorted(glob.glob(os.path.join(build.CSRC, "*.h"))))
    assert " W " in listing["mla_decode.hip"] and "vib3::" in listing["mla_decode.hip"]  # the names are as the check expects them
    assert defined_twice(listing, headers) == []
