"""Refusals of pages whose number of 16-byte chunks does not fit an int, in a process of their own: a count that wraps around to 0 would
end it. Nothing is launched, so no GPU is needed."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CODE = """
import ctypes as C
import test_gqa_args as T
from vib3_amd import _lib
kw = dict(pool=dict(runs={runs}, token_bytes={token_bytes}), page_size={page_size})
for name, d in (("vib3_launch_fork_pages", T.fork(**kw)), ("vib3_launch_compact_pages", T.compact(**kw))):
    print(getattr(_lib.load(), name)(C.byref(d), None))
"""


@pytest.mark.parametrize("runs,page_size,token_bytes", [
    (2 ** 30, 2 ** 16, 2 ** 22), (2 ** 30, 2 ** 16, 2 ** 22 + 16), (2 ** 31 - 1, 2 ** 16, 2 ** 31 - 16), (1, 2 ** 16, 2 ** 20),
    (2 ** 31 - 1, 1, 16), (2 ** 15, 2 ** 16, 16),
])
def test_pages_of_too_many_bytes(runs, page_size, token_bytes):
    path = os.pathsep.join([HERE, os.path.dirname(HERE)])
    out = subprocess.run([sys.executable, "-c", CODE.format(runs=runs, page_size=page_size, token_bytes=token_bytes)],
                         capture_output=True, text=True, env={**os.environ, "PYTHONPATH": path})
    assert out.returncode == 0 and out.stdout.split() == ["-2", "-2"], out.stderr[-2000:]
