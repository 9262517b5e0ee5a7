"""Refusal of more query rows than a chunk's numbering takes: it comes before anything is launched, so no GPU is needed."""
import ctypes as C

import pytest

from test_gqa_args import BAD_COUNT, chunk, refused
from vib3_amd import _lib


@pytest.mark.parametrize("heads,q_tokens", [(1, 2 ** 31 - 1), (1, 2 ** 31 - 256), (16, 2 ** 27 - 15), (1024, 2 ** 21)])
def test_rows_past_2_31(heads, q_tokens):
    refused("vib3_launch_gqa_chunk", chunk(cache_kv_heads=1, heads=heads, q_tokens=q_tokens), BAD_COUNT)


def test_no_tokens_are_taken():
    assert _lib.load().vib3_launch_gqa_chunk(C.byref(chunk(cache_kv_heads=1, heads=1, q_tokens=0)), None) == 0
