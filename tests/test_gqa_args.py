"""Refusals of the grouped-query attention and page launchers: every one returns its code before anything is launched, so they run
without a GPU, on addresses that are never read."""
import ctypes as C
import os
import subprocess

import pytest

from vib3_amd import _lib

UNSUPPORTED, BAD_COUNT, BAD_POINTER, WORKSPACE = -1, -2, -3, -4
AT = 0x10000  # an aligned address


def fill(d, base, kw):
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def cache(**kw):
    return fill(_lib.GqaCacheDesc(), dict(keys=AT, values=AT, dtype=_lib.DT_BF16, num_pages=4, page_size=16, kv_heads=2, dim=128,
                                          page_stride=16 * 256, token_stride=256, head_stride=128, block_table=AT, num_seqs=2,
                                          max_pages=2), kw)


def with_cache(cls, base, kw):
    inner = {k[6:]: v for k, v in kw.items() if k.startswith("cache_")}
    return fill(cls(), {**base, "cache": cache(**inner)}, {k: v for k, v in kw.items() if not k.startswith("cache_")})


def append(**kw):
    return with_cache(_lib.GqaAppendDesc, dict(
        tokens=3, heads=8, seqs=AT, positions=AT, src_dtype=_lib.DT_BF16, q=AT, q_token_stride=1536, q_head_stride=128, k=AT,
        k_token_stride=1536, k_head_stride=128, v=AT, v_token_stride=1536, v_head_stride=128, q_norm=AT, k_norm=AT,
        norm_dtype=_lib.DT_F32, norm_eps=1e-6, inv_freq=AT, rot=128, rope_scale=1.0, interleaved=0, q_out=AT, q_out_token_stride=1024,
        q_out_head_stride=128), kw)


def decode(**kw):
    return with_cache(_lib.GqaDecodeDesc, dict(
        rows=2, heads=8, seqs=None, lens=AT, q=AT, q_row_stride=1024, q_head_stride=128, scale=0.1, window=0, sinks=0, out=AT,
        out_row_stride=1024, out_head_stride=128, workspace=AT, workspace_bytes=1 << 40), kw)


def chunk(**kw):
    return with_cache(_lib.GqaChunkDesc, dict(
        heads=8, q_tokens=5, cu_q=AT, lens=AT, q=AT, q_token_stride=1024, q_head_stride=128, scale=0.1, window=0, sinks=0, out=AT,
        out_token_stride=1024, out_head_stride=128, workspace=AT, workspace_bytes=1 << 40), kw)


def pools(n=1, **kw):
    one = dict(base=AT, page_stride=8192, run_stride=0, token_stride=512, runs=1, token_bytes=512)
    return (_lib.PagePoolDesc * n)(*[fill(_lib.PagePoolDesc(), one, kw) for _ in range(n)])


def fork(pool=None, **kw):
    return fill(_lib.ForkPagesDesc(), dict(pools=pools(**(pool or {})), num_pools=1, num_pages=4, page_size=16, block_table=AT, num_seqs=2,
                                           max_pages=2, lens=AT, count=1, parents=AT, children=AT, new_pages=AT), kw)


def compact(pool=None, **kw):
    return fill(_lib.CompactPagesDesc(), dict(pools=pools(**(pool or {})), num_pools=1, num_pages=4, page_size=16, block_table=AT,
                                              num_seqs=2, max_pages=2, lens=AT, out_table=AT, live=AT, workspace=AT,
                                              workspace_bytes=1 << 30), kw)


def refused(name, d, code):
    assert getattr(_lib.load(), name)(C.byref(d), None) == code
    with pytest.raises(_lib.Vib3Error) as e:
        _lib.call(name, C.byref(d), None)
    assert e.value.code == code


CACHE = [
    (dict(cache_dtype=_lib.DT_F32), UNSUPPORTED), (dict(cache_dim=96), UNSUPPORTED), (dict(cache_dim=32), UNSUPPORTED),
    (dict(cache_page_size=0), BAD_COUNT), (dict(cache_page_size=65537), BAD_COUNT), (dict(cache_num_pages=-1), BAD_COUNT),
    (dict(cache_num_seqs=-1), BAD_COUNT), (dict(cache_max_pages=-1), BAD_COUNT), (dict(cache_kv_heads=0), BAD_COUNT),
    (dict(cache_kv_heads=1025), BAD_COUNT), (dict(cache_token_stride=120), BAD_COUNT), (dict(cache_head_stride=64), BAD_COUNT),
    (dict(cache_page_stride=-8), BAD_COUNT), (dict(cache_keys=None), BAD_POINTER), (dict(cache_values=AT + 8), BAD_POINTER),
    (dict(cache_block_table=None), BAD_POINTER), (dict(cache_token_stride=260), BAD_POINTER), (dict(cache_head_stride=132), BAD_POINTER),
    (dict(cache_page_stride=16 * 256 + 4), BAD_POINTER),
]


@pytest.mark.parametrize("kw,code", CACHE + [
    (dict(src_dtype=7), UNSUPPORTED), (dict(norm_dtype=-1), UNSUPPORTED), (dict(rot=8), UNSUPPORTED), (dict(rot=-16), UNSUPPORTED),
    (dict(rot=144), UNSUPPORTED), (dict(tokens=-1), BAD_COUNT), (dict(heads=0), BAD_COUNT), (dict(heads=7), BAD_COUNT),
    (dict(heads=1026), BAD_COUNT), (dict(seqs=None), BAD_POINTER), (dict(positions=None), BAD_POINTER), (dict(inv_freq=None), BAD_POINTER),
    (dict(k=None), BAD_POINTER), (dict(v=AT + 2), BAD_POINTER), (dict(k_token_stride=1537), BAD_POINTER), (dict(v_head_stride=132), BAD_POINTER),
    (dict(q_norm=AT + 2), BAD_POINTER), (dict(k_norm=AT + 4), BAD_POINTER), (dict(q=AT + 4), BAD_POINTER), (dict(q_out=None), BAD_POINTER),
    (dict(q_head_stride=129), BAD_POINTER), (dict(q_out_token_stride=1020), BAD_POINTER),
])
def test_append_refusals(kw, code):
    refused("vib3_launch_gqa_append", append(**kw), code)


ATTENTION = CACHE + [
    (dict(heads=0), BAD_COUNT), (dict(heads=9), BAD_COUNT), (dict(heads=1026), BAD_COUNT), (dict(window=-1), BAD_COUNT),
    (dict(sinks=-1), BAD_COUNT), (dict(lens=None), BAD_POINTER), (dict(q=AT + 2), BAD_POINTER), (dict(q_head_stride=100), BAD_POINTER),
    (dict(out=None), BAD_POINTER), (dict(out_head_stride=1023), BAD_POINTER), (dict(workspace=None), BAD_POINTER),
    (dict(workspace=AT + 16), BAD_POINTER), (dict(workspace_bytes=0), WORKSPACE), (dict(scale=float("nan")), UNSUPPORTED),
    (dict(scale=float("-inf")), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", ATTENTION + [
    (dict(rows=-1), BAD_COUNT), (dict(rows=65537), BAD_COUNT), (dict(q_row_stride=1023), BAD_POINTER), (dict(out_row_stride=4), BAD_POINTER),
])
def test_decode_refusals(kw, code):
    refused("vib3_launch_gqa_decode", decode(**kw), code)


@pytest.mark.parametrize("kw,code", ATTENTION + [
    (dict(q_tokens=-1), BAD_COUNT), (dict(q_tokens=2 ** 31 - 1, heads=1024), BAD_COUNT), (dict(cu_q=None), BAD_POINTER),
    (dict(q_token_stride=1023), BAD_POINTER), (dict(out_token_stride=4), BAD_POINTER),
])
def test_chunk_refusals(kw, code):
    refused("vib3_launch_gqa_chunk", chunk(**kw), code)


POOLS = [
    (dict(num_pools=-1), BAD_COUNT), (dict(num_pages=-1), BAD_COUNT), (dict(page_size=0), BAD_COUNT), (dict(page_size=65537), BAD_COUNT),
    (dict(num_seqs=-1), BAD_COUNT), (dict(max_pages=-1), BAD_COUNT), (dict(pools=None), BAD_POINTER), (dict(pool=dict(runs=0)), BAD_COUNT),
    (dict(pool=dict(token_bytes=0)), BAD_COUNT), (dict(pool=dict(page_stride=-16)), BAD_COUNT), (dict(pool=dict(run_stride=-16)), BAD_COUNT),
    (dict(pool=dict(token_stride=-16)), BAD_COUNT), (dict(pool=dict(base=None)), BAD_POINTER), (dict(pool=dict(base=AT + 8)), BAD_POINTER),
    (dict(pool=dict(token_bytes=520)), BAD_POINTER), (dict(pool=dict(page_stride=8200)), BAD_POINTER),
    (dict(pool=dict(token_stride=520)), BAD_POINTER), (dict(pool=dict(run_stride=8)), BAD_POINTER),
    (dict(pool=dict(runs=2 ** 30, token_bytes=512)), BAD_COUNT), (dict(lens=None), BAD_POINTER), (dict(block_table=None), BAD_POINTER),
]


@pytest.mark.parametrize("kw,code", POOLS + [
    (dict(count=-1), BAD_COUNT), (dict(parents=None), BAD_POINTER), (dict(children=None), BAD_POINTER), (dict(new_pages=None), BAD_POINTER),
    (dict(count=2 ** 31 - 1), BAD_COUNT),
])
def test_fork_refusals(kw, code):
    refused("vib3_launch_fork_pages", fork(**kw), code)


@pytest.mark.parametrize("kw,code", POOLS + [
    (dict(num_pages=2 ** 20 + 1), BAD_COUNT), (dict(out_table=None), BAD_POINTER), (dict(live=None), BAD_POINTER),
    (dict(workspace=None), BAD_POINTER), (dict(workspace=AT + 64), BAD_POINTER), (dict(workspace_bytes=0), WORKSPACE),
])
def test_compact_refusals(kw, code):
    refused("vib3_launch_compact_pages", compact(**kw), code)


@pytest.mark.parametrize("name,d", [
    ("vib3_launch_gqa_append", append(tokens=0)), ("vib3_launch_gqa_decode", decode(rows=0)), ("vib3_launch_gqa_chunk", chunk(q_tokens=0)),
    ("vib3_launch_gqa_chunk", chunk(cache_num_seqs=0)), ("vib3_launch_fork_pages", fork(count=0)), ("vib3_launch_fork_pages", fork(num_seqs=0)),
])
def test_nothing_to_do(name, d):
    assert getattr(_lib.load(), name)(C.byref(d), None) == 0


@pytest.mark.parametrize("name", ["gqa_append", "gqa_decode", "gqa_chunk", "fork_pages", "compact_pages"])
def test_no_description(name):
    assert getattr(_lib.load(), "vib3_launch_" + name)(None, None) == BAD_POINTER


def test_workspaces():
    lib = _lib.load()
    for size, make, bad in ((lib.vib3_gqa_decode_workspace_bytes, decode, (dict(rows=-1), dict(rows=65537), dict(heads=0), dict(heads=9))),
                            (lib.vib3_gqa_chunk_workspace_bytes, chunk, (dict(q_tokens=-1), dict(heads=0), dict(heads=9))),
                            (lib.vib3_compact_pages_workspace_bytes, compact, (dict(num_pages=-1), dict(num_pages=2 ** 20 + 1)))):
        n = size(C.byref(make()))
        assert n > 0 and n % 256 == 0 and size(None) == 0
        assert all(size(C.byref(make(**kw))) == 0 for kw in bad)
    for launch, size, make in (("vib3_launch_gqa_decode", lib.vib3_gqa_decode_workspace_bytes, decode),
                               ("vib3_launch_gqa_chunk", lib.vib3_gqa_chunk_workspace_bytes, chunk),
                               ("vib3_launch_compact_pages", lib.vib3_compact_pages_workspace_bytes, compact)):
        refused(launch, make(workspace_bytes=size(C.byref(make())) - 1), WORKSPACE)


def test_workspace_of_fewer_tokens_and_sequences_fits():
    """What is made for the most rows serves every call with fewer."""
    lib = _lib.load()
    for heads, kv in ((8, 2), (64, 1), (5, 5), (48, 3)):
        c = dict(cache_kv_heads=kv, heads=heads)
        most = lib.vib3_gqa_decode_workspace_bytes(C.byref(decode(rows=300, **c)))
        assert all(0 < lib.vib3_gqa_decode_workspace_bytes(C.byref(decode(rows=n, **c))) <= most for n in range(1, 301))
        most = lib.vib3_gqa_chunk_workspace_bytes(C.byref(chunk(q_tokens=3000, cache_num_seqs=20, **c)))
        assert all(0 < lib.vib3_gqa_chunk_workspace_bytes(C.byref(chunk(q_tokens=n, cache_num_seqs=s, **c))) <= most
                   for n in (1, 2, 31, 32, 33, 64, 100, 127, 128, 129, 255, 500, 1000, 1999, 2000, 2500, 3000) for s in range(1, 21))


def test_host_functions_refuse_cpu_tensors():
    torch = pytest.importorskip("torch")
    from vib3_amd import gqa, pages
    with pytest.raises(TypeError):
        gqa.GqaCache(*[torch.zeros(2, 4, 2, 128, dtype=torch.bfloat16)] * 2)
    with pytest.raises(TypeError):
        pages.fork_pages([torch.zeros(2)], None, None, None, None, None)
    with pytest.raises(ValueError):
        pages.PageCompaction([])


def test_descriptions_lie_as_the_header_says(tmp_path):
    """Sizes and offsets of the ctypes descriptions against a C compiler's."""
    pairs = {"vib3_gqa_cache": _lib.GqaCacheDesc, "vib3_gqa_append": _lib.GqaAppendDesc, "vib3_gqa_decode": _lib.GqaDecodeDesc,
             "vib3_gqa_chunk": _lib.GqaChunkDesc, "vib3_page_pool": _lib.PagePoolDesc, "vib3_fork_pages": _lib.ForkPagesDesc,
             "vib3_compact_pages": _lib.CompactPagesDesc}
    lines = [f'printf("%zu %zu\\n", sizeof({name}), offsetof({name}, {f[0]}));' for name, d in pairs.items() for f in d._fields_]
    source = tmp_path / "lay.c"
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"vib3_hip.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, "-o", str(tmp_path / "lay"), str(source)], check=True, capture_output=True)
    out = subprocess.run([str(tmp_path / "lay")], check=True, capture_output=True, text=True).stdout.split("\n")
    want = [f"{C.sizeof(d)} {getattr(d, f[0]).offset}" for d in pairs.values() for f in d._fields_]
    assert out[:-1] == want
