"""Refusals of the latent-attention launchers: every one returns its code before anything is launched, so they run
without a GPU, on addresses that are never read."""
import ctypes as C

import pytest

from vib3_amd import _lib

UNSUPPORTED, BAD_COUNT, BAD_POINTER, WORKSPACE = -1, -2, -3, -4
AT = 0x10000  # an aligned address


def cache(**kw):
    d = _lib.MlaCacheDesc()
    base = dict(pool=AT, dtype=_lib.DT_BF16, num_pages=4, page_size=16, rank=512, rope=64, page_stride=16 * 576, row_stride=576,
                block_table=AT, num_seqs=2, max_pages=2)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def desc(cls, base, kw):
    d = cls()
    inner = {k[6:]: v for k, v in kw.items() if k.startswith("cache_")}
    if hasattr(d, "cache"):
        d.cache = cache(**inner)
    for k, v in {**base, **{k: v for k, v in kw.items() if not k.startswith("cache_")}}.items():
        setattr(d, k, v)
    return d


def append(**kw):
    return desc(_lib.MlaAppendDesc, dict(
        tokens=3, seqs=AT, positions=AT, kv=AT, kv_dtype=_lib.DT_BF16, kv_stride=576, norm_weight=AT, norm_eps=1e-6, inv_freq=AT,
        rope_scale=1.0, interleaved=1, q_rope=AT, heads=4, q_token_stride=4 * 192, q_head_stride=192, q_out=AT,
        q_out_token_stride=256, q_out_head_stride=64, kv_out=AT, kv_out_stride=576), kw)


def decode(**kw):
    return desc(_lib.MlaDecodeDesc, dict(
        rows=2, heads=8, seqs=None, lens=AT, q_nope=AT, q_nope_row_stride=8 * 192, q_nope_head_stride=192, q_rope=AT,
        q_rope_row_stride=512, q_rope_head_stride=64, kv_b=AT, nope=128, v_dim=128, scale=0.1, out=AT, out_row_stride=1024,
        out_head_stride=128, workspace=AT, workspace_bytes=1 << 40), kw)


def prefill(**kw):
    return desc(_lib.MlaPrefillDesc, dict(
        dtype=_lib.DT_F16, heads=8, nope=128, rope=64, v_dim=128, num_seqs=1, q_tokens=5, k_tokens=5, cu_q=AT, cu_k=AT, q_nope=AT,
        q_nope_token_stride=1536, q_nope_head_stride=192, q_rope=AT, q_rope_token_stride=1536, q_rope_head_stride=192, kv=AT,
        kv_token_stride=2048, kv_head_stride=256, k_rope=AT, k_rope_stride=64, scale=0.1, out=AT, out_token_stride=1024,
        out_head_stride=128), kw)


CACHE = [
    (dict(cache_dtype=_lib.DT_F32), UNSUPPORTED), (dict(cache_rank=384), UNSUPPORTED), (dict(cache_rope=16), UNSUPPORTED),
    (dict(cache_page_size=0), BAD_COUNT), (dict(cache_page_size=65537), BAD_COUNT), (dict(cache_num_pages=-1), BAD_COUNT),
    (dict(cache_num_seqs=-1), BAD_COUNT), (dict(cache_max_pages=-1), BAD_COUNT), (dict(cache_row_stride=512), BAD_COUNT),
    (dict(cache_pool=None), BAD_POINTER), (dict(cache_pool=AT + 8), BAD_POINTER), (dict(cache_block_table=None), BAD_POINTER),
    (dict(cache_row_stride=580), BAD_POINTER), (dict(cache_page_stride=16 * 576 + 4), BAD_POINTER),
]


def refused(name, d, code):
    assert getattr(_lib.load(), name)(C.byref(d), None) == code
    with pytest.raises(_lib.Vib3Error) as e:
        _lib.call(name, C.byref(d), None)
    assert e.value.code == code


@pytest.mark.parametrize("kw,code", CACHE + [
    (dict(kv_dtype=7), UNSUPPORTED), (dict(tokens=-1), BAD_COUNT), (dict(heads=0), BAD_COUNT), (dict(seqs=None), BAD_POINTER),
    (dict(positions=None), BAD_POINTER), (dict(inv_freq=None), BAD_POINTER), (dict(kv=None), BAD_POINTER),
    (dict(kv=AT + 2), BAD_POINTER), (dict(kv_stride=577), BAD_POINTER), (dict(norm_weight=AT + 2), BAD_POINTER),
    (dict(kv_out=AT + 2), BAD_POINTER), (dict(kv_out_stride=578), BAD_POINTER), (dict(q_rope=AT + 4), BAD_POINTER),
    (dict(q_out=None), BAD_POINTER), (dict(q_head_stride=193), BAD_POINTER), (dict(q_out_token_stride=250), BAD_POINTER),
    (dict(tokens=2 ** 31 - 1, heads=128), BAD_COUNT),
])
def test_append_refusals(kw, code):
    refused("vib3_launch_mla_append", append(**kw), code)


@pytest.mark.parametrize("kw,code", CACHE + [
    (dict(rows=-1), BAD_COUNT), (dict(heads=0), BAD_COUNT), (dict(heads=129), BAD_COUNT), (dict(nope=100), UNSUPPORTED),
    (dict(v_dim=288), UNSUPPORTED), (dict(v_dim=0), UNSUPPORTED), (dict(lens=None), BAD_POINTER), (dict(q_nope=AT + 2), BAD_POINTER),
    (dict(q_rope=None), BAD_POINTER), (dict(kv_b=AT + 8), BAD_POINTER), (dict(out=None), BAD_POINTER),
    (dict(q_nope_head_stride=100), BAD_POINTER), (dict(out_row_stride=1023), BAD_POINTER), (dict(workspace=None), BAD_POINTER),
    (dict(scale=float("nan")), UNSUPPORTED), (dict(scale=float("inf")), UNSUPPORTED),
    (dict(workspace=AT + 16), BAD_POINTER), (dict(workspace_bytes=0), WORKSPACE), (dict(rows=2 ** 30), BAD_COUNT),
])
def test_decode_refusals(kw, code):
    refused("vib3_launch_mla_decode", decode(**kw), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.DT_F32), UNSUPPORTED), (dict(nope=96), UNSUPPORTED), (dict(v_dim=32), UNSUPPORTED), (dict(rope=16), UNSUPPORTED),
    (dict(heads=0), BAD_COUNT), (dict(heads=70000), BAD_COUNT), (dict(num_seqs=-1), BAD_COUNT), (dict(q_tokens=-1), BAD_COUNT),
    (dict(k_tokens=-1), BAD_COUNT), (dict(cu_q=None), BAD_POINTER), (dict(cu_k=None), BAD_POINTER), (dict(q_nope=None), BAD_POINTER),
    (dict(q_rope=AT + 2), BAD_POINTER), (dict(kv=None), BAD_POINTER), (dict(k_rope=None), BAD_POINTER), (dict(out=AT + 8), BAD_POINTER),
    (dict(kv_head_stride=252), BAD_POINTER), (dict(k_rope_stride=60), BAD_POINTER), (dict(out_head_stride=129), BAD_POINTER),
    (dict(q_tokens=2 ** 31 - 1, heads=65535), BAD_COUNT),
    (dict(scale=float("-inf")), UNSUPPORTED),
])
def test_prefill_refusals(kw, code):
    refused("vib3_launch_mla_prefill", prefill(**kw), code)


@pytest.mark.parametrize("name,d", [("vib3_launch_mla_append", append(tokens=0)), ("vib3_launch_mla_decode", decode(rows=0)),
                                    ("vib3_launch_mla_prefill", prefill(q_tokens=0)),
                                    ("vib3_launch_mla_prefill", prefill(num_seqs=0))])
def test_nothing_to_do(name, d):
    assert getattr(_lib.load(), name)(C.byref(d), None) == 0


@pytest.mark.parametrize("name", ["vib3_launch_mla_append", "vib3_launch_mla_decode", "vib3_launch_mla_prefill"])
def test_no_description(name):
    assert getattr(_lib.load(), name)(None, None) == BAD_POINTER


def test_workspace_grows_with_the_rows_and_refuses_bad_counts():
    size = _lib.load().vib3_mla_decode_workspace_bytes
    small, large = size(C.byref(decode(rows=1))), size(C.byref(decode(rows=512)))
    assert 0 < small <= large and large % 256 == 0
    for bad in (dict(rows=-1), dict(heads=0), dict(heads=129), dict(rows=2 ** 30)):
        assert size(C.byref(decode(**bad))) == 0
    assert size(None) == 0
    assert _lib.load().vib3_launch_mla_decode(C.byref(decode(workspace_bytes=small - 1, rows=1)), None) == WORKSPACE


def test_host_functions_refuse_cpu_tensors():
    torch = pytest.importorskip("torch")
    from vib3_amd import mla
    with pytest.raises(TypeError):
        mla.MlaCache(torch.zeros(2, 4, 576, dtype=torch.bfloat16), 512)
    with pytest.raises(TypeError):
        mla.mla_prefill(*[torch.zeros(2, 2, 64, dtype=torch.float16)] * 4, cu_q=None, cu_k=None, scale=1.0)
