"""Latent attention (MLA), the sublayer in front of the MoE block (host side, torch for memory).

A cached token is one row of a paged pool: the latent (rank values, which every head's key and value
are expanded from), then the rotated key part that all heads share (rope values). ``mla_append``
writes new tokens, ``MlaDecode`` attends to the cache with single query tokens in the latent space,
and ``mla_prefill`` attends within whole prompts with a key and a value per head. The C ABI and
what each of them computes are in include/vib3_hip.h (vib3_mla_*). Every call runs on the current
torch stream of the tensors' device; there is no CPU branch.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import DT_BF16, DT_F16, DT_F32

_DT = {torch.float16: DT_F16, torch.bfloat16: DT_BF16}
_IN_DT = {torch.float32: DT_F32, **_DT}


def _launch(name: str, desc, device: torch.device) -> None:
    index = device.index if device.index is not None else torch.cuda.current_device()
    if index == torch.cuda.current_device():
        _lib.call(name, C.byref(desc), _lib.current_stream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, C.byref(desc), _lib.current_stream(index))


def _check(t: torch.Tensor, name: str, dtype, shape, device=None) -> torch.Tensor:
    """t as a device tensor of the dtype(s) and shape given (-1: any), innermost dimension contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a device tensor (no CPU fallback in vib3_amd)")
    if t.dtype not in (dtype if isinstance(dtype, (tuple, dict)) else (dtype,)):
        raise TypeError(f"{name}: unsupported dtype {t.dtype}")
    if t.dim() != len(shape) or any(w not in (-1, s) for w, s in zip(shape, t.shape)):
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call on {device}")
    return t


def _flat(t: torch.Tensor, name: str, dtype, shape, device) -> int:
    if not _check(t, name, dtype, shape, device).is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


class MlaCache:
    """A paged latent cache over pool [num_pages, page_size, rank + rope] (f16 or bf16)."""

    def __init__(self, pool: torch.Tensor, rank: int):
        _check(pool, "pool", _DT, (-1, -1, -1))
        self.pool, self.rank, self.rope = pool, rank, pool.shape[2] - rank
        if rank not in (256, 512) or self.rope not in (32, 64):
            raise ValueError(f"a row of {pool.shape[2]} with a latent of {rank}: the latent must be 256 or 512 and the "
                             "rotary part 32 or 64")

    def _desc(self, block_table: torch.Tensor) -> _lib.MlaCacheDesc:
        p = self.pool
        d = _lib.MlaCacheDesc()
        d.pool, d.dtype = p.data_ptr(), _DT[p.dtype]
        d.num_pages, d.page_size, d.rank, d.rope = p.shape[0], p.shape[1], self.rank, self.rope
        d.page_stride, d.row_stride = p.stride(0), p.stride(1)
        d.block_table = _flat(block_table, "block_table", torch.int32, (-1, -1), p.device)
        d.num_seqs, d.max_pages = block_table.shape
        return d


def mla_append(cache: MlaCache, block_table: torch.Tensor, seqs: torch.Tensor, positions: torch.Tensor, kv: torch.Tensor,
               inv_freq: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
               rope_scale: float = 1.0, interleaved: bool = True, q_rope: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, kv_out: Optional[torch.Tensor] = None) -> None:
    """Write the rows of new tokens to the cache (vib3_launch_mla_append).

    Token t is token positions[t] of sequence seqs[t] (int32 [tokens]; a negative sequence is padding, of
    which nothing is written). kv [tokens, rank + rope] (f32, f16 or bf16) holds the latent and the shared key as projected: the
    latent is RMS-normalised with norm_weight (f16 [rank]; None: as it is), the key rotated by
    positions[t] * inv_freq (f32 [rope / 2]) and scaled by rope_scale, in pairs (2i, 2i + 1) or, not
    interleaved, (i, i + rope / 2). q_out [tokens, heads, rope] receives q_rope rotated alike (it may be q_rope itself), kv_out
    [tokens, rank + rope] the rows as cached, which mla_prefill takes its k_rope from."""
    dev, dt = cache.pool.device, cache.pool.dtype
    tokens = _check(kv, "kv", _IN_DT, (-1, cache.rank + cache.rope), dev).shape[0]
    a = _lib.MlaAppendDesc()
    a.cache = cache._desc(block_table)
    a.tokens = tokens
    a.seqs = _flat(seqs, "seqs", torch.int32, (tokens,), dev)
    a.positions = _flat(positions, "positions", torch.int32, (tokens,), dev)
    a.kv, a.kv_dtype, a.kv_stride = kv.data_ptr(), _IN_DT[kv.dtype], kv.stride(0)
    if norm_weight is not None:
        a.norm_weight = _flat(norm_weight, "norm_weight", torch.float16, (cache.rank,), dev)
    a.norm_eps = eps
    a.inv_freq = _flat(inv_freq, "inv_freq", torch.float32, (cache.rope // 2,), dev)
    a.rope_scale, a.interleaved = rope_scale, int(interleaved)
    if q_rope is not None:
        _check(q_rope, "q_rope", dt, (tokens, -1, cache.rope), dev)
        _check(q_out, "q_out", dt, q_rope.shape, dev)
        a.q_rope, a.heads = q_rope.data_ptr(), q_rope.shape[1]
        a.q_token_stride, a.q_head_stride = q_rope.stride(0), q_rope.stride(1)
        a.q_out, a.q_out_token_stride, a.q_out_head_stride = q_out.data_ptr(), q_out.stride(0), q_out.stride(1)
    if kv_out is not None:
        _check(kv_out, "kv_out", dt, (tokens, cache.rank + cache.rope), dev)
        a.kv_out, a.kv_out_stride = kv_out.data_ptr(), kv_out.stride(0)
    _launch("vib3_launch_mla_append", a, dev)


class MlaDecode:
    """Attention over a latent cache, absorbed form: owns the workspace and the output for up to max_rows query
    tokens. Launches that may overlap (other streams, captured graphs) need an MlaDecode each."""

    def __init__(self, cache: MlaCache, heads: int, nope: int, v_dim: int, max_rows: int):
        self.cache, self.heads, self.nope, self.v_dim, self.max_rows = cache, heads, nope, v_dim, max_rows
        d = _lib.MlaDecodeDesc()
        d.cache = self._shape()
        d.rows, d.heads, d.nope, d.v_dim = max_rows, heads, nope, v_dim
        n = _lib.load().vib3_mla_decode_workspace_bytes(C.byref(d))
        if n == 0:
            raise ValueError(f"MlaDecode: unsupported heads={heads}, nope={nope}, v_dim={v_dim} or max_rows={max_rows}")
        self.workspace = torch.empty(n + 256, dtype=torch.uint8, device=cache.pool.device)
        self.out = torch.empty((max_rows, heads, v_dim), dtype=cache.pool.dtype, device=cache.pool.device)

    def _shape(self) -> _lib.MlaCacheDesc:
        d = _lib.MlaCacheDesc()
        d.dtype, d.rank, d.rope = _DT[self.cache.pool.dtype], self.cache.rank, self.cache.rope
        return d

    def launch(self, q_nope: torch.Tensor, q_rope: torch.Tensor, kv_b: Optional[torch.Tensor], block_table: torch.Tensor,
               lens: torch.Tensor, scale: float, seqs: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Row r attends to the first lens[r] cached tokens of sequence seqs[r] (None: sequence r).

        q_nope [rows, heads, nope], q_rope [rows, heads, rope], kv_b [heads, nope + v_dim, rank]; the result
        [rows, heads, v_dim] is in out (default: the head of self.out). With kv_b None, q_nope [rows, heads, rank] is in the
        latent space already and out [rows, heads, rank] receives the weighted latent."""
        c, dev, dt = self.cache, self.cache.pool.device, self.cache.pool.dtype
        rows = _check(q_nope, "q_nope", dt, (-1, self.heads, self.nope if kv_b is not None else c.rank), dev).shape[0]
        if rows > self.max_rows:
            raise ValueError(f"{rows} rows, made for {self.max_rows}")
        _check(q_rope, "q_rope", dt, (rows, self.heads, c.rope), dev)
        if out is None:
            if kv_b is None:
                out = torch.empty((rows, self.heads, c.rank), dtype=dt, device=dev)
            else:
                out = self.out[:rows]
        _check(out, "out", dt, (rows, self.heads, self.v_dim if kv_b is not None else c.rank), dev)
        a = _lib.MlaDecodeDesc()
        a.cache = c._desc(block_table)
        a.rows, a.heads, a.nope, a.v_dim, a.scale = rows, self.heads, self.nope, self.v_dim, scale
        if seqs is not None:
            a.seqs = _flat(seqs, "seqs", torch.int32, (rows,), dev)
        elif block_table.shape[0] < rows:
            raise ValueError(f"block_table has {block_table.shape[0]} sequences for {rows} rows and no seqs")
        a.lens = _flat(lens, "lens", torch.int32, (rows,), dev)
        a.q_nope, a.q_nope_row_stride, a.q_nope_head_stride = q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1)
        a.q_rope, a.q_rope_row_stride, a.q_rope_head_stride = q_rope.data_ptr(), q_rope.stride(0), q_rope.stride(1)
        if kv_b is not None:
            a.kv_b = _flat(kv_b, "kv_b", dt, (self.heads, self.nope + self.v_dim, c.rank), dev)
        a.out, a.out_row_stride, a.out_head_stride = out.data_ptr(), out.stride(0), out.stride(1)
        base = self.workspace.data_ptr()
        a.workspace = (base + 255) // 256 * 256
        a.workspace_bytes = self.workspace.numel() - (a.workspace - base)
        _launch("vib3_launch_mla_decode", a, dev)
        return out


def mla_prefill(q_nope: torch.Tensor, q_rope: torch.Tensor, kv: torch.Tensor, k_rope: torch.Tensor, cu_q: torch.Tensor,
                cu_k: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention within prompts, expanded form (vib3_launch_mla_prefill).

    Sequence s has the queries cu_q[s]..cu_q[s+1] and the keys cu_k[s]..cu_k[s+1] (int32 [num_seqs + 1]); its
    queries are its newest tokens. q_nope [q, heads, nope], q_rope [q, heads, rope] (rotated), kv [k, heads, nope + v_dim] (the latent through
    kv_b), k_rope [k, rope] (rotated); returns out [q, heads, v_dim]."""
    dev, dt = q_nope.device, q_nope.dtype
    tokens, heads, nope = _check(q_nope, "q_nope", _DT, (-1, -1, -1)).shape
    rope = _check(q_rope, "q_rope", dt, (tokens, heads, -1), dev).shape[2]
    keys, _, width = _check(kv, "kv", dt, (-1, heads, -1), dev).shape
    _check(k_rope, "k_rope", dt, (keys, rope), dev)
    v_dim = width - nope
    if v_dim < 1:
        raise ValueError(f"kv holds {width} values a head, the key's part alone is {nope}")
    if out is None:
        out = torch.empty((tokens, heads, v_dim), dtype=dt, device=dev)
    _check(out, "out", dt, (tokens, heads, v_dim), dev)
    a = _lib.MlaPrefillDesc()
    a.dtype, a.heads, a.nope, a.rope, a.v_dim = _DT[dt], heads, nope, rope, v_dim
    a.num_seqs, a.q_tokens, a.k_tokens = cu_q.shape[0] - 1, tokens, keys
    if a.num_seqs < 0:
        raise ValueError("cu_q must hold num_seqs + 1 offsets")
    a.cu_q = _flat(cu_q, "cu_q", torch.int32, (a.num_seqs + 1,), dev)
    a.cu_k = _flat(cu_k, "cu_k", torch.int32, (a.num_seqs + 1,), dev)
    a.q_nope, a.q_nope_token_stride, a.q_nope_head_stride = q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1)
    a.q_rope, a.q_rope_token_stride, a.q_rope_head_stride = q_rope.data_ptr(), q_rope.stride(0), q_rope.stride(1)
    a.kv, a.kv_token_stride, a.kv_head_stride = kv.data_ptr(), kv.stride(0), kv.stride(1)
    a.k_rope, a.k_rope_stride = k_rope.data_ptr(), k_rope.stride(0)
    a.scale = scale
    a.out, a.out_token_stride, a.out_head_stride = out.data_ptr(), out.stride(0), out.stride(1)
    _launch("vib3_launch_mla_prefill", a, dev)
    return out
