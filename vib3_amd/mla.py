"""Latent attention (MLA), the sublayer in front of the MoE block (host side, torch for memory).

A cached token is one row of a paged pool: the latent (rank values, which every head's key and value
are expanded from), then the rotated key part that all heads share (rope values). ``mla_append``
writes new tokens, ``MlaDecode`` attends to the cache with single query tokens in the latent space,
and ``mla_prefill`` attends within whole prompts with a key and a value per head. The C ABI and
what each of them computes are in include/vib3_hip.h (vib3_mla_*). Every call runs on the current
torch stream of the tensors' device; there is no CPU branch.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import DT_BF16, DT_F16, DT_F32

_DT = {torch.float16: DT_F16, torch.bfloat16: DT_BF16}
_IN_DT = {torch.float32: DT_F32, **_DT}
_INT = torch.int32
_current_device = torch._C._cuda_getDevice  # torch.cuda.current_device() without its lazy-initialisation check


def _launch(name: str, desc, index: int) -> None:
    fn = getattr(_lib.load(), name)
    if index == _current_device():
        rc = fn(desc, _lib.current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(desc, _lib.current_stream(index))
    if rc:
        raise _lib.Vib3Error(name, rc)


def _refuse(t, name: str, dtype, shape, index: int) -> None:
    """Raise for what is wrong with t (the checks' slow path)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a device tensor (no CPU fallback in vib3_amd)")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the call on device {index}")
    raise ValueError(f"{name}: the last dimension must be contiguous")


def _rows(t, name: str, dtype, shape, index: int) -> int:
    """Address of a device tensor of this dtype, shape and device whose innermost dimension is contiguous."""
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.stride(-1) == 1:
            return t.data_ptr()
    except AttributeError:
        pass
    if isinstance(t, torch.Tensor) and t.numel() == 0 and t.dtype is dtype and t.shape == shape and t.get_device() == index:
        return t.data_ptr()
    _refuse(t, name, dtype, shape, index)


def _flat(t, name: str, dtype, shape, index: int) -> int:
    """The same for a tensor that must be contiguous as a whole."""
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == index:
        raise ValueError(f"{name} must be contiguous")
    _refuse(t, name, dtype, shape, index)


def _dims(t, name: str, dtypes, dims: int):
    """Shape of a device tensor of one of these dtypes with so many dimensions."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a device tensor (no CPU fallback in vib3_amd)")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, not {t.dim()}")
    return t.shape


class MlaCache:
    """A paged latent cache over pool [num_pages, page_size, rank + rope] (f16 or bf16)."""

    def __init__(self, pool: torch.Tensor, rank: int):
        pages, page_size, width = _dims(pool, "pool", _DT, 3)
        self.pool, self.rank, self.rope = pool, rank, width - rank
        if rank not in (256, 512) or self.rope not in (32, 64):
            raise ValueError(f"a row of {width} with a latent of {rank}: the latent must be 256 or 512 and the rotary part 32 or 64")
        self.dtype, self.index = pool.dtype, pool.get_device()
        self._head = (_rows(pool, "pool", pool.dtype, pool.shape, self.index), _DT[pool.dtype], pages, page_size, rank, self.rope,
                      pool.stride(0), pool.stride(1))

    def _desc(self, block_table: torch.Tensor) -> _lib.MlaCacheDesc:
        seqs, pages = _dims(block_table, "block_table", (_INT,), 2)
        return _lib.MlaCacheDesc(*self._head, _flat(block_table, "block_table", _INT, block_table.shape, self.index), seqs, pages)


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
    index, dt, rank, rope = cache.index, cache.dtype, cache.rank, cache.rope
    desc = cache._desc(block_table)
    tokens = _dims(kv, "kv", _IN_DT, 2)[0]
    row, one = (tokens, rank + rope), (tokens,)
    kv_at = _rows(kv, "kv", kv.dtype, row, index)
    weight = 0 if norm_weight is None else _flat(norm_weight, "norm_weight", torch.float16, (rank,), index)
    q = (0, 0, 0, 0, 0, 0, 0)
    if q_rope is not None:
        heads = _dims(q_rope, "q_rope", (dt,), 3)[1]
        shape = (tokens, heads, rope)
        q = (_rows(q_rope, "q_rope", dt, shape, index), heads, q_rope.stride(0), q_rope.stride(1),
             _rows(q_out, "q_out", dt, shape, index), q_out.stride(0), q_out.stride(1))
    copy = (0, 0) if kv_out is None else (_rows(kv_out, "kv_out", dt, row, index), kv_out.stride(0))
    a = _lib.MlaAppendDesc(desc, tokens, _flat(seqs, "seqs", _INT, one, index), _flat(positions, "positions", _INT, one, index),
                           kv_at, _IN_DT[kv.dtype], kv.stride(0), weight, eps,
                           _flat(inv_freq, "inv_freq", torch.float32, (rope // 2,), index), rope_scale, interleaved, *q, *copy)
    _launch("vib3_launch_mla_append", a, index)


class MlaDecode:
    """Attention over a latent cache, absorbed form: owns the workspace and the output for up to max_rows query
    tokens. Launches that may overlap (other streams, captured graphs) need an MlaDecode each."""

    def __init__(self, cache: MlaCache, heads: int, nope: int, v_dim: int, max_rows: int):
        self.cache, self.heads, self.nope, self.v_dim, self.max_rows = cache, heads, nope, v_dim, max_rows
        d = _lib.MlaDecodeDesc()
        d.cache = _lib.MlaCacheDesc(*cache._head, 0, 0, 0)
        d.rows, d.heads, d.nope, d.v_dim = max_rows, heads, nope, v_dim
        n = _lib.load().vib3_mla_decode_workspace_bytes(d)
        if n == 0:
            raise ValueError(f"MlaDecode: unsupported heads={heads}, nope={nope}, v_dim={v_dim} or max_rows={max_rows}")
        self.workspace = torch.empty(n + 256, dtype=torch.uint8, device=cache.pool.device)
        self.out = torch.empty((max_rows, heads, v_dim), dtype=cache.dtype, device=cache.pool.device)
        base = self.workspace.data_ptr()
        self._space = ((base + 255) // 256 * 256, n)

    def launch(self, q_nope: torch.Tensor, q_rope: torch.Tensor, kv_b: Optional[torch.Tensor], block_table: torch.Tensor,
               lens: torch.Tensor, scale: float, seqs: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Row r attends to the first lens[r] cached tokens of sequence seqs[r] (None: sequence r).

        q_nope [rows, heads, nope], q_rope [rows, heads, rope], kv_b [heads, nope + v_dim, rank]; the result
        [rows, heads, v_dim] is in out (default: the head of self.out). With kv_b None, q_nope [rows, heads, rank] is in the
        latent space already and out [rows, heads, rank] receives the weighted latent."""
        c, heads, nope, v_dim = self.cache, self.heads, self.nope, self.v_dim
        index, dt = c.index, c.dtype
        rows = _dims(q_nope, "q_nope", (dt,), 3)[0]
        if rows > self.max_rows:
            raise ValueError(f"{rows} rows, made for {self.max_rows}")
        width, v_width, weight = (nope, v_dim, 0) if kv_b is not None else (c.rank, c.rank, 0)
        qn = _rows(q_nope, "q_nope", dt, (rows, heads, width), index)
        qr = _rows(q_rope, "q_rope", dt, (rows, heads, c.rope), index)
        if kv_b is not None:
            weight = _flat(kv_b, "kv_b", dt, (heads, nope + v_dim, c.rank), index)
        if out is None:
            out = self.out[:rows] if kv_b is not None else torch.empty((rows, heads, v_width), dtype=dt, device=c.pool.device)
        to = _rows(out, "out", dt, (rows, heads, v_width), index)
        desc = c._desc(block_table)
        which = 0
        if seqs is not None:
            which = _flat(seqs, "seqs", _INT, (rows,), index)
        elif desc.num_seqs < rows:
            raise ValueError(f"block_table has {desc.num_seqs} sequences for {rows} rows and no seqs")
        a = _lib.MlaDecodeDesc(desc, rows, heads, which, _flat(lens, "lens", _INT, (rows,), index),
                               qn, q_nope.stride(0), q_nope.stride(1), qr, q_rope.stride(0), q_rope.stride(1),
                               weight, nope, v_dim, scale, to, out.stride(0), out.stride(1), *self._space)
        _launch("vib3_launch_mla_decode", a, index)
        return out


def mla_prefill(q_nope: torch.Tensor, q_rope: torch.Tensor, kv: torch.Tensor, k_rope: torch.Tensor, cu_q: torch.Tensor,
                cu_k: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention within prompts, expanded form (vib3_launch_mla_prefill).

    Sequence s has the queries cu_q[s]..cu_q[s+1] and the keys cu_k[s]..cu_k[s+1] (int32 [num_seqs + 1]); its
    queries are its newest tokens. q_nope [q, heads, nope], q_rope [q, heads, rope] (rotated), kv [k, heads, nope + v_dim] (the latent through
    kv_b), k_rope [k, rope] (rotated); returns out [q, heads, v_dim]."""
    tokens, heads, nope = _dims(q_nope, "q_nope", _DT, 3)
    index, dt = q_nope.get_device(), q_nope.dtype
    rope = _dims(q_rope, "q_rope", (dt,), 3)[2]
    keys, _, width = _dims(kv, "kv", (dt,), 3)
    v_dim = width - nope
    if v_dim < 1:
        raise ValueError(f"kv holds {width} values a head, the key's part alone is {nope}")
    qn = _rows(q_nope, "q_nope", dt, (tokens, heads, nope), index)
    qr = _rows(q_rope, "q_rope", dt, (tokens, heads, rope), index)
    kv_at = _rows(kv, "kv", dt, (keys, heads, width), index)
    kr = _rows(k_rope, "k_rope", dt, (keys, rope), index)
    if out is None:
        out = torch.empty((tokens, heads, v_dim), dtype=dt, device=q_nope.device)
    to = _rows(out, "out", dt, (tokens, heads, v_dim), index)
    seqs = _dims(cu_q, "cu_q", (_INT,), 1)[0] - 1
    if seqs < 0:
        raise ValueError("cu_q must hold num_seqs + 1 offsets")
    offsets = (seqs + 1,)
    a = _lib.MlaPrefillDesc(_DT[dt], heads, nope, rope, v_dim, seqs, tokens, keys, _flat(cu_q, "cu_q", _INT, offsets, index),
                            _flat(cu_k, "cu_k", _INT, offsets, index), qn, q_nope.stride(0), q_nope.stride(1),
                            qr, q_rope.stride(0), q_rope.stride(1), kv_at, kv.stride(0), kv.stride(1), kr, k_rope.stride(0), scale,
                            to, out.stride(0), out.stride(1))
    _launch("vib3_launch_mla_prefill", a, index)
    return out
