"""Grouped-query attention (GQA), the sublayer in front of the MoE block for models with a key and a value per group of heads
(host side, torch for memory).

A cached token is a key and a value per key/value head, in two pools of pages. ``gqa_append`` writes new tokens (norms and rotation
on the way), ``GqaDecode`` attends to the cache with single query tokens, ``GqaChunk`` with the newest tokens of each sequence: a
prompt, its next chunk, drafted tokens. The C ABI and what each of them computes are in include/vib3_hip.h (vib3_gqa_*);
vib3_amd/pages.py forks and compacts a cache's pages. Every call runs on the current torch stream of the tensors' device; there is
no CPU branch.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .mla import _DT, _IN_DT, _INT, _dims, _flat, _launch, _rows


class GqaCache:
    """A paged cache over keys and values [num_pages, page_size, kv_heads, dim] (f16 or bf16), both with the same strides: two
    tensors, two halves of one, or transposed views of [num_pages, kv_heads, page_size, dim]."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor):
        pages, page_size, kv_heads, dim = _dims(keys, "keys", _DT, 4)
        if dim not in (64, 128, 256):
            raise ValueError(f"a head of {dim}: it must be 64, 128 or 256")
        self.keys, self.values, self.kv_heads, self.dim = keys, values, kv_heads, dim
        self.dtype, self.index = keys.dtype, keys.get_device()
        at = [_rows(t, n, self.dtype, keys.shape, self.index) for t, n in ((keys, "keys"), (values, "values"))]
        if keys.stride() != values.stride():
            raise ValueError(f"keys and values must have the same strides, not {keys.stride()} and {values.stride()}")
        self._head = (*at, _DT[self.dtype], pages, page_size, kv_heads, dim, *keys.stride()[:3])

    def _desc(self, block_table: torch.Tensor) -> _lib.GqaCacheDesc:
        seqs, pages = _dims(block_table, "block_table", (_INT,), 2)
        return _lib.GqaCacheDesc(*self._head, _flat(block_table, "block_table", _INT, block_table.shape, self.index), seqs, pages)

    def _empty_desc(self) -> _lib.GqaCacheDesc:
        return _lib.GqaCacheDesc(*self._head, 0, 0, 0)


def gqa_append(cache: GqaCache, block_table: torch.Tensor, seqs: torch.Tensor, positions: torch.Tensor, q: Optional[torch.Tensor],
               k: torch.Tensor, v: torch.Tensor, inv_freq: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
               rope_scale: float = 1.0, interleaved: bool = False) -> Optional[torch.Tensor]:
    """Write the keys and values of new tokens to the cache and turn their queries (vib3_launch_gqa_append).

    Token t is token positions[t] of sequence seqs[t] (int32 [tokens]; a negative sequence is padding, of which nothing is
    written). q [tokens, heads, dim], k and v [tokens, kv_heads, dim] (all f32, f16 or bf16) are the projections: each head's query and key is
    RMS-normalised with q_norm / k_norm ([dim], both of one type; None: as it is) and its first 2 * len(inv_freq) elements (a
    multiple of 16; None: none) rotated by positions[t] * inv_freq (f32) and scaled by rope_scale, in pairs (i, i + len(inv_freq))
    or, interleaved, (2i, 2i + 1). Returns q_out [tokens, heads, dim] in the cache's dtype (default: a new tensor; it may be q
    itself where their types are one). q None: keys and values only."""
    index, dt, dim = cache.index, cache.dtype, cache.dim
    desc = cache._desc(block_table)
    tokens = _dims(k, "k", _IN_DT, 3)[0]
    src, shape, one = k.dtype, (tokens, cache.kv_heads, dim), (tokens,)
    at_k, at_v = _rows(k, "k", src, shape, index), _rows(v, "v", src, shape, index)
    heads, qs, outs = 0, (0, 0, 0), (0, 0, 0)
    if q is not None:
        heads = _dims(q, "q", (src,), 3)[1]
        if heads < 1 or heads % cache.kv_heads:
            raise ValueError(f"{heads} heads over {cache.kv_heads} key/value heads")
        q_shape = (tokens, heads, dim)
        qs = (_rows(q, "q", src, q_shape, index), q.stride(0), q.stride(1))
        if q_out is None:
            q_out = torch.empty(q_shape, dtype=dt, device=q.device)
        outs = (_rows(q_out, "q_out", dt, q_shape, index), q_out.stride(0), q_out.stride(1))
        if tokens == 0:  # an empty tensor has no address: nothing to turn
            qs = outs = (0, 0, 0)
    norms, norm_dt = (0, 0), 0
    if q_norm is not None or k_norm is not None:
        kind = (q_norm if q_norm is not None else k_norm).dtype
        if kind not in _IN_DT:
            raise TypeError(f"q_norm and k_norm: unsupported dtype {kind}")
        norms = tuple(0 if w is None else _flat(w, n, kind, (dim,), index) for w, n in ((q_norm, "q_norm"), (k_norm, "k_norm")))
        norm_dt = _IN_DT[kind]
    freq, rot = 0, 0
    if inv_freq is not None:
        rot = 2 * _dims(inv_freq, "inv_freq", (torch.float32,), 1)[0]
        if rot % 16 or rot > dim:
            raise ValueError(f"inv_freq turns {rot} elements of a head of {dim}: it must be a multiple of 16 up to that")
        freq = _flat(inv_freq, "inv_freq", torch.float32, (rot // 2,), index)
    a = _lib.GqaAppendDesc(desc, tokens, heads, _flat(seqs, "seqs", _INT, one, index), _flat(positions, "positions", _INT, one, index),
                           _IN_DT[src], *qs, at_k, k.stride(0), k.stride(1), at_v, v.stride(0), v.stride(1), *norms, norm_dt, eps,
                           freq, rot, rope_scale, interleaved, *outs)
    _launch("vib3_launch_gqa_append", a, index)
    return q_out


class _Attention:
    """What the two forms share: the workspace and the output."""

    def _make(self, cache: GqaCache, heads: int, tokens: int, desc, size: str, what: str):
        n = getattr(_lib.load(), size)(desc)
        if n == 0:
            raise ValueError(f"{type(self).__name__}: unsupported heads={heads} over {cache.kv_heads}, or {what}")
        self.cache, self.heads = cache, heads
        self.workspace = torch.empty(n + 256, dtype=torch.uint8, device=cache.keys.device)
        self.out = torch.empty((tokens, heads, cache.dim), dtype=cache.dtype, device=cache.keys.device)
        self._space = ((self.workspace.data_ptr() + 255) // 256 * 256, n)

    def _to(self, q, out, most: int):
        """Addresses and strides of q and out, and out."""
        c = self.cache
        tokens = _dims(q, "q", (c.dtype,), 3)[0]
        if tokens > most:
            raise ValueError(f"{tokens} query tokens, made for {most}")
        shape = (tokens, self.heads, c.dim)
        at = _rows(q, "q", c.dtype, shape, c.index)
        if out is None:
            out = self.out[:tokens]
        return tokens, (at, q.stride(0), q.stride(1)), (_rows(out, "out", c.dtype, shape, c.index), out.stride(0), out.stride(1)), out


class GqaDecode(_Attention):
    """Attention of single query tokens over a paged cache: owns the workspace and the output for up to max_rows of them. Launches
    that may overlap (other streams, captured graphs) need a GqaDecode each."""

    def __init__(self, cache: GqaCache, heads: int, max_rows: int):
        self.max_rows = max_rows
        d = _lib.GqaDecodeDesc(cache._empty_desc(), max_rows, heads)
        self._make(cache, heads, max_rows, d, "vib3_gqa_decode_workspace_bytes", f"max_rows={max_rows}")

    def launch(self, q: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, scale: float,
               seqs: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Row r of q [rows, heads, dim] is the newest of the first lens[r] cached tokens of sequence seqs[r] (None: sequence r;
        int32 [rows]) and sees those or, with a window, the newest `window` and the first `sinks` of them. Returns out
        [rows, heads, dim] (default: the head of self.out), which is no part of q."""
        c = self.cache
        rows, qs, outs, out = self._to(q, out, self.max_rows)
        desc = c._desc(block_table)
        which = 0
        if seqs is not None:
            which = _flat(seqs, "seqs", _INT, (rows,), c.index)
        elif desc.num_seqs < rows:
            raise ValueError(f"block_table has {desc.num_seqs} sequences for {rows} rows and no seqs")
        a = _lib.GqaDecodeDesc(desc, rows, self.heads, which, _flat(lens, "lens", _INT, (rows,), c.index), *qs, scale, window, sinks,
                               *outs, *self._space)
        _launch("vib3_launch_gqa_decode", a, c.index)
        return out


class GqaChunk(_Attention):
    """Attention of each sequence's newest tokens over a paged cache: owns the workspace and the output for up to max_tokens query
    tokens of up to max_seqs sequences. Launches that may overlap (other streams, captured graphs) need a GqaChunk each."""

    def __init__(self, cache: GqaCache, heads: int, max_tokens: int, max_seqs: int):
        self.max_tokens, self.max_seqs = max_tokens, max_seqs
        d = _lib.GqaChunkDesc(cache._empty_desc(), heads, max_tokens)
        d.cache.num_seqs = max_seqs
        self._make(cache, heads, max_tokens, d, "vib3_gqa_chunk_workspace_bytes", f"max_tokens={max_tokens}, max_seqs={max_seqs}")

    def launch(self, q: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor, lens: torch.Tensor, scale: float,
               window: int = 0, sinks: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Sequence s (a row of block_table) has the queries cu_q[s]..cu_q[s + 1] of q [tokens, heads, dim] (int32 [seqs + 1]), the
        newest of its first lens[s] cached tokens (int32 [seqs]). Each sees the tokens up to its own or, with a window, the
        newest `window` and the first `sinks` of them. Returns out [tokens, heads, dim] (default: the head of self.out), which is no
        part of q."""
        c = self.cache
        tokens, qs, outs, out = self._to(q, out, self.max_tokens)
        desc = c._desc(block_table)
        seqs = desc.num_seqs
        if seqs > self.max_seqs:
            raise ValueError(f"{seqs} sequences, made for {self.max_seqs}")
        a = _lib.GqaChunkDesc(desc, self.heads, tokens, _flat(cu_q, "cu_q", _INT, (seqs + 1,), c.index),
                              _flat(lens, "lens", _INT, (seqs,), c.index), *qs, scale, window, sinks, *outs, *self._space)
        _launch("vib3_launch_gqa_chunk", a, c.index)
        return out
