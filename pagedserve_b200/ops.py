"""Tensor-level API over the C ABI: the batched hot path the engine calls.

* ``reshape_and_cache``  one launch per layer for all new tokens (replaces the
  per-token ``PagedKVCache.write_token`` loop,
  pagedserve/attention/batched_paged_attention.py:115-124)
* ``paged_decode``       split-K GQA decode over the paged pool (replaces
  pagedserve/attention/triton_paged_decode.py:10-95)
* ``varlen_prefill``     packed ragged causal prefill (replaces the per-request
  prefill of pagedserve/attention/qwen_paged_attention.py:121-128)
* ``pack_step``          GPU-side ragged-batch metadata for one engine step
  (replaces pagedserve/attention/triton_paged_decode.py:134-154)
* ``select_tokens``      greedy next token + stop check of every row on the
  device (replaces ``logits[:, -1, :].argmax`` and the per-row ``.item()``
  loop of pagedserve/engine/continuous_batcher.py:333-360)
* ``reshape_and_cache_int4``, ``rope_reshape_and_cache_int4``,
  ``gather_cache_int4``, ``paged_decode_int4``, ``paged_prefill_int4``  the
  write, read-back and attention over a pool of 4-bit codes
* ``extend_step``, ``trim_tables``  ``pack_step`` with the block allocation
  on the device too, and its reverse (``BlockManager``'s free list as a ring)
* ``fork_tables``, ``copy_blocks``, ``release_tables``  rows that share pages:
  several continuations of one prompt
* ``paged_decode_shared``  ``paged_decode`` for a batch that shares long prefixes
* ``verify_tokens``      drafted tokens against the target's probabilities, and
  sampling at a temperature, from given random numbers

Every function requires CUDA tensors, launches on the current stream and
returns without synchronising.  There is no CPU path.
"""

from __future__ import annotations

import ctypes
import functools
import math
import threading

import torch

from . import _native

_DTYPES = {torch.float32: _native.PSB_F32, torch.float16: _native.PSB_F16, torch.bfloat16: _native.PSB_BF16}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise ValueError(f"Unsupported dtype {dtype}") from None


try:  # the raw handle of the current stream, without building a Stream object (as torch's own codegen does)
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:  # pragma: no cover - older torch
    _raw_stream = None


def _stream(device: torch.device) -> int:
    if _raw_stream is not None:
        return _raw_stream(device.index if device.index is not None else torch.cuda.current_device())
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("B200 paged attention requires CUDA tensors")


def _pool_geometry(k_cache: torch.Tensor, v_cache: torch.Tensor):
    if k_cache.ndim != 5 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache/v_cache must be [num_layers, num_blocks, num_kv_heads, block_size, head_dim]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("KV pools must be contiguous")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache dtypes differ")
    return tuple(int(x) for x in k_cache.shape)


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, layer: int, error_flag: torch.Tensor | None = None) -> None:
    """Scatter ``key, value [T, Hkv, D]`` into ``k_cache/v_cache[layer]`` at ``slot_mapping [T]`` (int64).

    Bit-exact with ``PagedKVCache.write_token`` (paged_kv_cache.py:187-200); a
    negative slot writes nothing.
    """
    _require_cuda(key, value, k_cache, v_cache, slot_mapping)
    nl, nb, hkv, bs, d = _pool_geometry(k_cache, v_cache)
    if key.ndim != 3 or key.shape[1:] != (hkv, d) or value.shape != key.shape:
        raise ValueError(f"key/value must be [T, {hkv}, {d}]")
    if key.dtype != k_cache.dtype or value.dtype != k_cache.dtype:
        raise ValueError("key/value dtype must match the cache dtype")
    if key.stride(2) != 1 or value.stride(2) != 1:
        raise ValueError("key/value need unit stride along head_dim")
    if slot_mapping.dtype != torch.int64 or slot_mapping.ndim != 1 or slot_mapping.shape[0] != key.shape[0]:
        raise ValueError("slot_mapping must be int64 [T]")
    if not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.contiguous()
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    lib = _native.load()
    _native.check(lib.psb_reshape_and_cache(
        key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
        k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), key.shape[0], layer, nl, nb, hkv, bs, d,
        dtype_code(k_cache.dtype), _ptr(error_flag), _stream(key.device)), "reshape_and_cache")


def rope_reshape_and_cache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cos: torch.Tensor,
                           sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                           layer: int, query_out: torch.Tensor | None = None,
                           key_out: torch.Tensor | None | bool = None,
                           error_flag: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary embedding of ``query [T, Hq, D]`` and ``key [T, Hkv, D]`` with
    the per-token ``cos, sin [T, D]`` rows, fused with the slot-mapped write
    of the rotated keys and of ``value`` into ``k_cache/v_cache[layer]``
    (psb_rope_reshape_and_cache; bit-exact with the reference's
    ``apply_rotary_pos_emb`` then ``write_token``).

    Returns ``(query_out, key_out)``: ``query_out`` defaults to a new tensor
    (pass ``query`` to rotate in place); ``key_out`` defaults to a new tensor
    holding the rotated keys, ``False`` skips it (the pool still gets them).
    """
    _require_cuda(query, key, value, cos, sin, k_cache, v_cache, slot_mapping)
    nl, nb, hkv, bs, d = _pool_geometry(k_cache, v_cache)
    if query.ndim != 3 or query.shape[2] != d:
        raise ValueError(f"query must be [T, Hq, {d}]")
    t = query.shape[0]
    if key.shape != (t, hkv, d) or value.shape != (t, hkv, d):
        raise ValueError(f"key/value must be [{t}, {hkv}, {d}]")
    cos = cos.reshape(-1, d)
    sin = sin.reshape(-1, d)
    if cos.shape[0] != t or sin.shape != cos.shape:
        raise ValueError(f"cos/sin must hold one [{d}] row per token")
    if cos.stride(1) != 1 or sin.stride(1) != 1 or cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    for x in (query, key, value, cos, sin):
        if x.dtype != k_cache.dtype:
            raise ValueError("query/key/value/cos/sin dtype must match the cache dtype")
        if x.stride(-1) != 1:
            raise ValueError("unit stride along head_dim is required")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (t,):
        raise ValueError("slot_mapping must be int64 [T]")
    slot_mapping = slot_mapping.contiguous()
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    if query_out is None:
        query_out = torch.empty_like(query)
    if query_out.shape != query.shape or query_out.dtype != query.dtype or query_out.stride(2) != 1:
        raise ValueError("query_out must match query's shape and dtype with unit stride along head_dim")
    if key_out is None:
        key_out = torch.empty_like(key)
    elif key_out is False:
        key_out = None
    if key_out is not None and (key_out.shape != key.shape or key_out.dtype != key.dtype or key_out.stride(2) != 1):
        raise ValueError("key_out must match key's shape and dtype with unit stride along head_dim")
    lib = _native.load()
    _native.check(lib.psb_rope_reshape_and_cache(
        query.data_ptr(), query.stride(0), query.stride(1), query_out.data_ptr(), query_out.stride(0),
        query_out.stride(1), key.data_ptr(), key.stride(0), key.stride(1), _ptr(key_out),
        key_out.stride(0) if key_out is not None else 0, key_out.stride(1) if key_out is not None else 0,
        value.data_ptr(), value.stride(0), value.stride(1), cos.data_ptr(), sin.data_ptr(), cos.stride(0),
        k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), t, query.shape[1], layer, nl, nb, hkv, bs, d,
        dtype_code(k_cache.dtype), _ptr(error_flag), _stream(query.device)), "rope_reshape_and_cache")
    return query_out, key_out


class DecodeWorkspace:
    """Split-K scratch for ``paged_decode``: one growable buffer per device.

    The first bytes hold per-(sequence, kv head) arrival counters that must be
    zero before a launch; every launch leaves them zero, so the buffer is
    zeroed only when it is (re)allocated.  Launches sharing a workspace must be
    ordered (same stream), which is what the per-device default gives.
    """

    _lock = threading.Lock()
    _per_device: dict[int, "DecodeWorkspace"] = {}

    def __init__(self, device: torch.device):
        self.device = device
        self.buffer = torch.empty(0, dtype=torch.uint8, device=device)

    @classmethod
    def for_device(cls, device: torch.device) -> "DecodeWorkspace":
        idx = device.index if device.index is not None else torch.cuda.current_device()
        with cls._lock:
            ws = cls._per_device.get(idx)
            if ws is None:
                ws = cls._per_device[idx] = DecodeWorkspace(torch.device("cuda", idx))
            return ws

    def get(self, nbytes: int, batch: int, hkv: int) -> torch.Tensor:
        if self.buffer.numel() < nbytes:
            self.buffer = torch.empty(max(nbytes, 2 * self.buffer.numel()), dtype=torch.uint8, device=self.device)
            lib = _native.load()
            # zero the whole buffer once: covers the counters of any later, larger batch too
            self.buffer.zero_()
        return self.buffer


@functools.lru_cache(maxsize=256)
def decode_workspace_bytes(batch: int, q_heads: int, hkv: int, head_dim: int, block_size: int, max_context: int,
                           dtype: torch.dtype) -> int:
    lib = _native.load()
    return int(lib.psb_paged_decode_workspace_size(batch, q_heads, hkv, head_dim, block_size, max_context,
                                                   dtype_code(dtype)))


def paged_decode(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, layer: int, scale: float | None = None, out: torch.Tensor | None = None,
                 max_context: int | None = None, workspace: torch.Tensor | None = None,
                 error_flag: torch.Tensor | None = None, new_key: torch.Tensor | None = None,
                 new_value: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention for ``query [B, Hq, D]`` (or ``[B, Hq, 1, D]``) over the paged pool.

    ``block_tables [B, M]`` int32 and ``context_lens [B]`` int32 live on the
    device; ``max_context`` (default ``M * block_size``) bounds every length.
    With ``new_key`` / ``new_value`` (``[B, Hkv, D]`` or ``[B, Hkv, 1, D]``)
    the same launch first stores row b's new token at position
    ``context_lens[b] - 1`` through its block table (psb_paged_decode_append).
    Returns ``out`` with ``query``'s shape and dtype.
    """
    _require_cuda(query, k_cache, v_cache, block_tables, context_lens)
    nl, nb, hkv, bs, d = _pool_geometry(k_cache, v_cache)
    q3 = query.squeeze(2) if query.ndim == 4 else query
    if q3.ndim != 3 or q3.shape[2] != d:
        raise ValueError("query must be [B, Hq, D] or [B, Hq, 1, D]")
    bsz, hq, _ = q3.shape
    if bsz == 0:
        raise ValueError("Batch must not be empty")
    if hq % hkv:
        raise ValueError("Query heads must be divisible by KV heads")
    if q3.dtype != k_cache.dtype:
        raise ValueError("Query dtype must match cache dtype")
    if q3.stride(2) != 1:
        q3 = q3.contiguous()
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2 or block_tables.shape[0] != bsz:
        raise ValueError("block_tables must be int32 [B, max_blocks]")
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    if context_lens.dtype != torch.int32 or context_lens.shape != (bsz,):
        raise ValueError("context_lens must be int32 [B]")
    context_lens = context_lens.contiguous()
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    if max_context is None:
        max_context = block_tables.shape[1] * bs
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if out is None:
        out = torch.empty_like(query)
    o3 = out.squeeze(2) if out.ndim == 4 else out
    if o3.shape != q3.shape or o3.stride(2) != 1 or o3.dtype != q3.dtype:
        raise ValueError("out must match query's shape/dtype with unit stride along head_dim")
    need = decode_workspace_bytes(bsz, hq, hkv, d, bs, max_context, q3.dtype)
    if workspace is None:
        workspace = DecodeWorkspace.for_device(query.device).get(need, bsz, hkv)
    lib = _native.load()
    if (new_key is None) != (new_value is None):
        raise ValueError("new_key and new_value go together")
    if new_key is not None:
        _require_cuda(new_key, new_value)
        nk = new_key.squeeze(2) if new_key.ndim == 4 else new_key
        nv = new_value.squeeze(2) if new_value.ndim == 4 else new_value
        for t in (nk, nv):
            if t.shape != (bsz, hkv, d) or t.dtype != q3.dtype or t.stride(2) != 1:
                raise ValueError(f"new K/V must be [{bsz}, {hkv}, {d}] {q3.dtype} with unit stride along head_dim")
        _native.check(lib.psb_paged_decode_append(
            q3.data_ptr(), q3.stride(0), q3.stride(1), o3.data_ptr(), o3.stride(0), o3.stride(1), k_cache.data_ptr(),
            v_cache.data_ptr(), nk.data_ptr(), nk.stride(0), nk.stride(1), nv.data_ptr(), nv.stride(0), nv.stride(1),
            block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), bsz, hq, layer, nl, nb, hkv, bs,
            d, dtype_code(q3.dtype), int(max_context), scale, workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _ptr(error_flag), _stream(query.device)),
            "paged_decode_append")
        return out
    _native.check(lib.psb_paged_decode(
        q3.data_ptr(), q3.stride(0), q3.stride(1), o3.data_ptr(), o3.stride(0), o3.stride(1), k_cache.data_ptr(),
        v_cache.data_ptr(), block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), bsz, hq, layer,
        nl, nb, hkv, bs, d, dtype_code(q3.dtype), int(max_context), scale, workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), _ptr(error_flag), _stream(query.device)), "paged_decode")
    return out


class DecodeLaunch:
    """The launch arguments of one decode batch that stay the same for all
    the layer calls of an iteration (pools, device table and lengths,
    geometry, workspace), kept by the reference-facing wrappers next to the
    batch's metadata as one ``psb_decode_args`` struct, so a repeat layer call
    passes only the query, output, new rows, layer and stream
    (``psb_paged_decode_args``).

    Built from arguments the wrappers have already checked: pools contiguous
    and of the query's dtype, device table ``[B, M]`` int32 with unit inner
    stride and contiguous int32 lengths.  The workspace it sized, and the
    table and lengths, are held here, so a later growth of the per-device
    workspace never leaves this launch pointing at freed memory."""

    __slots__ = ("lib", "k_ptr", "v_ptr", "batch", "q_heads", "dtype", "dev", "ws", "keep", "args", "args_ptr")

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                 batch: int, q_heads: int, max_context: int, dtype: torch.dtype):
        nl, nb, hkv, bs, d = (int(x) for x in k_cache.shape)
        if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
            raise ValueError("KV pools must be contiguous")
        self.lib = _native.load()
        self.k_ptr, self.v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
        self.batch, self.q_heads, self.dtype = int(batch), int(q_heads), dtype
        self.dev = k_cache.device.index if k_cache.device.index is not None else torch.cuda.current_device()
        need = decode_workspace_bytes(self.batch, self.q_heads, hkv, d, bs, int(max_context), dtype)
        self.ws = DecodeWorkspace.for_device(k_cache.device).get(need, self.batch, hkv)
        self.keep = (tables, lengths)
        self.args = _native.DecodeArgs(
            k_cache=self.k_ptr, v_cache=self.v_ptr, block_tables=tables.data_ptr(), table_stride=tables.stride(0),
            context_lens=lengths.data_ptr(), num_blocks=nb, workspace=self.ws.data_ptr(),
            workspace_bytes=self.ws.numel() * self.ws.element_size(), error_flag=None, batch=self.batch,
            q_heads=self.q_heads, num_layers=nl, num_kv_heads=hkv, block_size=bs, head_dim=d,
            dtype=_DTYPES[dtype], max_context=int(max_context), scale=1.0 / math.sqrt(d), reserved=0)
        self.args_ptr = ctypes.addressof(self.args)

    def with_lengths(self, lengths: torch.Tensor) -> "DecodeLaunch":
        """The same launch over another lengths array (contiguous int32 [B]
        on the same device) with the same table and bound."""
        new = object.__new__(DecodeLaunch)
        for name in ("lib", "k_ptr", "v_ptr", "batch", "q_heads", "dtype", "dev", "ws"):
            setattr(new, name, getattr(self, name))
        new.keep = (self.keep[0], lengths)
        new.args = _native.DecodeArgs.from_buffer_copy(self.args)
        new.args.context_lens = lengths.data_ptr()
        new.args_ptr = ctypes.addressof(new.args)
        return new

    def matches(self, k_cache: torch.Tensor, v_cache: torch.Tensor, query: torch.Tensor) -> bool:
        return (k_cache.data_ptr() == self.k_ptr and v_cache.data_ptr() == self.v_ptr
                and query.shape[0] == self.batch and query.shape[1] == self.q_heads and query.dtype == self.dtype)

    def __call__(self, query: torch.Tensor, layer: int, new_key: torch.Tensor | None = None,
                 new_value: torch.Tensor | None = None) -> torch.Tensor:
        """Decode (with ``new_key``/``new_value``: the fused write + decode)
        for ``query [B, Hq, (1,) D]``; returns a new output of its shape."""
        if query.stride(-1) != 1:
            query = query.contiguous()
        out = torch.empty_like(query)
        stream = _raw_stream(self.dev) if _raw_stream is not None else torch.cuda.current_stream(self.dev).cuda_stream
        if new_key is None:
            _native.check(self.lib.psb_paged_decode_args(
                self.args_ptr, query.data_ptr(), query.stride(0), query.stride(1), out.data_ptr(), out.stride(0),
                out.stride(1), None, 0, 0, None, 0, 0, layer, stream), "paged_decode")
            return out
        if new_key.stride(-1) != 1:
            new_key = new_key.contiguous()
        if new_value.stride(-1) != 1:
            new_value = new_value.contiguous()
        _native.check(self.lib.psb_paged_decode_args(
            self.args_ptr, query.data_ptr(), query.stride(0), query.stride(1), out.data_ptr(), out.stride(0),
            out.stride(1), new_key.data_ptr(), new_key.stride(0), new_key.stride(1), new_value.data_ptr(),
            new_value.stride(0), new_value.stride(1), layer, stream), "paged_decode_append")
        return out


def varlen_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int,
                   scale: float | None = None, out: torch.Tensor | None = None,
                   error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """Packed causal prefill: ``q [T, Hq, D]``, ``k, v [T, Hkv, D]``, ``cu_seqlens [B+1]`` int32."""
    _require_cuda(q, k, v, cu_seqlens)
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("q must be [T, Hq, D] and k, v [T, Hkv, D]")
    t, hq, d = q.shape
    hkv = k.shape[1]
    if hq % hkv:
        raise ValueError("Query heads must be divisible by KV heads")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q, k, v dtypes differ")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be int32 [B+1]")
    q, k, v = (x if x.stride(2) == 1 else x.contiguous() for x in (q, k, v))
    cu_seqlens = cu_seqlens.contiguous()
    if out is None:
        out = torch.empty_like(q)
    if out.shape != q.shape or out.stride(2) != 1:
        raise ValueError("out must match q with unit stride along head_dim")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    lib = _native.load()
    _native.check(lib.psb_varlen_prefill(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
        v.stride(1), out.data_ptr(), out.stride(0), out.stride(1), cu_seqlens.data_ptr(), cu_seqlens.shape[0] - 1,
        t, int(max_seqlen), hq, hkv, d, dtype_code(q.dtype), scale, _ptr(error_flag), _stream(q.device)),
        "varlen_prefill")
    return out


def paged_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, layer: int,
                  scale: float | None = None, out: torch.Tensor | None = None, max_context: int | None = None,
                  error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """Prefix-aware (chunked) causal prefill over the paged pool.

    ``q [T, Hq, D]`` packs each sequence's new rows (``cu_seqlens [B+1]``
    int32); sequence ``b`` holds ``context_lens[b]`` tokens in the pool,
    read through ``block_tables[b]``, its query rows being the last
    ``cu_seqlens[b+1] - cu_seqlens[b]`` of them (their K/V already written,
    e.g. by ``rope_reshape_and_cache``).  Row ``i`` of sequence ``b`` attends
    to positions ``0 .. context_lens[b] - n_b + i``: the reference's
    ``paged_attention(query, cache, request, layer, query_start_position)``
    (pagedserve/attention/paged_attention.py:10-146) for a whole batch.
    """
    _require_cuda(q, k_cache, v_cache, block_tables, context_lens, cu_seqlens)
    nl, nb, hkv, bs, d = _pool_geometry(k_cache, v_cache)
    if q.ndim != 3 or q.shape[2] != d:
        raise ValueError(f"q must be [T, Hq, {d}]")
    t, hq, _ = q.shape
    if hq % hkv:
        raise ValueError("Query heads must be divisible by KV heads")
    if q.dtype != k_cache.dtype:
        raise ValueError("q dtype must match the cache dtype")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be int32 [B+1]")
    batch = cu_seqlens.shape[0] - 1
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2 or block_tables.shape[0] != batch:
        raise ValueError("block_tables must be int32 [B, max_blocks]")
    if context_lens.dtype != torch.int32 or context_lens.shape != (batch,):
        raise ValueError("context_lens must be int32 [B]")
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    if q.stride(2) != 1:
        q = q.contiguous()
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    cu_seqlens, context_lens = cu_seqlens.contiguous(), context_lens.contiguous()
    if max_context is None:
        max_context = block_tables.shape[1] * bs
    if out is None:
        out = torch.empty_like(q)
    if out.shape != q.shape or out.stride(2) != 1 or out.dtype != q.dtype:
        raise ValueError("out must match q with unit stride along head_dim")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    lib = _native.load()
    _native.check(lib.psb_paged_prefill(
        q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(),
        block_tables.stride(0), context_lens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1),
        cu_seqlens.data_ptr(), batch, t, int(max_seqlen), int(max_context), hq, layer, nl, nb, hkv, bs, d,
        dtype_code(q.dtype), scale, _ptr(error_flag), _stream(q.device)), "paged_prefill")
    return out


def pack_step(table_store: torch.Tensor, req_rows: torch.Tensor, starts: torch.Tensor, query_lens: torch.Tensor,
              total: int, block_size: int, out_width: int | None = None, error_flag: torch.Tensor | None = None,
              out: tuple | None = None):
    """Build one step's ragged-batch metadata on the GPU.

    ``table_store [R, W]`` int32 holds every live request's block table (one
    row each); ``req_rows, starts, query_lens [B]`` int32 are the scheduler's
    step plan.  Returns ``(cu_seqlens, context_lens, slot_mapping, positions,
    block_tables)``, written into ``out`` (the same five tensors, e.g. the
    static buffers of a captured step) when given.
    """
    _require_cuda(table_store, req_rows, starts, query_lens)
    for name, x in (("req_rows", req_rows), ("starts", starts), ("query_lens", query_lens)):
        if x.dtype != torch.int32 or x.ndim != 1:
            raise ValueError(f"{name} must be int32 [B]")
    if table_store.dtype != torch.int32 or table_store.ndim != 2 or table_store.stride(1) != 1:
        raise ValueError("table_store must be int32 [R, W] with unit column stride")
    bsz = req_rows.shape[0]
    out_width = table_store.shape[1] if out_width is None else int(out_width)
    dev = table_store.device
    if out is None:
        cu = torch.empty(bsz + 1, dtype=torch.int32, device=dev)
        ctx = torch.empty(bsz, dtype=torch.int32, device=dev)
        slots = torch.empty(total, dtype=torch.int64, device=dev)
        pos = torch.empty(total, dtype=torch.int64, device=dev)
        tables = torch.empty((bsz, out_width), dtype=torch.int32, device=dev)
    else:
        cu, ctx, slots, pos, tables = out
        ok = (cu.shape == (bsz + 1,) and cu.dtype == torch.int32 and ctx.shape == (bsz,) and ctx.dtype == torch.int32
              and slots.shape == (total,) and slots.dtype == torch.int64 and pos.shape == (total,)
              and pos.dtype == torch.int64 and tables.shape == (bsz, out_width) and tables.dtype == torch.int32
              and all(t.is_contiguous() for t in out))
        if not ok:
            raise ValueError("out must be contiguous (cu_seqlens [B+1] i32, context_lens [B] i32, slot_mapping [T] "
                             "i64, positions [T] i64, block_tables [B, out_width] i32)")
    lib = _native.load()
    _native.check(lib.psb_pack_step(
        table_store.data_ptr(), table_store.stride(0), table_store.shape[0], req_rows.contiguous().data_ptr(),
        starts.contiguous().data_ptr(), query_lens.contiguous().data_ptr(), bsz, int(total), int(block_size),
        cu.data_ptr(), ctx.data_ptr(), slots.data_ptr(), pos.data_ptr(), tables.data_ptr(), out_width,
        _ptr(error_flag), _stream(dev)), "pack_step")
    return cu, ctx, slots, pos, tables


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm of ``x [R, H]`` (Qwen2RMSNorm), or, with ``residual [R, H]``,
    ``residual += x`` (rounded, in place) followed by RMSNorm of the sum, in
    one launch (psb_add_rms_norm).  Returns ``out``."""
    _require_cuda(x, weight)
    if x.ndim != 2 or weight.shape != (x.shape[1],):
        raise ValueError("x must be [R, H] and weight [H]")
    if x.stride(1) != 1 or weight.stride(0) != 1:
        raise ValueError("x and weight need unit stride along H")
    if out is None:
        out = torch.empty_like(x)
    for t in (out,) + ((residual,) if residual is not None else ()):
        if t.shape != x.shape or t.dtype != x.dtype or t.stride(1) != 1:
            raise ValueError("out / residual must match x's shape and dtype with unit stride along H")
    if weight.dtype != x.dtype:
        raise ValueError("weight dtype must match x")
    lib = _native.load()
    _native.check(lib.psb_add_rms_norm(
        x.data_ptr(), x.stride(0), _ptr(residual), residual.stride(0) if residual is not None else 0,
        weight.data_ptr(), out.data_ptr(), out.stride(0), x.shape[0], x.shape[1], float(eps), dtype_code(x.dtype),
        _stream(x.device)), "add_rms_norm")
    return out


def silu_and_mul(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(gate) * up`` of a fused ``gate_up [R, 2I]`` projection -> ``[R, I]`` (psb_silu_and_mul)."""
    _require_cuda(gate_up)
    if gate_up.ndim != 2 or gate_up.shape[1] % 2 or gate_up.stride(1) != 1:
        raise ValueError("gate_up must be [R, 2 * I] with unit column stride")
    rows, inter = gate_up.shape[0], gate_up.shape[1] // 2
    if out is None:
        out = torch.empty((rows, inter), dtype=gate_up.dtype, device=gate_up.device)
    if out.shape != (rows, inter) or out.dtype != gate_up.dtype or out.stride(1) != 1:
        raise ValueError(f"out must be [{rows}, {inter}] of gate_up's dtype with unit column stride")
    lib = _native.load()
    _native.check(lib.psb_silu_and_mul(gate_up.data_ptr(), gate_up.stride(0), out.data_ptr(), out.stride(0), rows,
                                       inter, dtype_code(gate_up.dtype), _stream(gate_up.device)), "silu_and_mul")
    return out


SELECT_DONE, SELECT_EOS, SELECT_LIMIT = 1, 2, 4


def select_tokens(logits: torch.Tensor, eos_ids: torch.Tensor, remaining: torch.Tensor,
                  tokens: torch.Tensor | None = None, status: torch.Tensor | None = None,
                  error_flag: torch.Tensor | None = None, ctas_per_row: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Greedy next token of every row and the reference's stop test, in one launch.

    ``logits`` is ``[B, V]`` or the model's ``[B, S, V]`` (the last position is
    used, as ``logits[:, -1, :]``), unit stride along V.  ``eos_ids`` int64
    ``[E]`` (E <= 64), ``remaining`` int32 ``[B]``: tokens each request may
    still generate, decremented in place.  Returns ``(tokens [B] int64,
    status [B] uint8)``: ``tokens`` is ``argmax(dim=-1)`` with torch's rules
    (first maximum, NaN largest); ``status`` holds SELECT_DONE (the request
    finishes: EOS or its last allowed token), SELECT_EOS, and SELECT_LIMIT
    (no tokens were left: the reference's add_generated_token raises; the
    row is also flagged in ``error_flag`` with 64).
    """
    _require_cuda(logits, eos_ids, remaining)
    if logits.ndim == 3:
        logits = logits[:, -1, :]
    if logits.ndim != 2:
        raise ValueError("logits must be [B, V] or [B, S, V]")
    b, v = int(logits.shape[0]), int(logits.shape[1])
    if v == 0:
        raise ValueError("logits have an empty vocabulary axis")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    if eos_ids.dtype != torch.int64 or eos_ids.ndim != 1 or eos_ids.shape[0] > 64:
        raise ValueError("eos_ids must be int64 [E] with E <= 64")
    if not eos_ids.is_contiguous():
        eos_ids = eos_ids.contiguous()
    if remaining.dtype != torch.int32 or remaining.shape != (b,) or not remaining.is_contiguous():
        raise ValueError("remaining must be a contiguous int32 [B] tensor (updated in place)")
    if tokens is None:
        tokens = torch.empty(b, dtype=torch.int64, device=logits.device)
    if status is None:
        status = torch.empty(b, dtype=torch.uint8, device=logits.device)
    if tokens.dtype != torch.int64 or tokens.shape != (b,) or not tokens.is_contiguous():
        raise ValueError("tokens must be a contiguous int64 [B] tensor")
    if status.dtype != torch.uint8 or status.shape != (b,) or not status.is_contiguous():
        raise ValueError("status must be a contiguous uint8 [B] tensor")
    if not 0 <= ctas_per_row <= 8:
        raise ValueError("ctas_per_row must be 0 (auto) or 1..8")
    if b == 0:
        return tokens, status
    row_stride = int(logits.stride(0)) if b > 1 else v
    lib = _native.load()
    _native.check(lib.psb_select_tokens(
        logits.data_ptr(), row_stride, b, v, dtype_code(logits.dtype), eos_ids.data_ptr() if eos_ids.numel() else None,
        int(eos_ids.shape[0]), remaining.data_ptr(), tokens.data_ptr(), status.data_ptr(), ctas_per_row,
        _ptr(error_flag), _stream(logits.device)), "select_tokens")
    return tokens, status


# -- 4-bit KV pool ---------------------------------------------------------------------------------------------
#
# A call's host time is most of a small batch's step: each function first hands
# its arguments to its counterpart in csrc/calls.cpp, which checks and launches
# the ordinary case in one call.  What that does not take (it returns None) is
# checked here, with the errors' wording, and launched through the C ABI with
# the copies that unusual strides need.

INT4_MAX_HEAD_DIM = 256


def _cuda_index(*tensors: torch.Tensor | None) -> int:
    """The CUDA device index all of ``tensors`` are on (the last of a call's checks)."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"every tensor must be on {tensors[0].device}: got one on {t.device}")
    if dev < 0:
        raise ValueError("B200 paged attention requires CUDA tensors")
    return dev


def _call(dev: int, fn, what: str, *args) -> None:
    """``fn(*args, stream)`` on ``dev``'s current stream with ``dev`` the current device."""
    if _raw_stream is not None and torch._C._cuda_getDevice() == dev:
        status = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    if status != _native.PSB_OK:
        _native.check(status, what)


def _done(result, what: str):
    """What a call of csrc/calls.cpp returned: its result, or a failure's status."""
    if type(result) is int:
        _native.check(result, what)
    return result


def _int4_geometry(kv_codes: torch.Tensor, kv_params: torch.Tensor):
    """(layers, blocks, kv heads, block size, head dim, dtype, its code) of a 4-bit pool."""
    cs, ps = kv_codes.shape, kv_params.shape
    if len(cs) != 6 or cs[3] != 2 or kv_codes.dtype != torch.uint8:
        raise ValueError("kv_codes must be uint8 [num_layers, num_blocks, num_kv_heads, 2, block_size, head_dim / 2]")
    nl, nb, hkv, _, bs, half = cs
    if ps != (nl, nb, hkv, 2, bs, 2):
        raise ValueError("kv_params must be [num_layers, num_blocks, num_kv_heads, 2, block_size, 2] like kv_codes")
    dtype = kv_params.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"Unsupported dtype {dtype}")
    if not (kv_codes.is_contiguous() and kv_params.is_contiguous()):
        raise ValueError("KV pools must be contiguous")
    if (kv_codes.data_ptr() | kv_params.data_ptr()) & 15:
        raise ValueError("KV pools must start on 16 bytes")
    if half > INT4_MAX_HEAD_DIM // 2:
        raise ValueError(f"4-bit pools hold head_dim up to {INT4_MAX_HEAD_DIM}")
    return nl, nb, hkv, bs, 2 * half, dtype, code


def _check_flag(error_flag: torch.Tensor | None) -> None:
    if error_flag is not None and (error_flag.dtype != torch.int32 or error_flag.numel() < 1):
        raise ValueError("error_flag must be an int32 tensor of at least one element")


def _int4_rows(key: torch.Tensor, value: torch.Tensor, hkv: int, d: int, dtype) -> int:
    shape = key.shape
    if len(shape) != 3 or shape[1] != hkv or shape[2] != d or value.shape != shape:
        raise ValueError(f"key/value must be [T, {hkv}, {d}]")
    if key.dtype != dtype or value.dtype != dtype:
        raise ValueError("key/value dtype must match the cache dtype (that of kv_params)")
    if key.stride()[2] != 1 or value.stride()[2] != 1:
        raise ValueError("key/value need unit stride along head_dim")
    return shape[0]


def _int4_slots(slot_mapping: torch.Tensor, t: int) -> torch.Tensor:
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (t,):
        raise ValueError("slot_mapping must be int64 [T]")
    return slot_mapping.contiguous()


def reshape_and_cache_int4(key: torch.Tensor, value: torch.Tensor, kv_codes: torch.Tensor, kv_params: torch.Tensor,
                           slot_mapping: torch.Tensor, layer: int, error_flag: torch.Tensor | None = None) -> None:
    """``reshape_and_cache`` into a 4-bit pool (psb_reshape_and_cache_int4).

    ``key, value [T, Hkv, D]`` of ``kv_params``' dtype are quantised row by
    row (one step and one offset per token and kv head) into
    ``kv_codes[layer]`` / ``kv_params[layer]`` at ``slot_mapping [T]`` (int64;
    negative: nothing is written; live slots distinct).
    """
    if key.is_cuda:
        done = (_native._calls or _native.calls()).write(key, value, kv_codes, kv_params, slot_mapping, layer, error_flag)
        if done is not None:
            _done(done, "reshape_and_cache_int4")
            return
    nl, nb, hkv, bs, d, dtype, code = _int4_geometry(kv_codes, kv_params)
    t = _int4_rows(key, value, hkv, d, dtype)
    slot_mapping = _int4_slots(slot_mapping, t)
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    _check_flag(error_flag)
    dev = _cuda_index(kv_codes, kv_params, key, value, slot_mapping, error_flag)
    ks, vs = key.stride(), value.stride()
    _call(dev, _native.load().psb_reshape_and_cache_int4, "reshape_and_cache_int4",
          key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1], kv_codes.data_ptr(), kv_params.data_ptr(),
          slot_mapping.data_ptr(), t, layer, nl, nb, hkv, bs, d, code, _ptr(error_flag))


def rope_reshape_and_cache_int4(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cos: torch.Tensor,
                                sin: torch.Tensor, kv_codes: torch.Tensor, kv_params: torch.Tensor,
                                slot_mapping: torch.Tensor, layer: int, query_out: torch.Tensor | None = None,
                                key_out: torch.Tensor | None | bool = None,
                                error_flag: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``rope_reshape_and_cache`` into a 4-bit pool
    (psb_rope_reshape_and_cache_int4): the rotated query and key are
    bit-identical to that call's, and the rotated key is what is quantised.

    Returns ``(query_out, key_out)`` with the same defaults: new tensors,
    ``query_out=query`` to rotate in place, ``key_out=False`` for none.
    """
    if query_out is None and query.is_cuda:
        done = (_native._calls or _native.calls()).rope_write(query, key, value, cos, sin, kv_codes, kv_params,
                                                              slot_mapping, layer, key_out, error_flag)
        if done is not None:
            return _done(done, "rope_reshape_and_cache_int4")
    nl, nb, hkv, bs, d, dtype, code = _int4_geometry(kv_codes, kv_params)
    shape = query.shape
    if len(shape) != 3 or shape[2] != d:
        raise ValueError(f"query must be [T, Hq, {d}]")
    t = shape[0]
    if _int4_rows(key, value, hkv, d, dtype) != t:
        raise ValueError(f"key/value must be [{t}, {hkv}, {d}]")
    if cos.shape != (t, d) or sin.shape != (t, d):
        cos, sin = cos.reshape(-1, d), sin.reshape(-1, d)
        if cos.shape[0] != t or sin.shape != cos.shape:
            raise ValueError(f"cos/sin must hold one [{d}] row per token")
    cst = cos.stride()
    if cst != sin.stride() or cst[1] != 1:
        cos, sin = cos.contiguous(), sin.contiguous()
        cst = (d, 1)
    if query.dtype != dtype or cos.dtype != dtype or sin.dtype != dtype:
        raise ValueError("query/key/value/cos/sin dtype must match the cache dtype (that of kv_params)")
    qs = query.stride()
    if qs[2] != 1:
        raise ValueError("unit stride along head_dim is required")
    slot_mapping = _int4_slots(slot_mapping, t)
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    _check_flag(error_flag)
    if query_out is None:
        query_out = torch.empty_like(query)
    elif query_out.shape != shape or query_out.dtype != dtype:
        raise ValueError("query_out must match query's shape and dtype with unit stride along head_dim")
    if key_out is None:
        key_out = torch.empty_like(key)
    elif key_out is False:
        key_out = None
    elif key_out.shape != key.shape or key_out.dtype != dtype:
        raise ValueError("key_out must match key's shape and dtype with unit stride along head_dim")
    qos, kos = query_out.stride(), key_out.stride() if key_out is not None else (0, 0, 1)
    if qos[2] != 1 or kos[2] != 1:
        raise ValueError("query_out / key_out need unit stride along head_dim")
    dev = _cuda_index(kv_codes, kv_params, query, key, value, cos, sin, slot_mapping, query_out, key_out, error_flag)
    ks, vs = key.stride(), value.stride()
    _call(dev, _native.load().psb_rope_reshape_and_cache_int4, "rope_reshape_and_cache_int4",
          query.data_ptr(), qs[0], qs[1], query_out.data_ptr(), qos[0], qos[1], key.data_ptr(), ks[0], ks[1],
          _ptr(key_out), kos[0], kos[1], value.data_ptr(), vs[0], vs[1], cos.data_ptr(), sin.data_ptr(), cst[0],
          kv_codes.data_ptr(), kv_params.data_ptr(), slot_mapping.data_ptr(), t, shape[1], layer, nl, nb, hkv, bs, d,
          code, _ptr(error_flag))
    return query_out, key_out


def gather_cache_int4(kv_codes: torch.Tensor, kv_params: torch.Tensor, slot_mapping: torch.Tensor, layer: int,
                      key_out: torch.Tensor | None = None, value_out: torch.Tensor | None = None,
                      error_flag: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(key, value) [T, Hkv, D]``: the values a 4-bit pool holds at
    ``slot_mapping [T]`` (int64; zeros for a negative slot), in ``kv_params``'
    dtype (psb_gather_cache_int4)."""
    if key_out is None and value_out is None and kv_codes.is_cuda:
        done = (_native._calls or _native.calls()).gather(kv_codes, kv_params, slot_mapping, layer, error_flag)
        if done is not None:
            return _done(done, "gather_cache_int4")
    nl, nb, hkv, bs, d, dtype, code = _int4_geometry(kv_codes, kv_params)
    t = slot_mapping.shape[0] if slot_mapping.ndim == 1 else -1
    slot_mapping = _int4_slots(slot_mapping, t)
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    _check_flag(error_flag)
    shape = (t, hkv, d)
    if key_out is None:
        key_out = kv_params.new_empty(shape)
    if value_out is None:
        value_out = kv_params.new_empty(shape)
    ks, vs = key_out.stride(), value_out.stride()
    if (key_out.shape != shape or value_out.shape != shape or key_out.dtype != dtype or value_out.dtype != dtype
            or ks[2] != 1 or vs[2] != 1):
        raise ValueError(f"key_out/value_out must be [{t}, {hkv}, {d}] {dtype} with unit stride along head_dim")
    dev = _cuda_index(kv_codes, kv_params, slot_mapping, key_out, value_out, error_flag)
    _call(dev, _native.load().psb_gather_cache_int4, "gather_cache_int4",
          kv_codes.data_ptr(), kv_params.data_ptr(), slot_mapping.data_ptr(), key_out.data_ptr(), ks[0], ks[1],
          value_out.data_ptr(), vs[0], vs[1], t, layer, nl, nb, hkv, bs, d, code, _ptr(error_flag))
    return key_out, value_out


@functools.lru_cache(maxsize=1024)
def decode_int4_workspace_bytes(batch: int, q_heads: int, hkv: int, head_dim: int, block_size: int, max_context: int,
                                dtype: torch.dtype) -> int:
    """Scratch bytes of ``paged_decode_int4`` (psb_paged_decode_int4_workspace_size)."""
    lib = _native.load()
    return int(lib.psb_paged_decode_int4_workspace_size(batch, q_heads, hkv, head_dim, block_size, max_context,
                                                        dtype_code(dtype)))


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    return (a.nbytes > 0 and b.nbytes > 0 and a.device == b.device
            and a.data_ptr() < b.data_ptr() + b.nbytes and b.data_ptr() < a.data_ptr() + a.nbytes)


def _check_workspace(workspace: torch.Tensor) -> None:
    if not workspace.is_contiguous() or workspace.data_ptr() % 16:
        raise ValueError("workspace must be contiguous and start on 16 bytes")


def paged_decode_int4(query: torch.Tensor, kv_codes: torch.Tensor, kv_params: torch.Tensor,
                      block_tables: torch.Tensor, context_lens: torch.Tensor, layer: int, scale: float | None = None,
                      out: torch.Tensor | None = None, max_context: int | None = None,
                      workspace: torch.Tensor | None = None, error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_decode`` over a 4-bit pool (psb_paged_decode_int4).

    ``query [B, Hq, D]`` or ``[B, Hq, 1, D]`` of ``kv_params``' dtype; tables,
    lengths, ``max_context`` and ``scale`` as in ``paged_decode``.  Each call
    takes its split-K scratch from PyTorch's allocator unless ``workspace``
    (``decode_int4_workspace_bytes``) is given, which calls that may overlap
    on the GPU must not share.

    bf16 and f16 with head_dim 64 or 128, ``block_size`` a multiple of 16, rows
    that start on 16 bytes and at most 2560 sequences run on the tensor cores;
    anything else, fp32 among it, on a CUDA-core kernel that takes 25 to 200
    times as long.  The tensor-core path rounds step * probability to f16's 11
    bits (f16: a relative error of 3e-4 against 64 bits, where fp32 arithmetic
    has 2e-4; bf16: the output's own rounding hides it).
    """
    if query.is_cuda:
        done = (_native._calls or _native.calls()).decode(query, kv_codes, kv_params, block_tables, context_lens, layer,
                                                          scale, out, max_context, workspace, error_flag)
        if done is not None:
            return _done(done, "paged_decode_int4")
    nl, nb, hkv, bs, d, dtype, code = _int4_geometry(kv_codes, kv_params)
    q3 = query.squeeze(2) if query.ndim == 4 else query
    shape = q3.shape
    if len(shape) != 3 or shape[2] != d:
        raise ValueError("query must be [B, Hq, D] or [B, Hq, 1, D]")
    bsz, hq, _ = shape
    if bsz == 0:
        raise ValueError("Batch must not be empty")
    if hq == 0 or hq % hkv:
        raise ValueError("Query heads must be divisible by KV heads")
    if q3.dtype != dtype:
        raise ValueError("Query dtype must match cache dtype (that of kv_params)")
    qs = q3.stride()
    if qs[2] != 1:
        q3 = q3.contiguous()
        qs = q3.stride()
    ts = block_tables.shape
    if block_tables.dtype != torch.int32 or len(ts) != 2 or ts[0] != bsz:
        raise ValueError("block_tables must be int32 [B, max_blocks]")
    tst = block_tables.stride()
    if tst[1] != 1:
        block_tables = block_tables.contiguous()
        tst = block_tables.stride()
    if context_lens.dtype != torch.int32 or context_lens.shape != (bsz,):
        raise ValueError("context_lens must be int32 [B]")
    context_lens = context_lens.contiguous()
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    width = ts[1] * bs
    if max_context is None:
        max_context = width
    elif not 0 <= max_context <= width:
        raise ValueError("max_context must be at most block_tables' width in tokens")
    if max_context >= 1 << 31:
        raise ValueError("max_context must be below 2^31 tokens")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _check_flag(error_flag)
    dev = _cuda_index(kv_codes, kv_params, q3, block_tables, context_lens, out, workspace, error_flag)
    if out is None:
        out = torch.empty_like(query)
        if out.stride()[-1] != 1:
            out = out.contiguous()
    o3 = out.squeeze(2) if out.ndim == 4 else out
    os_ = o3.stride()
    if o3.shape != shape or o3.dtype != dtype or os_[2] != 1:
        raise ValueError("out must match query's shape/dtype with unit stride along head_dim")
    if workspace is None:
        workspace = torch.empty(decode_int4_workspace_bytes(bsz, hq, hkv, d, bs, int(max_context), dtype),
                                dtype=torch.uint8, device=query.device)
    else:
        _check_workspace(workspace)
    _call(dev, _native.load().psb_paged_decode_int4, "paged_decode_int4",
          q3.data_ptr(), qs[0], qs[1], o3.data_ptr(), os_[0], os_[1], kv_codes.data_ptr(), kv_params.data_ptr(),
          block_tables.data_ptr(), tst[0], context_lens.data_ptr(), bsz, hq, layer, nl, nb, hkv, bs, d, code,
          int(max_context), scale, workspace.data_ptr(), workspace.nbytes, _ptr(error_flag))
    return out


@functools.lru_cache(maxsize=1024)
def prefill_int4_workspace_bytes(total: int, num_seqs: int, q_heads: int, hkv: int, head_dim: int, block_size: int,
                                 max_context: int, dtype: torch.dtype) -> int:
    """Scratch bytes of ``paged_prefill_int4`` (psb_paged_prefill_int4_workspace_size)."""
    lib = _native.load()
    return int(lib.psb_paged_prefill_int4_workspace_size(total, num_seqs, q_heads, hkv, head_dim, block_size,
                                                         max_context, dtype_code(dtype)))


def paged_prefill_int4(q: torch.Tensor, kv_codes: torch.Tensor, kv_params: torch.Tensor, block_tables: torch.Tensor,
                       context_lens: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, layer: int,
                       scale: float | None = None, out: torch.Tensor | None = None, max_context: int | None = None,
                       workspace: torch.Tensor | None = None, error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_prefill`` over a 4-bit pool (psb_paged_prefill_int4): ``q [T,
    Hq, D]`` of ``kv_params``' dtype, the rest as in ``paged_prefill``.  Rows
    of ``out`` that belong to no sequence keep what they held.  Scratch as in
    ``paged_decode_int4`` (``prefill_int4_workspace_bytes``).

    bf16 and f16 with head_dim 64, rows of ``q`` that start on 16 bytes, at most
    128 q heads per kv head and 2048 sequences run on the tensor cores, with
    probabilities of f16's 11 bits (errors as in ``paged_decode_int4``);
    anything else, head_dim 128 and fp32 among it, on a CUDA-core kernel that
    decodes every key again for every row and takes 50 to 300 times as long.
    """
    if q.is_cuda:
        done = (_native._calls or _native.calls()).prefill(q, kv_codes, kv_params, cu_seqlens, max_seqlen, block_tables,
                                                           context_lens, layer, scale, out, max_context, workspace,
                                                           error_flag)
        if done is not None:
            return _done(done, "paged_prefill_int4")
    nl, nb, hkv, bs, d, dtype, code = _int4_geometry(kv_codes, kv_params)
    shape = q.shape
    if len(shape) != 3 or shape[2] != d:
        raise ValueError(f"q must be [T, Hq, {d}]")
    t, hq, _ = shape
    if hq == 0 or hq % hkv:
        raise ValueError("Query heads must be divisible by KV heads")
    if q.dtype != dtype:
        raise ValueError("q dtype must match the cache dtype (that of kv_params)")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be int32 [B+1]")
    batch = cu_seqlens.shape[0] - 1
    ts = block_tables.shape
    if block_tables.dtype != torch.int32 or len(ts) != 2 or ts[0] != batch:
        raise ValueError("block_tables must be int32 [B, max_blocks]")
    if context_lens.dtype != torch.int32 or context_lens.shape != (batch,):
        raise ValueError("context_lens must be int32 [B]")
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    qs = q.stride()
    if qs[2] != 1:
        q = q.contiguous()
        qs = q.stride()
    tst = block_tables.stride()
    if tst[1] != 1:
        block_tables = block_tables.contiguous()
        tst = block_tables.stride()
    cu_seqlens, context_lens = cu_seqlens.contiguous(), context_lens.contiguous()
    width = ts[1] * bs
    if max_context is None:
        max_context = width
    elif max_context > width:
        raise ValueError("max_context must be at most block_tables' width in tokens")
    if max_context >= 1 << 31:
        raise ValueError("max_context must be below 2^31 tokens")
    if not 0 <= max_seqlen <= max_context:
        raise ValueError("max_seqlen must be at most max_context")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _check_flag(error_flag)
    dev = _cuda_index(kv_codes, kv_params, q, block_tables, context_lens, cu_seqlens, out, workspace, error_flag)
    if out is None:
        out = torch.empty_like(q)
    os_ = out.stride()
    if out.shape != shape or out.dtype != dtype or os_[2] != 1:
        raise ValueError("out must match q with unit stride along head_dim")
    if workspace is None:
        workspace = torch.empty(prefill_int4_workspace_bytes(t, batch, hq, hkv, d, bs, int(max_context), dtype),
                                dtype=torch.uint8, device=q.device)
    else:
        _check_workspace(workspace)
    _call(dev, _native.load().psb_paged_prefill_int4, "paged_prefill_int4",
          q.data_ptr(), qs[0], qs[1], kv_codes.data_ptr(), kv_params.data_ptr(), block_tables.data_ptr(), tst[0],
          context_lens.data_ptr(), out.data_ptr(), os_[0], os_[1], cu_seqlens.data_ptr(), batch, t, int(max_seqlen),
          int(max_context), hq, layer, nl, nb, hkv, bs, d, code, scale, workspace.data_ptr(), workspace.nbytes,
          _ptr(error_flag))
    return out


# -- block tables that grow on the device ------------------------------------------------------------------------


def _tables_args(table_store, rows, first, second, free_blocks, free_state, names, error_flag):
    """The checks extend_step and trim_tables share; returns the store's
    (row stride, rows, width), the batch, and the three plan rows, contiguous."""
    i32 = torch.int32
    shape = table_store.shape
    stride = table_store.stride()
    if table_store.dtype != i32 or len(shape) != 2 or stride[1] != 1 or stride[0] < shape[1]:
        raise ValueError("table_store must be int32 [R, W] with unit column stride and rows that do not overlap")
    plan = rows.shape
    if (rows.dtype != i32 or first.dtype != i32 or second.dtype != i32 or len(plan) != 1 or first.shape != plan
            or second.shape != plan):
        raise ValueError(f"{', '.join(names)} must be int32 [B]")
    fs = free_blocks.shape
    if free_blocks.dtype != i32 or len(fs) != 1 or fs[0] == 0 or not free_blocks.is_contiguous():
        raise ValueError("free_blocks must be a contiguous int32 [num_blocks] tensor")
    if free_state.dtype != i32 or free_state.shape != (4,) or not free_state.is_contiguous():
        raise ValueError("free_state must be a contiguous int32 [4] tensor (head, count, 0, 0)")
    _check_flag(error_flag)
    return (stride[0], shape[0], shape[1]), plan[0], rows.contiguous(), first.contiguous(), second.contiguous()


def free_list(num_blocks: int, device: torch.device | str, order=None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(free_blocks, free_state)`` for ``extend_step``: every block of a pool
    free, in the order ``BlockManager`` hands them out (``order``: another
    permutation of the ids, its ``free_order``)."""
    if num_blocks <= 0:
        raise ValueError("num_blocks must be positive")
    ids = list(range(num_blocks)) if order is None else [int(x) for x in order]
    if order is not None and sorted(ids) != list(range(num_blocks)):
        raise ValueError("order must be a permutation of range(num_blocks)")
    return (torch.tensor(ids, dtype=torch.int32, device=device),
            torch.tensor([0, num_blocks, 0, 0], dtype=torch.int32, device=device))


def extend_step(table_store: torch.Tensor, req_rows: torch.Tensor, starts: torch.Tensor, query_lens: torch.Tensor,
                free_blocks: torch.Tensor, free_state: torch.Tensor, total: int, block_size: int,
                out_width: int | None = None, error_flag: torch.Tensor | None = None, out: tuple | None = None):
    """``pack_step`` that also allocates, on the GPU (psb_extend_step).

    The blocks each request lacks for its ``query_lens[b]`` new tokens are
    taken from the head of the free ring (``free_list``) in entry order and
    appended to its row of ``table_store``; returns ``(cu_seqlens,
    context_lens, slot_mapping, positions, block_tables)`` as ``pack_step``
    does.  Between this call and a ``paged_decode`` over a 16-bit pool, which
    reads lengths and tables ahead of its stream predecessor, there must be an
    ordinary launch (any PyTorch operator).  ``req_rows[b] < 0`` marks a padding entry.  A step that cannot be
    carried out whole changes nothing, sets ``error_flag`` (128: not enough
    free blocks, 256: a row named twice, 4: a bad row, start, count or width,
    1: an id outside the pool would be taken, 32: ``total`` is not the sum) and
    gives slots of -1 and lengths of 0.  It also sets bit 512, with which every
    ``extend_step`` and ``trim_tables`` on that flag is refused in turn - they
    count on blocks that were not taken - until the flag is cleared.
    """
    if out is None and table_store.is_cuda:
        done = (_native._calls or _native.calls()).extend(table_store, req_rows, starts, query_lens, free_blocks,
                                                          free_state, total, block_size, out_width, error_flag)
        if done is not None:
            return _done(done, "extend_step")
    store, bsz, rows, starts, query_lens = _tables_args(table_store, req_rows, starts, query_lens, free_blocks,
                                                        free_state, ("req_rows", "starts", "query_lens"), error_flag)
    total = int(total)
    width = store[2] if out_width is None else int(out_width)
    if total < 0 or width <= 0 or block_size <= 0:
        raise ValueError("total must not be negative, out_width and block_size must be positive")
    dev = _cuda_index(table_store, rows, starts, query_lens, free_blocks, free_state, error_flag)
    if out is None:
        cu = rows.new_empty(bsz + 1)
        ctx = rows.new_empty(bsz)
        slots = rows.new_empty(total, dtype=torch.int64)
        pos = rows.new_empty(total, dtype=torch.int64)
        tables = rows.new_empty((bsz, width))
    else:
        cu, ctx, slots, pos, tables = out
        ok = (cu.shape == (bsz + 1,) and cu.dtype == torch.int32 and ctx.shape == (bsz,) and ctx.dtype == torch.int32
              and slots.shape == (total,) and slots.dtype == torch.int64 and pos.shape == (total,)
              and pos.dtype == torch.int64 and tables.shape == (bsz, width) and tables.dtype == torch.int32
              and all(t.is_contiguous() for t in out))
        if not ok:
            raise ValueError("out must be contiguous (cu_seqlens [B+1] i32, context_lens [B] i32, slot_mapping [T] "
                             "i64, positions [T] i64, block_tables [B, out_width] i32)")
        _cuda_index(table_store, *out)
    if bsz == 0:
        if total:
            raise ValueError("total must be 0 for an empty batch")
        cu.zero_()
        return cu, ctx, slots, pos, tables
    _call(dev, _native.load().psb_extend_step, "extend_step",
          table_store.data_ptr(), *store, rows.data_ptr(), starts.data_ptr(), query_lens.data_ptr(), bsz,
          free_blocks.data_ptr(), free_blocks.shape[0], free_state.data_ptr(), total, int(block_size), cu.data_ptr(),
          ctx.data_ptr(), slots.data_ptr(), pos.data_ptr(), tables.data_ptr(), width, _ptr(error_flag))
    return cu, ctx, slots, pos, tables


def trim_tables(table_store: torch.Tensor, req_rows: torch.Tensor, held_lens: torch.Tensor, keep_lens: torch.Tensor,
                free_blocks: torch.Tensor, free_state: torch.Tensor, block_size: int,
                error_flag: torch.Tensor | None = None) -> None:
    """Give back, on the GPU, the blocks requests no longer need
    (psb_trim_tables): entry b of ``held_lens[b]`` tokens keeps
    ``keep_lens[b]`` (0: it has finished).  The blocks go to the tail of the
    free ring entry by entry, in table order, as ``BlockManager.free`` returns
    them.  Checked and refused as a whole, like ``extend_step``.  Behind a step
    of ``extend_step`` that may have been refused, pass its ``error_flag`` (the
    trim is then refused too) or its ``context_lens`` as ``held_lens``.
    """
    if table_store.is_cuda:
        done = (_native._calls or _native.calls()).trim(table_store, req_rows, held_lens, keep_lens, free_blocks,
                                                        free_state, block_size, error_flag)
        if done is not None:
            _done(done, "trim_tables")
            return
    store, bsz, rows, held_lens, keep_lens = _tables_args(table_store, req_rows, held_lens, keep_lens, free_blocks,
                                                          free_state, ("req_rows", "held_lens", "keep_lens"),
                                                          error_flag)
    if block_size <= 0:
        raise ValueError("block_size must be positive")
    dev = _cuda_index(table_store, rows, held_lens, keep_lens, free_blocks, free_state, error_flag)
    _call(dev, _native.load().psb_trim_tables, "trim_tables",
          table_store.data_ptr(), *store, rows.data_ptr(), held_lens.data_ptr(), keep_lens.data_ptr(), bsz,
          free_blocks.data_ptr(), free_blocks.shape[0], free_state.data_ptr(), int(block_size), _ptr(error_flag))


# -- several continuations of one prompt -------------------------------------------------------------------------


def share_counts(num_blocks: int, device: torch.device | str) -> torch.Tensor:
    """``shares`` for ``fork_tables`` and ``release_tables``: int32
    ``[2, num_blocks]`` of zeros, every block of a pool with one holder at most."""
    if num_blocks <= 0:
        raise ValueError("num_blocks must be positive")
    return torch.zeros((2, num_blocks), dtype=torch.int32, device=device)


def _check_shares(shares: torch.Tensor, num_blocks: int) -> None:
    if shares.dtype != torch.int32 or shares.shape != (2, num_blocks) or not shares.is_contiguous():
        raise ValueError(f"shares must be a contiguous int32 [2, {num_blocks}] tensor like free_blocks")


def fork_tables(table_store: torch.Tensor, parent_rows: torch.Tensor, child_rows: torch.Tensor, lens: torch.Tensor,
                shares: torch.Tensor, free_blocks: torch.Tensor, free_state: torch.Tensor, block_size: int,
                error_flag: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows that share their parents' pages (psb_fork_tables).

    Entry b makes row ``child_rows[b]`` of ``table_store`` (which holds nothing)
    a continuation of the first ``lens[b]`` tokens of row ``parent_rows[b]``: it
    shares their whole blocks (counted in ``shares``, ``share_counts``), and where
    they end inside a block it gets one of its own from the free ring.  Returns
    ``(src, dst)`` int32 ``[B]``: the blocks ``copy_blocks`` has to copy for that
    (-1: none).  One parent may have many children; a child is no parent of the
    same call; ``child_rows[b] < 0`` is padding.  Rows that share blocks give them
    back with ``release_tables`` (not ``trim_tables``).  Checked and refused as a
    whole, like ``extend_step``; and as behind it there must be an ordinary launch
    between this call, ``copy_blocks`` or ``release_tables`` and ``paged_decode``.
    """
    if table_store.is_cuda:
        done = (_native._calls or _native.calls()).fork(table_store, parent_rows, child_rows, lens, free_blocks, free_state,
                                                        shares, block_size, error_flag)
        if done is not None:
            return _done(done, "fork_tables")
    store, bsz, parents, children, lens = _tables_args(table_store, parent_rows, child_rows, lens, free_blocks, free_state,
                                                       ("parent_rows", "child_rows", "lens"), error_flag)
    _check_shares(shares, free_blocks.shape[0])
    if block_size <= 0:
        raise ValueError("block_size must be positive")
    dev = _cuda_index(table_store, parents, children, lens, shares, free_blocks, free_state, error_flag)
    src, dst = lens.new_empty(bsz), lens.new_empty(bsz)
    _call(dev, _native.load().psb_fork_tables, "fork_tables",
          table_store.data_ptr(), *store, parents.data_ptr(), children.data_ptr(), lens.data_ptr(), bsz, shares.data_ptr(),
          free_blocks.data_ptr(), free_blocks.shape[0], free_state.data_ptr(), int(block_size), src.data_ptr(),
          dst.data_ptr(), _ptr(error_flag))
    return src, dst


def release_tables(table_store: torch.Tensor, req_rows: torch.Tensor, held_lens: torch.Tensor, keep_lens: torch.Tensor,
                   shares: torch.Tensor, free_blocks: torch.Tensor, free_state: torch.Tensor, block_size: int,
                   error_flag: torch.Tensor | None = None) -> None:
    """``trim_tables`` for rows that may share blocks (psb_release_tables).

    Of the blocks past what entry b keeps, in entry and table order, one that
    others hold too loses a holder, any other goes to the tail of the free ring.
    ``keep_lens[b]`` may end inside a block only if nobody else holds that block
    afterwards: the call is refused otherwise (``error_flag`` 1024).
    """
    if table_store.is_cuda:
        done = (_native._calls or _native.calls()).release(table_store, req_rows, held_lens, keep_lens, free_blocks,
                                                           free_state, shares, block_size, error_flag)
        if done is not None:
            _done(done, "release_tables")
            return
    store, bsz, rows, held_lens, keep_lens = _tables_args(table_store, req_rows, held_lens, keep_lens, free_blocks,
                                                          free_state, ("req_rows", "held_lens", "keep_lens"),
                                                          error_flag)
    _check_shares(shares, free_blocks.shape[0])
    if block_size <= 0:
        raise ValueError("block_size must be positive")
    dev = _cuda_index(table_store, rows, held_lens, keep_lens, shares, free_blocks, free_state, error_flag)
    _call(dev, _native.load().psb_release_tables, "release_tables",
          table_store.data_ptr(), *store, rows.data_ptr(), held_lens.data_ptr(), keep_lens.data_ptr(), bsz,
          shares.data_ptr(), free_blocks.data_ptr(), free_blocks.shape[0], free_state.data_ptr(), int(block_size),
          _ptr(error_flag))


def copy_blocks(pools, src: torch.Tensor, dst: torch.Tensor, error_flag: torch.Tensor | None = None) -> None:
    """Block ``dst[i]`` of every layer becomes what block ``src[i]`` is, in each of
    ``pools`` (psb_copy_blocks): up to four contiguous tensors ``[num_layers,
    num_blocks, ...]`` of any types, e.g. ``(k_cache, v_cache)`` or ``(kv_codes,
    kv_params)``.  ``src, dst [N]`` int32; a pair with a negative id is skipped.
    Destinations are distinct and none is a source.
    """
    pools = tuple(pools)
    if src.is_cuda:
        done = (_native._calls or _native.calls()).copy(pools, src, dst, error_flag)
        if done is not None:
            _done(done, "copy_blocks")
            return
    if not 1 <= len(pools) <= 4:
        raise ValueError("pools must be one to four tensors")
    if src.dtype != torch.int32 or src.ndim != 1 or dst.dtype != torch.int32 or dst.shape != src.shape:
        raise ValueError("src and dst must be int32 [N]")
    lead = tuple(pools[0].shape[:2])
    for x in pools:
        if x.ndim < 3 or tuple(x.shape[:2]) != lead or not x.is_contiguous() or x.numel() == 0:
            raise ValueError("pools must be contiguous [num_layers, num_blocks, ...] of the same layers and blocks")
    _check_flag(error_flag)
    src, dst = src.contiguous(), dst.contiguous()
    dev = _cuda_index(*pools, src, dst, error_flag)
    n = len(pools)
    ptrs = (ctypes.c_void_p * n)(*[x.data_ptr() for x in pools])
    sizes = (ctypes.c_int64 * n)(*[x.numel() // (lead[0] * lead[1]) * x.element_size() for x in pools])
    _call(dev, _native.load().psb_copy_blocks, "copy_blocks", ptrs, sizes, n, src.data_ptr(), dst.data_ptr(), src.shape[0],
          lead[0], lead[1], _ptr(error_flag))


@functools.lru_cache(maxsize=1024)
def decode_shared_workspace_bytes(batch: int, groups: int, q_heads: int, hkv: int, head_dim: int, block_size: int,
                                  max_context: int, dtype: torch.dtype) -> int:
    """Scratch of one ``paged_decode_shared`` call; 0 for a geometry that ``paged_decode`` answers in its place."""
    return int(_native.load().psb_paged_decode_shared_workspace_size(batch, groups, q_heads, hkv, head_dim, block_size,
                                                                     max_context, dtype_code(dtype)))


def paged_decode_shared(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, cu_groups: torch.Tensor, prefix_lens: torch.Tensor, layer: int,
                        scale: float | None = None, out: torch.Tensor | None = None, max_context: int | None = None,
                        workspace: torch.Tensor | None = None, error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_decode`` for a batch whose sequences share long prefixes (psb_paged_decode_shared).

    Sequences ``cu_groups[g] .. cu_groups[g + 1] - 1`` (int32 ``[G + 1]``) agree in
    their first ``prefix_lens[g]`` tokens (int32 ``[G]``): their rows of
    ``block_tables`` name the same blocks there (``fork_tables``), or blocks of the
    same contents.  The prefix is read and multiplied once for the whole group, what
    lies behind it sequence by sequence.  Sequences of no group are on their own;
    one without tokens gets zeros.  Returns ``out`` with ``query``'s shape
    (``[B, Hq, D]`` or ``[B, Hq, 1, D]``) and dtype.

    Prefixes are shared for bf16/f16, head_dim 64 or 128, up to 16 q heads per kv
    head, blocks of 16, 32, 64 or a multiple of 64 tokens, up to 2048 sequences
    (12 bytes a sequence and 24 a group have to fit 33 KB); the rest is answered by
    ``paged_decode``, each sequence on its own.  ``scale`` must be positive.
    ``workspace``: ``decode_shared_workspace_bytes`` of scratch (where that is 0,
    ``decode_workspace_bytes``; of less there, the call takes its own); without it the
    scratch comes from PyTorch's allocator.  Calls that may overlap need one each.
    """
    if query.is_cuda:
        done = (_native._calls or _native.calls()).decode_shared(query, k_cache, v_cache, block_tables, context_lens, cu_groups,
                                                                 prefix_lens, layer, scale, out, max_context, workspace,
                                                                 error_flag)
        if done is not None:
            return _done(done, "paged_decode_shared")
    nl, nb, hkv, bs, d = _pool_geometry(k_cache, v_cache)
    q3 = query.squeeze(2) if query.ndim == 4 and query.shape[2] == 1 else query
    if q3.ndim != 3 or q3.shape[2] != d:
        raise ValueError("query must be [B, Hq, D] or [B, Hq, 1, D]")
    bsz, hq, _ = q3.shape
    if bsz == 0:
        raise ValueError("Batch must not be empty")
    if hq == 0 or hq % hkv:
        raise ValueError("Query heads must be divisible by KV heads")
    if q3.dtype != k_cache.dtype:
        raise ValueError("Query dtype must match cache dtype")
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2 or block_tables.shape[0] != bsz:
        raise ValueError("block_tables must be int32 [B, max_blocks]")
    if context_lens.dtype != torch.int32 or context_lens.shape != (bsz,):
        raise ValueError("context_lens must be int32 [B]")
    if prefix_lens.dtype != torch.int32 or prefix_lens.ndim != 1:
        raise ValueError("prefix_lens must be int32 [G]")
    groups = prefix_lens.shape[0]
    if cu_groups.dtype != torch.int32 or cu_groups.shape != (groups + 1,):
        raise ValueError("cu_groups must be int32 [G + 1]")
    if not 0 <= layer < nl:
        raise ValueError("Invalid layer")
    width = block_tables.shape[1] * bs
    max_context = width if max_context is None else int(max_context)
    if not 0 <= max_context <= width:
        raise ValueError(f"max_context must lie in [0, {width}] (the block tables' width)")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive")
    _check_flag(error_flag)
    if out is None:
        out = torch.empty_like(query)
    o3 = out.squeeze(2) if out.ndim == 4 and out.shape[2] == 1 else out
    if o3.shape != q3.shape or o3.stride(2) != 1 or o3.dtype != q3.dtype:
        raise ValueError("out must match query's shape/dtype with unit stride along head_dim")
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    context_lens, cu_groups, prefix_lens = context_lens.contiguous(), cu_groups.contiguous(), prefix_lens.contiguous()
    need = decode_shared_workspace_bytes(bsz, groups, hq, hkv, d, bs, max_context, q3.dtype)
    if need == 0 or (k_cache.data_ptr() | v_cache.data_ptr()) & 15 or nl * nb * hkv > 0x7fffffff:
        dev = _cuda_index(q3, k_cache, v_cache, block_tables, context_lens, cu_groups, prefix_lens, out, workspace, error_flag)
        if error_flag is not None:
            _call(dev, _native.load().psb_check_groups, "paged_decode_shared", cu_groups.data_ptr(), prefix_lens.data_ptr(), bsz,
                  groups, error_flag.data_ptr())
        # scratch as of the calls that share: the caller's, or the allocator's (paged_decode's own is one for all streams)
        need = decode_workspace_bytes(bsz, hq, hkv, d, bs, max_context, q3.dtype)
        if workspace is not None:
            _check_workspace(workspace)
        if workspace is None or workspace.nbytes < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q3.device)
        with torch.cuda.device(q3.device):
            # paged_decode may read lengths and tables while the library's launch in front of it still writes them: the
            # copy of the lengths is the ordinary work that has to lie between
            paged_decode(q3, k_cache, v_cache, block_tables, context_lens.clone(), layer, scale=scale, out=o3,
                         max_context=max_context, workspace=workspace, error_flag=error_flag)
        return out
    qs = q3.stride()
    if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or qs[0] <= 0 or qs[1] <= 0 or q3.data_ptr() & 15:
        q3 = q3.contiguous() if not q3.is_contiguous() else q3.clone()
        qs = (hq * d, d, 1)
    dev = _cuda_index(q3, k_cache, v_cache, block_tables, context_lens, cu_groups, prefix_lens, out, workspace, error_flag)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q3.device)
    else:
        _check_workspace(workspace)
    os_ = o3.stride()
    _call(dev, _native.load().psb_paged_decode_shared, "paged_decode_shared",
          q3.data_ptr(), qs[0], qs[1], o3.data_ptr(), os_[0], os_[1], k_cache.data_ptr(), v_cache.data_ptr(),
          block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), cu_groups.data_ptr(),
          prefix_lens.data_ptr(), bsz, groups, hq, layer, nl, nb, hkv, bs, d, _DTYPES[q3.dtype], max_context, scale,
          workspace.data_ptr(), workspace.nbytes, _ptr(error_flag))
    return out


def verify_tokens(logits: torch.Tensor, tokens: torch.Tensor, cu_seqlens: torch.Tensor, uniforms: torch.Tensor,
                  temperature: torch.Tensor, draft_probs: torch.Tensor | None = None,
                  error_flag: torch.Tensor | None = None, out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Drafted tokens against the target's probabilities, from given random numbers (psb_verify_tokens).

    Sequence b was fed ``tokens[cu_seqlens[b] : cu_seqlens[b + 1]]`` (int64
    ``[T]``): its last token, then its drafts; ``logits [T, V]`` are the rows that
    step gave.  Row r stands for ``p = softmax(logits[r] / temperature[b])`` (fp32
    ``[B]``; 0: the first maximum); the draft ``d = tokens[r + 1]``, drawn from
    ``q = draft_probs[r]`` (``[T, V]``; None: a draft that was looked up), is taken
    if ``uniforms[r, 0] q(d) < p(d)`` (fp32 ``[T, 2]`` in [0, 1)).  At the first row
    whose draft is not taken the new token is drawn from ``max(p - q, 0)`` with
    ``uniforms[r, 1]``, at the last row (or one whose draft is -1) from p, so
    the tokens are distributed as if each had been drawn from p.  A batch of
    one row a sequence is plain sampling.

    Returns ``(new_tokens [T] int64, counts [B] int32)`` (``out``: the same two):
    sequence b's new tokens from ``cu_seqlens[b]`` on, -1 behind them, and how many;
    its cache keeps ``counts[b]`` of the rows fed (``trim_tables`` takes the rest).
    Decided as in 64-bit arithmetic.  A row without probabilities (NaN, +inf, all
    -inf) takes no draft, gives its first maximum and is flagged (2048).
    """
    if out is None and logits.is_cuda:
        done = (_native._calls or _native.calls()).verify(logits, tokens, cu_seqlens, uniforms, temperature, draft_probs,
                                                          error_flag)
        if done is not None:
            return _done(done, "verify_tokens")
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [T, V]")
    t, v = (int(x) for x in logits.shape)
    code = dtype_code(logits.dtype)
    if logits.stride(1) != 1 or (t > 1 and logits.stride(0) < v):
        logits = logits.contiguous()
    if tokens.dtype != torch.int64 or tokens.shape != (t,):
        raise ValueError("tokens must be int64 [T]")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be int32 [B + 1]")
    b = cu_seqlens.shape[0] - 1
    if b == 0 and t > 0:
        raise ValueError("logits hold rows but cu_seqlens no sequence")
    if uniforms.dtype != torch.float32 or uniforms.shape != (t, 2):
        raise ValueError("uniforms must be float32 [T, 2]")
    if temperature.dtype != torch.float32 or temperature.shape != (b,):
        raise ValueError("temperature must be float32 [B]")
    tokens, cu_seqlens, uniforms, temperature = (x.contiguous() for x in (tokens, cu_seqlens, uniforms, temperature))
    qcode = 0
    if draft_probs is not None:
        if draft_probs.shape != (t, v):
            raise ValueError("draft_probs must be [T, V] like logits")
        qcode = dtype_code(draft_probs.dtype)
        if draft_probs.stride(1) != 1 or (t > 1 and draft_probs.stride(0) < v):
            draft_probs = draft_probs.contiguous()
    _check_flag(error_flag)
    if out is None:
        new, counts = tokens.new_empty(t), cu_seqlens.new_empty(b)
    else:
        new, counts = out
        if (new.dtype != torch.int64 or new.shape != (t,) or not new.is_contiguous() or counts.dtype != torch.int32
                or counts.shape != (b,) or not counts.is_contiguous()):
            raise ValueError("out must be contiguous (new_tokens [T] int64, counts [B] int32)")
        if t and new.data_ptr() == tokens.data_ptr():
            raise ValueError("new_tokens may not be tokens itself")
        for x in (new, counts):
            if any(_overlap(x, y) for y in (tokens, cu_seqlens, uniforms, temperature, counts if x is new else new)):
                raise ValueError("out may not overlap the inputs, nor each other")
    dev = _cuda_index(logits, tokens, cu_seqlens, uniforms, temperature, draft_probs, new, counts, error_flag)
    workspace = torch.empty(max(1, 2 * b), dtype=torch.int64, device=logits.device)  # 16 bytes a sequence
    _call(dev, _native.load().psb_verify_tokens, "verify_tokens",
          logits.data_ptr(), logits.stride(0), t, v, code, tokens.data_ptr(), cu_seqlens.data_ptr(), b, uniforms.data_ptr(),
          temperature.data_ptr(), _ptr(draft_probs), 0 if draft_probs is None else draft_probs.stride(0), qcode,
          new.data_ptr(), counts.data_ptr(), workspace.data_ptr(), workspace.nbytes, _ptr(error_flag))
    return new, counts
