"""Host-side paged-KV bookkeeping with PagedServe's interface.

The B200 kernels address the pool through block tables; this module owns
them.  Class names, method names, argument meaning and the exception types
raised follow the reference so callers can switch without edits:

* ``BlockManager``  - pagedserve/engine/block_manager.py:6-155 (FIFO free list:
  allocation takes from the head, ``free`` returns blocks to the tail)
* ``BlockTable``    - pagedserve/engine/block_table.py:4-49
* ``KVCache``       - pagedserve/engine/kv_cache.py:6-164, layout
  ``[layer, physical_block, kv_head, token_in_block, head_dim]``
* ``PagedKVCache``  - pagedserve/engine/paged_kv_cache.py:10-233

Added for the batched path: ``PagedKVCache.table_rows`` (a padded int32
table for a list of requests, built in one numpy pass) and
``PagedKVCache.slot_of`` (the int64 slot a position maps to); pools that
hold 4-bit codes (``kv_bits=4``: ``kv_codes`` and ``kv_params`` in place of
``k_cache`` and ``v_cache``, the layout of ``ops.reshape_and_cache_int4``); and
requests that share their first blocks (``fork``; ``shared_prefixes`` tells a
decode step which).
"""

from __future__ import annotations

from collections import deque

import numpy as np
import torch

from . import ops


class BlockManager:
    """Ownership of physical KV blocks; allocates no tensors."""

    def __init__(self, num_blocks: int, block_size: int = 16, free_order=None):
        if num_blocks <= 0:
            raise ValueError("num_blocks must be positive")
        if block_size <= 0:
            raise ValueError("block_size must be positive")
        self.num_blocks = num_blocks
        self.block_size = block_size
        # ``free_order`` (a permutation of the block ids) seeds the free list in
        # another order, e.g. a shuffled pool for fragmentation studies.
        order = range(num_blocks) if free_order is None else [int(b) for b in free_order]
        if free_order is not None and sorted(order) != list(range(num_blocks)):
            raise ValueError("free_order must be a permutation of range(num_blocks)")
        self._free: deque[int] = deque(order)
        self._owned: dict[str, list[int]] = {}
        self._shares: dict[int, int] = {}  # holders of a block beyond the first (of shared blocks alone)

    @property
    def free_blocks(self) -> int:
        return len(self._free)

    @property
    def used_blocks(self) -> int:
        return self.num_blocks - len(self._free)

    def blocks_needed(self, num_tokens: int) -> int:
        """ceil(num_tokens / block_size); 0 tokens need 0 blocks."""
        if num_tokens < 0:
            raise ValueError("num_tokens cannot be negative")
        return -(-num_tokens // self.block_size)

    def _take(self, count: int) -> list[int]:
        if count > len(self._free):
            raise RuntimeError(f"Not enough KV blocks: required={count}, free={len(self._free)}")
        return [self._free.popleft() for _ in range(count)]

    def allocate(self, request_id: str, num_tokens: int) -> list[int]:
        """Blocks for a new request, taken from the head of the free list."""
        if request_id in self._owned:
            raise ValueError(f"Request {request_id!r} already has blocks")
        blocks = self._take(self.blocks_needed(num_tokens))
        self._owned[request_id] = blocks
        return list(blocks)

    def allocate_blocks(self, request_id: str, num_blocks: int) -> list[int]:
        """Additional blocks for an existing request."""
        if request_id not in self._owned:
            raise KeyError(f"Unknown request: {request_id!r}")
        if num_blocks <= 0:
            raise ValueError("num_blocks must be positive")
        blocks = self._take(num_blocks)
        self._owned[request_id].extend(blocks)
        return list(blocks)

    def fork(self, parent_id: str, request_id: str, num_tokens: int) -> tuple[list[int], tuple[int, int] | None]:
        """Blocks for a request that continues the first ``num_tokens`` tokens of
        ``parent_id``: the parent's whole blocks, shared, and where those tokens end
        inside a block one from the free list, returned with the block it has to be a
        copy of: ``(blocks, (source, copy) or None)``."""
        if parent_id not in self._owned:
            raise KeyError(f"Unknown request: {parent_id!r}")
        if request_id in self._owned:
            raise ValueError(f"Request {request_id!r} already has blocks")
        parent = self._owned[parent_id]
        if self.blocks_needed(num_tokens) > len(parent):
            raise ValueError(f"Request {parent_id!r} holds fewer than {num_tokens} tokens")
        whole = num_tokens // self.block_size
        pair = None
        blocks = parent[:whole]
        if num_tokens % self.block_size:
            pair = (parent[whole], self._take(1)[0])
            blocks = blocks + [pair[1]]
        for blk in parent[:whole]:
            self._shares[blk] = self._shares.get(blk, 0) + 1
        self._owned[request_id] = blocks
        return list(blocks), pair

    def holders(self, block: int) -> int:
        """How many requests hold a block that is not free."""
        return 1 + self._shares.get(block, 0)

    def free(self, request_id: str) -> None:
        """Return all of a request's blocks to the tail of the free list (of a block
        that others hold, the last of them does)."""
        if request_id not in self._owned:
            raise KeyError(f"Unknown request: {request_id!r}")
        blocks = self._owned.pop(request_id)
        if not self._shares:
            self._free.extend(blocks)
            return
        for blk in blocks:
            others = self._shares.get(blk, 0)
            if others == 0:
                self._free.append(blk)
            elif others == 1:
                del self._shares[blk]
            else:
                self._shares[blk] = others - 1

    def get_blocks(self, request_id: str) -> list[int]:
        if request_id not in self._owned:
            raise KeyError(f"Unknown request: {request_id!r}")
        return list(self._owned[request_id])

    def has_request(self, request_id: str) -> bool:
        return request_id in self._owned


class BlockTable:
    """Logical -> physical block map of one request."""

    def __init__(self) -> None:
        self._blocks: list[int] = []
        self._owner: "PagedKVCache | None" = None  # told of every change (metadata epoch, table store)
        self._row = -1                              # this table's row in the owner's table store

    @property
    def num_blocks(self) -> int:
        return len(self._blocks)

    def append(self, physical_block_id: int) -> None:
        if physical_block_id < 0:
            raise ValueError("physical_block_id cannot be negative")
        self._blocks.append(physical_block_id)
        if self._owner is not None:
            self._owner._store_put(self._row, len(self._blocks) - 1, physical_block_id)
            self._owner._epoch += 1

    def get_physical_block(self, logical_block_id: int) -> int:
        if not 0 <= logical_block_id < len(self._blocks):
            raise IndexError(f"Invalid logical block: {logical_block_id}; valid range is [0, {len(self._blocks)})")
        return self._blocks[logical_block_id]

    def get_blocks(self) -> list[int]:
        return list(self._blocks)

    def clear(self) -> None:
        self._blocks.clear()
        if self._owner is not None:
            self._owner._store_clear(self._row)
            self._owner._epoch += 1


class KVCache:
    """The K and V pools, ``[num_layers, num_blocks, num_kv_heads, block_size, head_dim]`` each.

    ``kv_bits=4``: both in ``kv_codes`` (uint8 ``[num_layers, num_blocks,
    num_kv_heads, 2, block_size, head_dim / 2]``) and ``kv_params`` (``dtype``
    ``[..., 2, block_size, 2]``: the step and the offset of every row), with
    ``k_cache`` and ``v_cache`` None; rows go in and out as ``dtype`` on a
    CUDA device, and ``read_block`` returns copies instead of views.
    """

    def __init__(self, num_blocks: int, num_layers: int, num_kv_heads: int, head_dim: int, block_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: str | torch.device = "cuda", kv_bits: int = 16):
        for name, val in (("num_blocks", num_blocks), ("num_layers", num_layers), ("num_kv_heads", num_kv_heads),
                          ("head_dim", head_dim), ("block_size", block_size)):
            if val <= 0:
                raise ValueError(f"{name} must be positive")
        self.num_blocks = num_blocks
        self.num_layers = num_layers
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.block_size = block_size
        self.dtype = dtype
        self.device = torch.device(device)
        if kv_bits not in (4, 16):
            raise ValueError("kv_bits must be 4 or 16 (16: the pools hold dtype itself)")
        self.kv_bits = kv_bits
        self.kv_codes = self.kv_params = None
        if kv_bits == 4:
            if head_dim % 2 or head_dim > ops.INT4_MAX_HEAD_DIM:
                raise ValueError(f"4-bit pools need an even head_dim of at most {ops.INT4_MAX_HEAD_DIM}")
            ops.dtype_code(dtype)  # refuses what the kernels do not take
            shape = (num_layers, num_blocks, num_kv_heads, 2, block_size)
            self.kv_codes = torch.empty(shape + (head_dim // 2,), dtype=torch.uint8, device=self.device)
            self.kv_params = torch.empty(shape + (2,), dtype=dtype, device=self.device)
            self.k_cache = self.v_cache = None
            return
        shape = (num_layers, num_blocks, num_kv_heads, block_size, head_dim)
        self.k_cache = torch.empty(shape, dtype=dtype, device=self.device)
        self.v_cache = torch.empty(shape, dtype=dtype, device=self.device)

    @property
    def block_shape(self) -> tuple[int, ...]:
        return (self.num_kv_heads, self.block_size, self.head_dim)

    @property
    def block_bytes(self) -> int:
        """K+V bytes of one physical block across all layers."""
        esz = torch.empty((), dtype=self.dtype).element_size()
        row = self.head_dim // 2 + 2 * esz if self.kv_bits == 4 else self.head_dim * esz
        return self.num_layers * 2 * self.num_kv_heads * self.block_size * row

    @property
    def total_bytes(self) -> int:
        return self.num_blocks * self.block_bytes

    def copy_blocks(self, source: list[int], copy: list[int]) -> None:
        """Blocks ``copy`` become, in every layer, what blocks ``source`` are (one launch on a CUDA device)."""
        if len(source) != len(copy):
            raise ValueError("source and copy differ in length")
        for blk in (*source, *copy):
            self._check_block(blk)
        if not source:
            return
        pools = (self.kv_codes, self.kv_params) if self.kv_bits == 4 else (self.k_cache, self.v_cache)
        if self.device.type == "cuda":
            pair = torch.tensor([source, copy], dtype=torch.int32).to(pools[0].device)
            with torch.cuda.device(pools[0].device):
                ops.copy_blocks(pools, pair[0], pair[1])
            return
        for pool in pools:
            pool[:, copy] = pool[:, source]

    def _check_layer(self, layer: int) -> None:
        if not 0 <= layer < self.num_layers:
            raise IndexError(f"Invalid layer: {layer}; valid range is [0, {self.num_layers})")

    def _check_block(self, block_id: int) -> None:
        if not 0 <= block_id < self.num_blocks:
            raise IndexError(f"Invalid block ID: {block_id}; valid range is [0, {self.num_blocks})")

    def write_block(self, layer: int, block_id: int, key: torch.Tensor, value: torch.Tensor) -> None:
        self._check_layer(layer)
        self._check_block(block_id)
        for name, t in (("key", key), ("value", value)):
            if tuple(t.shape) != self.block_shape:
                raise ValueError(f"Invalid {name} shape: expected {self.block_shape}, got {tuple(t.shape)}")
            if t.dtype != self.dtype:
                raise ValueError(f"Invalid {name} dtype: expected {self.dtype}, got {t.dtype}")
        if self.kv_bits == 4:
            self._write_rows(layer, self._block_slots(block_id), key.transpose(0, 1), value.transpose(0, 1))
            return
        self.k_cache[layer, block_id].copy_(key)
        self.v_cache[layer, block_id].copy_(value)

    def read_block(self, layer: int, block_id: int) -> tuple[torch.Tensor, torch.Tensor]:
        self._check_layer(layer)
        self._check_block(block_id)
        if self.kv_bits == 4:
            key, value = self._read_rows(layer, self._block_slots(block_id))
            return key.transpose(0, 1), value.transpose(0, 1)
        return self.k_cache[layer, block_id], self.v_cache[layer, block_id]

    # -- rows of a 4-bit pool ---------------------------------------------------
    def _block_slots(self, block_id: int) -> torch.Tensor:
        first = block_id * self.block_size
        return torch.arange(first, first + self.block_size, dtype=torch.int64, device=self.device)

    def _write_rows(self, layer: int, slots: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> None:
        """Quantise ``key, value [T, Hkv, D]`` into ``slots [T]``."""
        if not key.is_cuda:
            raise ValueError("4-bit pools are written and read on a CUDA device")
        key, value = (t if t.stride(-1) == 1 else t.contiguous() for t in (key, value))  # (a copy_ takes any strides)
        ops.reshape_and_cache_int4(key, value, self.kv_codes, self.kv_params, slots, layer)

    def _read_rows(self, layer: int, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        if not slots.is_cuda:
            raise ValueError("4-bit pools are written and read on a CUDA device")
        return ops.gather_cache_int4(self.kv_codes, self.kv_params, slots, layer)


class PagedKVCache:
    """Block allocation + per-request tables + the pools, behind one object."""

    def __init__(self, num_blocks: int, num_layers: int, num_kv_heads: int, head_dim: int, block_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: str | torch.device = "cuda", free_order=None,
                 kv_bits: int = 16):
        self.block_manager = BlockManager(num_blocks=num_blocks, block_size=block_size, free_order=free_order)
        self.kv_cache = KVCache(num_blocks=num_blocks, num_layers=num_layers, num_kv_heads=num_kv_heads,
                                head_dim=head_dim, block_size=block_size, dtype=dtype, device=device,
                                kv_bits=kv_bits)
        self._tables: dict[str, BlockTable] = {}
        self._counts: dict[str, int] = {}
        self._epoch = 0
        # Table store: one zero-padded int32 row of block ids per live
        # request, kept in step with the BlockTables, so a batch's block table
        # is one gather instead of a list-to-array copy per request.
        self._store = np.zeros((16, 16), dtype=np.int32)
        self._store_blocks = np.zeros(16, dtype=np.int64)   # blocks per store row
        self._store_tokens = np.zeros(16, dtype=np.int64)   # token count per store row
        self._free_rows: list[int] = []
        self._rows_used = 0
        self._row_of: dict[str, int] = {}  # live request -> its table-store row

    # -- allocation ---------------------------------------------------------
    def allocate(self, request_id: str, num_tokens: int) -> None:
        if request_id in self._tables:
            raise ValueError(f"Request {request_id!r} already exists")
        if num_tokens < 0:
            raise ValueError("num_tokens cannot be negative")
        self._adopt(request_id, num_tokens, self.block_manager.allocate(request_id=request_id, num_tokens=num_tokens))

    def fork(self, parent_id: str, request_ids, num_tokens: int | None = None) -> None:
        """Requests that continue the first ``num_tokens`` tokens of ``parent_id`` (default: all of them).

        They share the parent's whole blocks; of a block in which those tokens end
        each gets a copy of its own, in one launch for all of them.  Parent and
        children are then requests like any other: appended to, read, and freed in
        any order; only a token in a block that others hold too is not written again
        (``check_writable``).  If the free list does not have a block for each copy,
        RuntimeError and nothing has changed."""
        self._validate_request(parent_id)
        request_ids = list(request_ids)
        num_tokens = self._counts[parent_id] if num_tokens is None else num_tokens
        if not 0 <= num_tokens <= self._counts[parent_id]:
            raise ValueError(f"num_tokens must lie in [0, {self._counts[parent_id]}]")
        for i, request_id in enumerate(request_ids):
            if request_id in self._tables or request_id in request_ids[:i]:
                raise ValueError(f"Request {request_id!r} already exists")
        if num_tokens % self.block_size and len(request_ids) > self.free_blocks:
            raise RuntimeError(f"Not enough KV blocks: required={len(request_ids)}, free={self.free_blocks}")
        pairs = []
        for request_id in request_ids:
            blocks, pair = self.block_manager.fork(parent_id, request_id, num_tokens)
            self._adopt(request_id, num_tokens, blocks)
            if pair is not None:
                pairs.append(pair)
        self.kv_cache.copy_blocks([a for a, _ in pairs], [b for _, b in pairs])

    def _adopt(self, request_id: str, num_tokens: int, blocks: list[int]) -> None:
        table = BlockTable()
        table._owner = self
        table._row = self._store_row()
        self._row_of[request_id] = table._row
        for blk in blocks:
            table.append(blk)
        self._tables[request_id] = table
        self._counts[request_id] = num_tokens
        self._store_tokens[table._row] = num_tokens
        self._epoch += 1

    def append_tokens(self, request_id: str, num_tokens: int) -> None:
        """Grow a request's capacity; new blocks only when a block boundary is crossed."""
        self._validate_request(request_id)
        if num_tokens < 0:
            raise ValueError("num_tokens cannot be negative")
        if num_tokens == 0:
            return
        old = self._counts[request_id]
        extra = self.block_manager.blocks_needed(old + num_tokens) - self.block_manager.blocks_needed(old)
        if extra > 0:
            for blk in self.block_manager.allocate_blocks(request_id=request_id, num_blocks=extra):
                self._tables[request_id].append(blk)
        self._counts[request_id] = old + num_tokens
        self._store_tokens[self._tables[request_id]._row] = old + num_tokens
        self._epoch += 1

    def free(self, request_id: str) -> None:
        self._validate_request(request_id)
        table = self._tables.pop(request_id)
        self._store_clear(table._row)
        self._free_rows.append(table._row)
        del self._row_of[request_id]
        table._owner, table._row = None, -1
        del self._counts[request_id]
        self.block_manager.free(request_id)
        self._epoch += 1

    # -- table store -------------------------------------------------------------
    def _store_row(self) -> int:
        if self._free_rows:
            return self._free_rows.pop()
        row = self._rows_used
        self._rows_used += 1
        if row >= self._store.shape[0]:
            grow = self._store.shape[0]
            self._store = np.concatenate([self._store, np.zeros_like(self._store[:grow])])
            self._store_blocks = np.concatenate([self._store_blocks, np.zeros(grow, dtype=np.int64)])
            self._store_tokens = np.concatenate([self._store_tokens, np.zeros(grow, dtype=np.int64)])
        return row

    def _store_put(self, row: int, index: int, block: int) -> None:
        if index >= self._store.shape[1]:
            width = max(2 * self._store.shape[1], index + 1)
            wider = np.zeros((self._store.shape[0], width), dtype=np.int32)
            wider[:, : self._store.shape[1]] = self._store
            self._store = wider
        self._store[row, index] = block
        self._store_blocks[row] = index + 1

    def _store_clear(self, row: int) -> None:
        self._store[row, :] = 0
        self._store_blocks[row] = 0
        self._store_tokens[row] = 0

    def _rows_of(self, request_ids) -> np.ndarray:
        try:  # one C-level pass over the id -> row map
            return np.fromiter(map(self._row_of.__getitem__, request_ids), dtype=np.int64, count=len(request_ids))
        except KeyError as e:
            raise KeyError(f"Unknown request: {e.args[0]!r}") from None

    # -- queries ---------------------------------------------------------------
    def get_block_table(self, request_id: str) -> BlockTable:
        self._validate_request(request_id)
        return self._tables[request_id]

    def token_count(self, request_id: str) -> int:
        self._validate_request(request_id)
        return self._counts[request_id]

    @property
    def metadata_epoch(self) -> int:
        """Changes whenever a request's blocks or token count change; the
        batched path reuses device copies of block tables built at the same
        epoch for the same requests and positions."""
        return self._epoch

    @property
    def free_blocks(self) -> int:
        return self.block_manager.free_blocks

    @property
    def used_blocks(self) -> int:
        return self.block_manager.used_blocks

    @property
    def num_blocks(self) -> int:
        return self.block_manager.num_blocks

    @property
    def block_size(self) -> int:
        return self.block_manager.block_size

    def _validate_request(self, request_id: str) -> None:
        if request_id not in self._tables:
            raise KeyError(f"Unknown request: {request_id!r}")

    # -- per-token access (reference semantics) -------------------------------
    def _locate(self, request_id: str, token_position: int) -> tuple[int, int]:
        self._validate_request(request_id)
        count = self._counts[request_id]
        if not 0 <= token_position < count:
            raise IndexError(f"Invalid token position: {token_position}; valid range is [0, {count})")
        bs = self.block_size
        return self._tables[request_id].get_physical_block(token_position // bs), token_position % bs

    def check_writable(self, request_ids, positions) -> None:
        """ValueError where a token lies in a block that other requests hold too
        (``fork``): written through one of them it would change for all."""
        shares = self.block_manager._shares
        if not shares:
            return
        rows = self._rows_of(request_ids)
        at = np.fromiter(positions, dtype=np.int64, count=len(rows)) // self.block_size
        for request_id, block in zip(request_ids, self._store[rows, at].tolist()):
            if block in shares:
                raise ValueError(f"Block {block} of request {request_id!r} is held by other requests too")

    def write_token(self, request_id: str, layer: int, token_position: int, key: torch.Tensor,
                    value: torch.Tensor) -> None:
        """Write one token's ``[Hkv, D]`` K/V at its logical position."""
        self._validate_request(request_id)
        block, offset = self._locate(request_id, token_position)
        shape = (self.kv_cache.num_kv_heads, self.kv_cache.head_dim)
        if tuple(key.shape) != shape or tuple(value.shape) != shape:
            raise ValueError(f"Expected K/V shape {shape}; got key={tuple(key.shape)}, value={tuple(value.shape)}")
        if key.dtype != self.kv_cache.dtype or value.dtype != self.kv_cache.dtype:
            raise ValueError(f"K/V tensors must have dtype {self.kv_cache.dtype}")
        self.check_writable((request_id,), (token_position,))
        if self.kv_cache.kv_bits == 4:
            kv = self.kv_cache
            if key.device != kv.kv_codes.device or value.device != kv.kv_codes.device:
                raise ValueError("K/V tensors must be on the same devices as their respective cache tensors")
            kv._write_rows(layer, self._slot_tensor(block, offset), key[None], value[None])
            return
        if key.device != self.kv_cache.k_cache.device or value.device != self.kv_cache.v_cache.device:
            raise ValueError("K/V tensors must be on the same devices as their respective cache tensors")
        self.kv_cache.k_cache[layer, block, :, offset, :].copy_(key)
        self.kv_cache.v_cache[layer, block, :, offset, :].copy_(value)

    def read_token(self, request_id: str, layer: int, token_position: int) -> tuple[torch.Tensor, torch.Tensor]:
        block, offset = self._locate(request_id, token_position)
        if self.kv_cache.kv_bits == 4:
            key, value = self.kv_cache._read_rows(layer, self._slot_tensor(block, offset))
            return key[0], value[0]
        return (self.kv_cache.k_cache[layer, block, :, offset, :], self.kv_cache.v_cache[layer, block, :, offset, :])

    def _slot_tensor(self, block: int, offset: int) -> torch.Tensor:
        return torch.full((1,), block * self.block_size + offset, dtype=torch.int64, device=self.kv_cache.device)

    # -- batched helpers for the B200 path -----------------------------------
    def slot_of(self, request_id: str, token_position: int) -> int:
        """int64 slot (``block * block_size + offset``) of a logical position."""
        block, offset = self._locate(request_id, token_position)
        return block * self.block_size + offset

    def table_rows(self, request_ids, width: int | None = None) -> np.ndarray:
        """Zero-padded int32 ``[B, width]`` block table of ``request_ids``
        (width: the longest of their tables by default)."""
        rows = self._rows_of(request_ids)
        if width is None:
            width = int(self._store_blocks[rows].max()) if len(rows) else 0
        width = max(width, 1)
        have = min(width, self._store.shape[1])
        if have == width:
            return self._store[rows, :width]
        out = np.zeros((len(rows), width), dtype=np.int32)
        out[:, :have] = self._store[rows, :have]
        return out

    def table_store_rows(self, request_ids) -> np.ndarray:
        """int64 ``[B]`` rows of ``request_ids`` in the table store (for
        ``gather_tables``; raises KeyError for an unknown request)."""
        return self._rows_of(request_ids)

    def table_width(self, rows: np.ndarray) -> int:
        """Blocks in the longest table of store ``rows`` (at least 1)."""
        return max(int(self._store_blocks[rows].max()), 1) if len(rows) else 1

    def gather_tables(self, rows: np.ndarray, out: np.ndarray, width: int) -> None:
        """Write the block tables of store ``rows``, zero padded to ``width``
        (>= ``table_width(rows)``), into the first ``len(rows) * width``
        elements of ``out`` (int32, C-contiguous) as ``[B, width]``."""
        dst = out[: len(rows) * width].reshape(len(rows), width)
        have = min(width, self._store.shape[1])
        np.take(self._store[:, :have], rows, axis=0, out=dst[:, :have] if have == width else None, mode="clip")
        if have < width:
            dst[:, :have] = self._store[rows, :have]
            dst[:, have:] = 0

    def shared_prefixes(self, request_ids) -> tuple[np.ndarray, np.ndarray]:
        """``(cu_groups [G + 1], prefix_lens [G])`` int32 for ``ops.paged_decode_shared``
        over these requests in this order: neighbours with the same first block are a
        group, the blocks that all of it begins with are its prefix."""
        rows = self._rows_of(request_ids)
        n = len(rows)
        if n == 0:
            return np.zeros(1, dtype=np.int32), np.zeros(0, dtype=np.int32)
        first, have = self._store[rows, 0], self._store_blocks[rows]
        new = np.ones(n, dtype=bool)
        new[1:] = (first[1:] != first[:-1]) | (have[1:] == 0) | (have[:-1] == 0)
        cu = np.append(np.flatnonzero(new), n).astype(np.int32)
        prefix = np.zeros(len(cu) - 1, dtype=np.int32)
        for g in np.flatnonzero(np.diff(cu) > 1):
            members = rows[cu[g]:cu[g + 1]]
            most = int(self._store_blocks[members].min())
            tables = self._store[members, :most]
            differs = np.flatnonzero((tables != tables[0]).any(axis=0))
            blocks = int(differs[0]) if len(differs) else most
            prefix[g] = min(blocks * self.block_size, int(self._store_tokens[members].min()))
        return cu, prefix

    def store_token_counts(self, rows: np.ndarray) -> np.ndarray:
        """int64 token counts of store ``rows``."""
        return self._store_tokens[rows]

    def token_counts(self, request_ids) -> np.ndarray:
        """int64 ``[B]`` token counts of ``request_ids``."""
        return self._store_tokens[self._rows_of(request_ids)]
