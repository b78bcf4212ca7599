"""KV page pools for this package's own decode step, benchmarks and tests.

The reference runtime keeps its own pool class (``mini_engine/cache/kv_cache.py``);
through :func:`myvllm_mini_engine_b200.integration.install` it calls the kernels
here with that class's per-layer views.  The pools below hold the same layout,
``[layers, num_blocks, block_size, kv_heads, head_dim]`` per tensor
(kv_cache.py:50-52), and expose ``key``, ``value`` and ``shape`` under the same
names, so :class:`~myvllm_mini_engine_b200.engine.qwen3.Qwen3DecodeStep`
accepts either the reference pool or one of these.

* :class:`PagedKVPool`: 16-bit (or fp32) pages.  Both pools live in one
  allocation ``[2, layers, ...]``, so a step's K and V pages of a layer are one
  address range apart and a single free returns them.
* :class:`FP8KVCachePool`: one OCP FP8 byte per element plus a scale per pool.
* :class:`INT4KVCachePool`: 4-bit codes with a step and a base per row.

A 16-bit or 4-bit pool made with ``block_bounds=True`` also holds the key bounds
of its blocks (``kernels.update_block_bounds``), from which a decode step can
select the blocks it attends.

Page-id checks are done on the host for Python sequences (no device sync) and
with one reduction for device tensors.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from ..kernels.data import copy_blocks, write_kv_cache


@dataclass(frozen=True)
class PoolShape:
    """Geometry of a pool; the field names are the ones the reference pool's ``shape`` carries."""

    num_layers: int
    num_blocks: int
    block_size: int
    num_kv_heads: int
    head_dim: int

    @property
    def row_elems(self) -> int:
        return self.num_kv_heads * self.head_dim


def _geometry(values) -> PoolShape:
    if any(int(v) <= 0 for v in values):
        raise ValueError("all KV cache dimensions must be positive")
    return PoolShape(*(int(v) for v in values))


def _page_tensor(block_ids, shape: PoolShape, device) -> torch.Tensor:
    """Page ids as a flat int64 tensor on ``device``; IndexError if one is outside the pool."""
    if isinstance(block_ids, torch.Tensor):
        ids = block_ids.reshape(-1).to(device=device, dtype=torch.long)
        if ids.numel():
            lo, hi = torch.aminmax(ids)
            if int(lo) < 0 or int(hi) >= shape.num_blocks:
                raise IndexError("physical block id out of range")
        return ids
    host = np.asarray(list(block_ids), dtype=np.int64).reshape(-1)
    if host.size and (host.min() < 0 or host.max() >= shape.num_blocks):
        raise IndexError("physical block id out of range")
    return torch.from_numpy(host).to(device)


class _Pool:
    shape: PoolShape
    key: torch.Tensor
    value: torch.Tensor

    def _check_layer(self, layer):
        if not 0 <= layer < self.shape.num_layers:
            raise IndexError("layer out of range")

    def _check_range(self, ids, token_offset, tokens):
        if token_offset < 0 or token_offset + tokens > ids.numel() * self.shape.block_size:
            raise ValueError("write exceeds supplied block table capacity")

    @property
    def memory_bytes(self) -> int:
        """Bytes of the K and V pages (the block bounds of a pool that has them: ``bounds_bytes``)."""
        return (self.key.numel() + self.value.numel()) * self.key.element_size()

    def layer(self, index):
        """``(key, value)`` views of one layer: ``[num_blocks, block_size, kv_heads, head_dim]``."""
        self._check_layer(index)
        return self.key[index], self.value[index]


class _BoundedPool(_Pool):
    """Key bounds of a pool's blocks: ``bounds`` ``[layers, num_blocks, kv_heads, 2 * head_dim + 16]`` or None.

    Like the pages they belong to, they are the caller's to keep up to date: after
    every write of a layer's rows, :meth:`update_bounds`.
    """

    bounds: torch.Tensor | None = None

    @property
    def bounds_bytes(self) -> int:
        """Bytes of the block bounds, 0 without: at head_dim 128 and pages of 16 an eighth of a 4-bit pool's pages."""
        return 0 if self.bounds is None else self.bounds.numel()

    def _make_bounds(self, wanted):
        from ..kernels.sparse import block_bounds_bytes

        if wanted:
            s = self.shape
            self.bounds = torch.zeros((s.num_layers, s.num_blocks, s.num_kv_heads, block_bounds_bytes(s.head_dim)),
                                      dtype=torch.uint8, device=self.device)

    def _layer_bounds(self, layer):
        self._check_layer(layer)
        if self.bounds is None:
            raise ValueError("the pool holds no block bounds (block_bounds=True)")
        return self.bounds[layer]

    def update_bounds(self, layer, block_tables, query_starts, context_lens, *, validate=True, max_query_len=None):
        """Bounds of the blocks that hold rows ``[query_starts[r], context_lens[r])`` of each request."""
        from ..kernels.sparse import update_block_bounds

        update_block_bounds(self._layer_bounds(layer), self.key[layer], block_tables, query_starts, context_lens,
                            self.shape.block_size, validate=validate, max_query_len=max_query_len)

    def select_blocks(self, layer, query, block_tables, context_lens, max_blocks, *, sink_blocks=1, recent_blocks=1,
                      validate=True):
        """The blocks of highest score for each request and kv head (``kernels.select_blocks``)."""
        from ..kernels.sparse import select_blocks

        return select_blocks(query, self._layer_bounds(layer), block_tables, context_lens, self.shape.block_size,
                             max_blocks, sink_blocks=sink_blocks, recent_blocks=recent_blocks, validate=validate)

    def _copy_bounds(self, pairs) -> None:
        """Copy-on-write of the pages' bounds, as 16-bit words."""
        if self.bounds is not None:
            words = self.bounds.view(torch.bfloat16)
            words = words.view(*words.shape[:2], 1, *words.shape[2:])
            copy_blocks(words, words, pairs)  # the bounds are one pool: both copies write the same bytes


class PagedKVPool(_BoundedPool):
    """K and V pages of every layer, one contiguous allocation ``[2, layers, blocks, bs, kv_heads, D]``."""

    def __init__(self, num_layers, num_blocks, block_size, num_kv_heads, head_dim, *,
                 dtype=torch.bfloat16, device="cuda", block_bounds=False):
        self.shape = _geometry((num_layers, num_blocks, block_size, num_kv_heads, head_dim))
        self.dtype = dtype
        self.storage = torch.empty((2, *map(int, (num_layers, num_blocks, block_size, num_kv_heads, head_dim))),
                                   dtype=dtype, device=device)
        self.key, self.value = self.storage[0], self.storage[1]
        self.device = self.storage.device
        if block_bounds and dtype == torch.float32:
            raise ValueError("block bounds are kept for 16-bit and 4-bit pools")
        self._make_bounds(block_bounds)

    def write_range(self, layer, block_ids, token_offset, key, value, *, validate=True) -> None:
        """Write ``[tokens, kv_heads, head_dim]`` rows at logical positions ``token_offset...`` of a page list."""
        self._check_layer(layer)
        if key.ndim != 3 or key.shape != value.shape:
            raise ValueError("key and value must both have shape [tokens, kv_heads, head_dim]")
        ids = _page_tensor(block_ids, self.shape, self.device)
        self._check_range(ids, token_offset, key.shape[0])
        write_kv_cache(self.key[layer], self.value[layer], ids, token_offset, key, value, self.shape.block_size,
                       validate=validate)

    def copy_blocks(self, pairs) -> None:
        """Apply copy-on-write ``(src, dst)`` page pairs to every layer of both pools (and of the bounds)."""
        copy_blocks(self.key, self.value, pairs)
        self._copy_bounds(pairs)


class FP8KVCachePool(_Pool):
    """FP8 paged KV pool: the layout of :class:`PagedKVPool` with one byte per element.

    ``key``/``value`` are uint8 ``[layers, num_blocks, block_size, kv_heads,
    head_dim]`` tensors of OCP FP8 codes (``kv_format`` "e4m3" or "e5m2") with one
    fp32 scale for keys and one for values: an element ``x`` is stored as
    ``fp8(x * (1/scale))`` and read as ``code * scale``.  It holds twice the tokens
    of a bf16 pool in the same memory.  The reference has no FP8 pool;
    :meth:`attend` runs the decode attention of one layer.
    """

    def __init__(self, num_layers, num_blocks, block_size, num_kv_heads, head_dim, *, k_scale, v_scale,
                 kv_format="e4m3", device="cuda"):
        from ..kernels.fp8 import FORMATS, _scale

        self.shape = _geometry((num_layers, num_blocks, block_size, num_kv_heads, head_dim))
        if kv_format not in FORMATS:
            raise ValueError("kv_format must be 'e4m3' or 'e5m2'")
        if int(head_dim) % 2:
            raise ValueError("an fp8 pool needs an even head_dim (copy-on-write moves 16-bit words)")
        self.kv_format = kv_format
        self.k_scale, self.v_scale = _scale(k_scale, "k_scale"), _scale(v_scale, "v_scale")
        self.storage = torch.zeros((2, num_layers, num_blocks, block_size, num_kv_heads, head_dim),
                                   dtype=torch.uint8, device=device)
        self.key, self.value = self.storage[0], self.storage[1]
        self.device = self.storage.device

    def write_slots(self, layer, slot_mapping, key, value, *, validate=True) -> None:
        """Quantise ``key``/``value`` ``[tokens, kv_heads, head_dim]`` into rows ``slot_mapping`` of a layer."""
        from ..kernels.fp8 import write_kv_cache_slots_fp8

        self._check_layer(layer)
        write_kv_cache_slots_fp8(self.key[layer], self.value[layer], slot_mapping, key, value, self.k_scale,
                                 self.v_scale, kv_format=self.kv_format, validate=validate)

    def write_range(self, layer, block_ids, token_offset, key, value, *, validate=True) -> None:
        """Quantise a contiguous token range across pages; the slots are computed on the device."""
        if key.ndim != 3 or key.shape != value.shape:
            raise ValueError("key and value must both have shape [tokens, kv_heads, head_dim]")
        self._check_layer(layer)
        ids = _page_tensor(block_ids, self.shape, self.device)
        self._check_range(ids, token_offset, key.shape[0])
        if key.device != self.device or value.device != self.device:
            raise ValueError("CUDA KV write inputs must be on the cache device")
        bs = self.shape.block_size
        positions = torch.arange(key.shape[0], device=self.device, dtype=torch.long) + int(token_offset)
        self.write_slots(layer, ids[positions // bs] * bs + positions % bs, key, value, validate=False)

    def attend(self, layer, query, block_tables, context_lens, *, validate=True, workspace=None):
        """Decode attention of one layer over this pool (``paged_attention_fp8``)."""
        from ..kernels.fp8 import paged_attention_fp8

        self._check_layer(layer)
        return paged_attention_fp8(query, self.key[layer], self.value[layer], block_tables, context_lens,
                                   self.shape.block_size, self.k_scale, self.v_scale, kv_format=self.kv_format,
                                   validate=validate, workspace=workspace)

    def dequantized(self, layer, block_ids, token_count, dtype=torch.float32):
        """The first ``token_count`` logical rows of a page list, dequantised: ``(key, value)``."""
        self._check_layer(layer)
        ids = _page_tensor(block_ids, self.shape, self.device)
        if not 0 <= token_count <= ids.numel() * self.shape.block_size:
            raise ValueError("token_count must lie within the supplied block table capacity")
        fp8 = torch.float8_e4m3fn if self.kv_format == "e4m3" else torch.float8_e5m2
        out = []
        for codes, scale in ((self.key[layer], self.k_scale), (self.value[layer], self.v_scale)):
            rows = codes.index_select(0, ids).view(-1, self.shape.num_kv_heads, self.shape.head_dim)
            out.append(rows[:token_count].view(fp8).to(dtype) * scale)
        return tuple(out)

    def copy_blocks(self, pairs) -> None:
        """Apply copy-on-write ``(src, dst)`` pairs to every layer of both pools (16-bit word moves)."""
        copy_blocks(self.key.view(torch.bfloat16), self.value.view(torch.bfloat16), pairs)


class INT4KVCachePool(_BoundedPool):
    """4-bit paged KV pool: codes with an fp16 step and base per row (``kernels/int4.py``).

    ``key``/``value`` are uint8 ``[layers, num_blocks, kv_heads, page_bytes]``.  At
    head_dim 128 a row takes 68 bytes, so the pool holds 3.76 times the tokens of a
    bf16 pool in the same memory.  The reference has no 4-bit pool.
    """

    def __init__(self, num_layers, num_blocks, block_size, num_kv_heads, head_dim, *, device="cuda",
                 block_bounds=False):
        from ..kernels.int4 import int4_page_bytes

        self.shape = _geometry((num_layers, num_blocks, block_size, num_kv_heads, head_dim))
        self.page_bytes = int4_page_bytes(int(block_size), int(head_dim))
        self.storage = torch.zeros((2, num_layers, num_blocks, num_kv_heads, self.page_bytes), dtype=torch.uint8,
                                   device=device)
        self.key, self.value = self.storage[0], self.storage[1]
        self.device = self.storage.device
        self._make_bounds(block_bounds)

    def write_slots(self, layer, slot_mapping, key, value, *, validate=True) -> None:
        """Quantise ``key``/``value`` ``[tokens, kv_heads, head_dim]`` into rows ``slot_mapping`` of a layer."""
        from ..kernels.int4 import write_kv_cache_slots_int4

        self._check_layer(layer)
        write_kv_cache_slots_int4(self.key[layer], self.value[layer], slot_mapping, key, value,
                                  self.shape.block_size, validate=validate)

    def write_batch(self, layer, block_tables, token_offsets, key, value, *, validate=True) -> None:
        """Quantise one new row per request at position ``token_offsets[b]`` (the decode append)."""
        from ..kernels.int4 import write_kv_cache_batch_int4

        self._check_layer(layer)
        write_kv_cache_batch_int4(self.key[layer], self.value[layer], block_tables, token_offsets, key, value,
                                  self.shape.block_size, validate=validate)

    def write_range(self, layer, block_ids, token_offset, key, value, *, validate=True) -> None:
        """Quantise a contiguous token range across pages; the slots are computed on the device."""
        if key.ndim != 3 or key.shape != value.shape:
            raise ValueError("key and value must both have shape [tokens, kv_heads, head_dim]")
        self._check_layer(layer)
        ids = _page_tensor(block_ids, self.shape, self.device)
        self._check_range(ids, token_offset, key.shape[0])
        bs = self.shape.block_size
        positions = torch.arange(key.shape[0], device=self.device, dtype=torch.long) + int(token_offset)
        self.write_slots(layer, ids[positions // bs] * bs + positions % bs, key, value, validate=False)

    def attend(self, layer, query, block_tables, context_lens, *, selected=None, validate=True):
        """Decode attention of one layer over this pool, or over selected blocks of it (``paged_attention_int4``)."""
        from ..kernels.int4 import paged_attention_int4

        self._check_layer(layer)
        return paged_attention_int4(query, self.key[layer], self.value[layer], block_tables, context_lens,
                                    self.shape.block_size, selected=selected, validate=validate)

    def prefill(self, layer, q, cu_seqlens_q, query_starts, block_tables, context_lens, *, validate=True,
                max_query_len=None):
        """Ragged causal prefill of one layer over this pool (``paged_prefill_attention_int4``)."""
        from ..kernels.int4 import paged_prefill_attention_int4

        self._check_layer(layer)
        return paged_prefill_attention_int4(q, self.key[layer], self.value[layer], cu_seqlens_q, query_starts,
                                            block_tables, context_lens, self.shape.block_size, validate=validate,
                                            max_query_len=max_query_len)

    def dequantized(self, layer, block_ids, token_count, dtype=torch.float32):
        """The first ``token_count`` logical rows of a page list, dequantised: ``(key, value)``."""
        from ..kernels.int4 import read_kv_cache_slots_int4

        self._check_layer(layer)
        ids = _page_tensor(block_ids, self.shape, self.device)
        bs = self.shape.block_size
        if not 0 <= token_count <= ids.numel() * bs:
            raise ValueError("token_count must lie within the supplied block table capacity")
        positions = torch.arange(token_count, device=self.device, dtype=torch.long)
        return read_kv_cache_slots_int4(self.key[layer], self.value[layer], ids[positions // bs] * bs + positions % bs,
                                        bs, self.shape.head_dim, dtype=dtype, validate=False)

    def copy_blocks(self, pairs) -> None:
        """Apply copy-on-write ``(src, dst)`` pairs to every layer of both pools and of the bounds (16-bit words)."""
        key, value = (pool.view(torch.bfloat16).unsqueeze(2) for pool in (self.key, self.value))
        copy_blocks(key, value, pairs)
        self._copy_bounds(pairs)
