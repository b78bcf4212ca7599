"""Attention over selected blocks: block bounds, selection, and the decode over the selection.

No counterpart in the reference.  At long contexts most blocks (pages) of a
request get next to no weight.  Three steps read only those that can matter:

1. :func:`update_block_bounds` keeps, for every block and kv head, bounds of its
   keys in 8 bits (after each write: a prompt chunk, or a decode step's row);
2. :func:`select_blocks` scores every block of a request against the new query
   and lists the blocks of highest score for each kv head;
3. :func:`paged_attention_selected` (16-bit pools) or
   ``paged_attention_int4(..., selected=...)`` attends the listed blocks.

Bounds are a contiguous uint8 tensor ``[num_blocks, kv_heads, 2 * head_dim + 16]``:
``head_dim`` int8 codes of the keys' elementwise maximum, ``head_dim`` of their
minimum, one fp32 scale; a bound reads as ``code * scale`` (it holds up to two fp32
roundings, 2^-23 of it).  A score estimates the bound of ``sum_h q_h . k`` over the
query heads h of a kv head and the keys k of the block, with the query's parts
rounded to 8 bits; the codes' products sum to a whole number, so a selection is
the same whatever the batch, the split or the order of evaluation.
"""

from __future__ import annotations

import torch

from .. import _lib
from .int4 import _QUERY_DTYPES, INT4_HEAD_DIMS, _decode_pages, _device_of, int4_page_bytes
from .paged import _require, check_backend

_INT4 = 3  # MINIKV_INT4


def block_bounds_bytes(head_dim):
    """Bytes of one block's bounds for one kv head."""
    if head_dim not in INT4_HEAD_DIMS:
        raise ValueError("block bounds need head_dim 32, 64, 96, 128, 192 or 256")
    return 2 * head_dim + 16


def _check_bounds(bounds):
    """``(num_blocks, kv_heads, head_dim)`` of a bounds tensor."""
    shape = bounds.shape
    if len(shape) != 3 or bounds.dtype is not torch.uint8 or not bounds.is_contiguous() or 0 in shape:
        raise RuntimeError("block bounds must be contiguous uint8 [pages, kv_heads, 2 * head_dim + 16]")
    dim = (shape[2] - 16) // 2
    if dim not in INT4_HEAD_DIMS or shape[2] != 2 * dim + 16:
        raise RuntimeError("block bounds need head_dim 32, 64, 96, 128, 192 or 256")
    return shape[0], shape[1], dim


def update_block_bounds(bounds, key_cache, block_tables, query_starts, context_lens, block_size, *, backend="cuda",
                        validate=True, max_query_len=None):
    """Recompute the bounds of the blocks that hold rows ``[query_starts[r], context_lens[r])`` of each request.

    ``key_cache`` is a 16-bit or fp32 pool ``[num_blocks, block_size, kv_heads,
    head_dim]`` or a 4-bit pool ``[num_blocks, kv_heads, page_bytes]``.  A block's
    bounds cover all of its rows below ``context_lens[r]``.  For a decode step pass
    the new row's position and position + 1.  ``max_query_len`` (optional) bounds
    ``context_lens - query_starts`` on the host; blocks past it are not updated
    (refused with ``validate``).  Empty ranges update nothing; out-of-range requests
    and pages are skipped (refused with ``validate``).  A block that several requests
    name has to hold the same rows for each of them, as full shared blocks do; its
    bounds would depend on their order else (refused with ``validate``).
    """
    check_backend(backend)
    num_blocks, kv_heads, dim = _check_bounds(bounds)
    if type(block_size) is not int or block_size <= 0:
        raise RuntimeError("block size mismatch")
    if key_cache.dtype is torch.uint8:
        pool = _INT4
        if key_cache.shape != (num_blocks, kv_heads, int4_page_bytes(block_size, dim)):
            raise RuntimeError("4-bit key cache must be [pages, kv_heads, page_bytes] matching the bounds")
    else:
        pool = _lib.dtype_code(key_cache.dtype)
        if key_cache.shape != (num_blocks, block_size, kv_heads, dim):
            raise RuntimeError("key cache must be [pages, block_size, kv_heads, head_dim] matching the bounds")
    if not bounds.is_cuda:
        raise RuntimeError("bounds must be CUDA")
    device = _device_of((bounds, key_cache, block_tables, query_starts, context_lens), RuntimeError,
                        "all inputs must be on the same CUDA device")
    if not (key_cache.is_contiguous() and block_tables.is_contiguous() and query_starts.is_contiguous()
            and context_lens.is_contiguous()):
        raise RuntimeError("inputs must be contiguous")
    if (block_tables.dtype is not torch.int64 or query_starts.dtype is not torch.int64
            or context_lens.dtype is not torch.int64):
        raise RuntimeError("metadata must be int64")
    if (query_starts.dim() != 1 or context_lens.shape != query_starts.shape or block_tables.dim() != 2
            or block_tables.shape[0] != query_starts.shape[0] or block_tables.shape[1] <= 0):
        raise RuntimeError("block bounds metadata shapes do not match request count")
    requests, width = block_tables.shape
    if width * block_size > 1048576:
        raise RuntimeError("maximum table capacity is 1M tokens")
    if validate and requests:
        _require(not bool(((query_starts < 0) | (query_starts > context_lens)
                           | (context_lens > width * block_size)).any()), "invalid context length")
        column = torch.arange(width, device=bounds.device, dtype=torch.int64)
        active = ((column >= (query_starts // block_size)[:, None]) & (column * block_size < context_lens[:, None])
                  & (query_starts < context_lens)[:, None])
        _require(not bool((((block_tables < 0) | (block_tables >= num_blocks)) & active).any()),
                 "physical block id out of range")
        _require(max_query_len is None or not bool((context_lens - query_starts > int(max_query_len)).any()),
                 "max_query_len is below a request's rows")
        pages = block_tables[active]
        rows = (context_lens[:, None] - column * block_size).clamp(max=block_size)[active]
        _require(pages.unique().numel() == (pages * (block_size + 1) + rows).unique().numel(),
                 "a block of several requests must hold the same rows for each")
    if requests == 0:
        return
    longest = width * block_size if max_query_len is None else int(max_query_len)
    lib = _lib.load()
    with _lib.on_device(device):
        status = lib.minikv_block_bounds_update(
            bounds.data_ptr(), key_cache.data_ptr(), block_tables.data_ptr(), query_starts.data_ptr(),
            context_lens.data_ptr(), requests, width, num_blocks, block_size, kv_heads, dim, longest, pool,
            _lib.stream_of(device))
    if status:
        _lib.check(status, "update_block_bounds")


def read_block_bounds(bounds, block_ids, *, validate=True):
    """Values of the bounds of blocks ``block_ids`` (int64 ``[n]``): ``(lower, upper)`` fp32 ``[n, kv_heads, head_dim]``.

    A block outside the pool gives zeros (refused with ``validate``).
    """
    num_blocks, kv_heads, dim = _check_bounds(bounds)
    if not bounds.is_cuda or block_ids.get_device() != bounds.get_device():
        raise RuntimeError("all inputs must be on the same CUDA device")
    if block_ids.dim() != 1 or block_ids.dtype is not torch.int64 or not block_ids.is_contiguous():
        raise RuntimeError("block ids must be contiguous int64 [n]")
    count = block_ids.shape[0]
    if validate and count:
        _require(not bool(((block_ids < 0) | (block_ids >= num_blocks)).any()), "physical block id out of range")
    device = bounds.device
    lower = torch.empty((count, kv_heads, dim), dtype=torch.float32, device=device)
    upper = torch.empty_like(lower)
    if count == 0:
        return lower, upper
    lib = _lib.load()
    with _lib.on_device(device):
        status = lib.minikv_block_bounds_read(bounds.data_ptr(), block_ids.data_ptr(), count, lower.data_ptr(),
                                              upper.data_ptr(), num_blocks, kv_heads, dim, _lib.stream_of(device))
    if status:
        _lib.check(status, "read_block_bounds")
    return lower, upper


def select_blocks(query, bounds, block_tables, context_lens, block_size, max_blocks, *, sink_blocks=1,
                  recent_blocks=1, backend="cuda", validate=True):
    """The ``max_blocks`` blocks of highest score of each request and kv head: int64 ``[B, Hkv, max_blocks]``.

    ``query [B, Hq, D]`` fp32/fp16/bf16.  Logical block numbers in ascending order,
    -1 behind the last; equal scores go to the lowest block.  The first
    ``sink_blocks`` and the last ``recent_blocks`` blocks of a request are taken
    whatever their scores; a request of no more than ``max_blocks`` blocks takes all
    of them.  The bounds of every block below ``context_lens`` must be up to date.
    """
    check_backend(backend)
    if not query.is_cuda:
        raise RuntimeError("query must be CUDA")
    num_blocks, kv_heads, dim = _check_bounds(bounds)
    shape = query.shape
    if len(shape) != 3 or shape[2] != dim or shape[1] % kv_heads or 0 in shape:
        raise RuntimeError("head dimension or GQA mismatch")
    batch, heads, _ = shape
    code = _lib.dtype_code(query.dtype)
    device = _device_of((query, bounds, block_tables, context_lens), RuntimeError,
                        "all inputs must be on the same CUDA device")
    if not (query.is_contiguous() and block_tables.is_contiguous() and context_lens.is_contiguous()):
        raise RuntimeError("inputs must be contiguous")
    if block_tables.dtype is not torch.int64 or context_lens.dtype is not torch.int64:
        raise RuntimeError("metadata must be int64")
    if block_tables.dim() != 2 or block_tables.shape[0] != batch or block_tables.shape[1] <= 0:
        raise RuntimeError("invalid block table")
    if context_lens.shape != (batch,):
        raise RuntimeError("invalid context lengths")
    if type(block_size) is not int or block_size <= 0:
        raise RuntimeError("block size mismatch")
    width = block_tables.shape[1]
    if width * block_size > 1048576:
        raise RuntimeError("maximum table capacity is 1M tokens")
    if max_blocks <= 0 or sink_blocks < 0 or recent_blocks < 0 or sink_blocks + recent_blocks > max_blocks:
        raise RuntimeError("max_blocks must be positive and hold the sink and recent blocks")
    if validate:
        _require(not bool(((context_lens <= 0) | (context_lens > width * block_size)).any()),
                 "invalid context length")
        column = torch.arange(width, device=device, dtype=torch.int64) * block_size
        active = column.unsqueeze(0) < context_lens.unsqueeze(1)
        _require(not bool((((block_tables < 0) | (block_tables >= num_blocks)) & active).any()),
                 "physical block id out of range")
    lib = _lib.load()
    with _lib.on_device(device):
        workspace = torch.empty(batch * kv_heads * width, dtype=torch.int32, device=device)
        selected = torch.empty((batch, kv_heads, max_blocks), dtype=torch.int64, device=device)
        status = lib.minikv_select_blocks(
            query.data_ptr(), bounds.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), selected.data_ptr(),
            workspace.data_ptr(), workspace.numel() * 4, batch, heads, kv_heads, dim, num_blocks, block_size,
            width, max_blocks, sink_blocks, recent_blocks, code, _lib.stream_of(device))
    if status:
        _lib.check(status, "select_blocks")
    return selected


def paged_attention_selected(query, key_cache, value_cache, block_tables, context_lens, selected, block_size, *,
                             backend="cuda", validate=True):
    """Decode attention over the selected blocks of 16-bit pools.

    :func:`paged_attention` restricted, for each kv head, to the logical blocks
    ``selected [B, Hkv, K]`` (int64, from :func:`select_blocks`): ascending, -1
    behind the last; the first ``min(K, blocks of the request)`` entries are read.
    fp16/bf16 pools, head_dim 32, 64, 96, 128, 192 or 256.  A row whose every token
    is masked gives zeros.  Returns ``[B, Hq, D]``.
    """
    check_backend(backend)
    if not query.is_cuda:
        raise RuntimeError("query must be CUDA")
    shape = key_cache.shape
    if query.dim() != 3 or len(shape) != 4 or value_cache.shape != shape or 0 in shape:
        raise RuntimeError("invalid query/cache shapes")
    if query.dtype not in _QUERY_DTYPES:
        raise RuntimeError("FP16/BF16 required")
    if key_cache.dtype is not query.dtype or value_cache.dtype is not query.dtype:
        raise RuntimeError("cache dtype mismatch")
    num_blocks, bs, kv_heads, dim = shape
    if type(block_size) is not int or bs != block_size:
        raise RuntimeError("block size mismatch")
    if query.shape[2] != dim:
        raise RuntimeError("head dimension or GQA mismatch")
    if dim not in INT4_HEAD_DIMS:
        raise RuntimeError("selected blocks: supported head_dim: 32,64,96,128,192,256")
    return _decode_pages("minikv_paged_decode_selected", "minikv_paged_decode_selected_workspace_bytes", query,
                         key_cache, value_cache, block_tables, context_lens, selected, block_size, num_blocks,
                         kv_heads, validate)
