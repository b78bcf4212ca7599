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
minimum, one fp32 scale; a bound reads as ``code * scale``.  A score is a bound of
``sum_h q_h . k`` over the query heads h of a kv head and the keys k of the block;
the codes' products sum to a whole number, so a selection is the same whatever
the batch, the split or the order of evaluation.
"""

from __future__ import annotations

import torch

from .. import _lib
from .int4 import INT4_HEAD_DIMS, _decode_pages, int4_page_bytes
from .paged import _require, check_backend

_INT4 = 3  # MINIKV_INT4


def block_bounds_bytes(head_dim):
    """Bytes of one block's bounds for one kv head."""
    if head_dim not in INT4_HEAD_DIMS:
        raise ValueError("block bounds need head_dim 32, 64, 96, 128, 192 or 256")
    return 2 * head_dim + 16


def _check_bounds(bounds):
    """``(num_blocks, kv_heads, head_dim)`` of a bounds tensor."""
    _require(bounds.dim() == 3 and bounds.dtype == torch.uint8 and bounds.is_contiguous() and bounds.numel() > 0,
             "block bounds must be contiguous uint8 [pages, kv_heads, 2 * head_dim + 16]")
    dim = (bounds.shape[2] - 16) // 2
    _require(dim in INT4_HEAD_DIMS and bounds.shape[2] == 2 * dim + 16,
             "block bounds need head_dim 32, 64, 96, 128, 192 or 256")
    return bounds.shape[0], bounds.shape[1], dim


def update_block_bounds(bounds, key_cache, block_tables, query_starts, context_lens, block_size, *, backend="cuda",
                        validate=True, max_query_len=None):
    """Recompute the bounds of the blocks that hold rows ``[query_starts[r], context_lens[r])`` of each request.

    ``key_cache`` is a 16-bit or fp32 pool ``[num_blocks, block_size, kv_heads,
    head_dim]`` or a 4-bit pool ``[num_blocks, kv_heads, page_bytes]``.  A block's
    bounds cover all of its rows below ``context_lens[r]``.  For a decode step pass
    the new row's position and position + 1.  ``max_query_len`` (optional) bounds
    ``context_lens - query_starts`` on the host; blocks past it are not updated.
    Empty ranges update nothing; out-of-range requests and pages are skipped
    (refused with ``validate``).
    """
    check_backend(backend)
    num_blocks, kv_heads, dim = _check_bounds(bounds)
    if key_cache.dtype == torch.uint8:
        pool = _INT4
        _require(key_cache.dim() == 3 and type(block_size) is int and block_size > 0
                 and key_cache.shape == (num_blocks, kv_heads, int4_page_bytes(block_size, dim)),
                 "4-bit key cache must be [pages, kv_heads, page_bytes] matching the bounds")
    else:
        pool = _lib.dtype_code(key_cache.dtype)
        _require(key_cache.dim() == 4 and type(block_size) is int
                 and key_cache.shape == (num_blocks, block_size, kv_heads, dim),
                 "key cache must be [pages, block_size, kv_heads, head_dim] matching the bounds")
    _require(bounds.is_cuda, "bounds must be CUDA")
    tensors = (key_cache, block_tables, query_starts, context_lens)
    _require(all(t.device == bounds.device for t in tensors), "all inputs must be on the same CUDA device")
    _require(all(t.is_contiguous() for t in tensors), "inputs must be contiguous")
    _require(all(t.dtype == torch.int64 for t in tensors[1:]), "metadata must be int64")
    requests = query_starts.shape[0] if query_starts.dim() == 1 else -1
    _require(requests >= 0 and context_lens.dim() == 1 and context_lens.shape[0] == requests
             and block_tables.dim() == 2 and block_tables.shape[0] == requests and block_tables.shape[1] > 0,
             "block bounds metadata shapes do not match request count")
    width = block_tables.shape[1]
    _require(width * block_size <= 1048576, "maximum table capacity is 1M tokens")
    if validate and requests:
        _require(not bool(((query_starts < 0) | (query_starts > context_lens)
                           | (context_lens > width * block_size)).any()), "invalid context length")
        column = torch.arange(width, device=bounds.device, dtype=torch.int64)
        active = ((column >= (query_starts // block_size)[:, None]) & (column * block_size < context_lens[:, None])
                  & (query_starts < context_lens)[:, None])
        _require(not bool((((block_tables < 0) | (block_tables >= num_blocks)) & active).any()),
                 "physical block id out of range")
    if requests == 0:
        return
    longest = width * block_size if max_query_len is None else int(max_query_len)
    lib = _lib.load()
    with _lib.on_device(bounds.device):
        status = lib.minikv_block_bounds_update(
            bounds.data_ptr(), key_cache.data_ptr(), block_tables.data_ptr(), query_starts.data_ptr(),
            context_lens.data_ptr(), requests, width, num_blocks, block_size, kv_heads, dim, longest, pool,
            _lib.stream_of(bounds.device))
    _lib.check(status, "update_block_bounds")


def read_block_bounds(bounds, block_ids, *, validate=True):
    """Values of the bounds of blocks ``block_ids`` (int64 ``[n]``): ``(lower, upper)`` fp32 ``[n, kv_heads, head_dim]``.

    A block outside the pool gives zeros (refused with ``validate``).
    """
    num_blocks, kv_heads, dim = _check_bounds(bounds)
    _require(bounds.is_cuda and block_ids.device == bounds.device, "all inputs must be on the same CUDA device")
    _require(block_ids.dim() == 1 and block_ids.dtype == torch.int64 and block_ids.is_contiguous(),
             "block ids must be contiguous int64 [n]")
    count = block_ids.shape[0]
    if validate and count:
        _require(not bool(((block_ids < 0) | (block_ids >= num_blocks)).any()), "physical block id out of range")
    lower = torch.empty((count, kv_heads, dim), dtype=torch.float32, device=bounds.device)
    upper = torch.empty_like(lower)
    if count == 0:
        return lower, upper
    lib = _lib.load()
    with _lib.on_device(bounds.device):
        status = lib.minikv_block_bounds_read(bounds.data_ptr(), block_ids.data_ptr(), count, lower.data_ptr(),
                                              upper.data_ptr(), num_blocks, kv_heads, dim,
                                              _lib.stream_of(bounds.device))
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
    _require(query.is_cuda, "query must be CUDA")
    num_blocks, kv_heads, dim = _check_bounds(bounds)
    _require(query.dim() == 3 and query.shape[2] == dim and query.shape[1] % kv_heads == 0 and query.numel() > 0,
             "head dimension or GQA mismatch")
    code = _lib.dtype_code(query.dtype)
    device = query.device
    _require(bounds.device == block_tables.device == context_lens.device == device,
             "all inputs must be on the same CUDA device")
    _require(query.is_contiguous() and block_tables.is_contiguous() and context_lens.is_contiguous(),
             "inputs must be contiguous")
    _require(block_tables.dtype == torch.int64 and context_lens.dtype == torch.int64, "metadata must be int64")
    batch = query.shape[0]
    _require(block_tables.dim() == 2 and block_tables.shape[0] == batch and block_tables.shape[1] > 0,
             "invalid block table")
    _require(context_lens.dim() == 1 and context_lens.shape[0] == batch, "invalid context lengths")
    _require(type(block_size) is int and block_size > 0, "block size mismatch")
    width = block_tables.shape[1]
    _require(width * block_size <= 1048576, "maximum table capacity is 1M tokens")
    _require(max_blocks > 0 and sink_blocks >= 0 and recent_blocks >= 0 and sink_blocks + recent_blocks <= max_blocks,
             "max_blocks must be positive and hold the sink and recent blocks")
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
            workspace.data_ptr(), workspace.numel() * 4, batch, query.shape[1], kv_heads, dim, num_blocks, block_size,
            width, max_blocks, sink_blocks, recent_blocks, code, _lib.stream_of(device))
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
    _require(query.is_cuda, "query must be CUDA")
    _require(query.dim() == 3 and key_cache.dim() == 4 and value_cache.shape == key_cache.shape
             and key_cache.numel() > 0, "invalid query/cache shapes")
    _require(query.dtype in (torch.float16, torch.bfloat16), "FP16/BF16 required")
    _require(key_cache.dtype == query.dtype and value_cache.dtype == query.dtype, "cache dtype mismatch")
    num_blocks, bs, kv_heads, dim = key_cache.shape
    _require(type(block_size) is int and bs == block_size, "block size mismatch")
    _require(query.shape[2] == dim, "head dimension or GQA mismatch")
    _require(dim in INT4_HEAD_DIMS, "selected blocks: supported head_dim: 32,64,96,128,192,256")
    return _decode_pages("minikv_paged_decode_selected", "minikv_paged_decode_selected_workspace_bytes", query,
                         key_cache, value_cache, block_tables, context_lens, selected, block_size, num_blocks,
                         kv_heads, validate)
