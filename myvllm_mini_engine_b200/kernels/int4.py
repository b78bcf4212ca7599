"""4-bit KV pool: quantising writes, reading back, decode attention and ragged prefill.

The reference has no 4-bit KV pool; these operators extend its API in its own
style.  The writes mirror ``write_kv_cache_slots`` and ``write_kv_cache_batch``
(``mini_engine/kernels/data.py:67-130``), the decode ``paged_attention``
(``kernels/paged.py:8-22``) and the prefill ``paged_prefill_attention``
(``kernels/prefill.py:61-131``).

A pool is a contiguous uint8 tensor ``[num_blocks, kv_heads, page_bytes]`` with
``page_bytes = int4_page_bytes(block_size, head_dim)``.  The page of one kv head
holds ``block_size`` rows of ``head_dim / 2`` bytes (element 2i in the low half
of byte i), then ``block_size`` pairs of fp16 (step, base), padded to 16 bytes.
Element ``x`` of a row is stored as ``code = round((x - base) / step)`` in 0..15
with ``base = fp16(min)`` and ``step = fp16(max(2^-24, (max - min) / 15))`` of its
row (one token, one kv head, K or V by itself), and read as ``base + step * code``.
NaN counts as 0 and magnitudes saturate at 65504; the step is rounded down where
``base + 15 * step`` would pass that.  At head_dim 128 that is 4.25
bits an element: a decode step streams 68 bytes where a 16-bit pool has 256.

The decode's scratch memory is kept per stream for eager calls; a captured call
has its own.
"""

from __future__ import annotations

import threading

import torch

from .. import _lib
from .data import _backend
from .paged import _require, check_backend

INT4_HEAD_DIMS = (32, 64, 96, 128, 192, 256)
_HEAD_DIM_MESSAGE = "a 4-bit KV pool needs head_dim 32, 64, 96, 128, 192 or 256"
_QUERY_DTYPES = (torch.float16, torch.bfloat16)


def int4_page_bytes(block_size, head_dim):
    """Bytes of one kv head's part of a page of a 4-bit pool."""
    if type(block_size) is not int or block_size <= 0:
        raise ValueError("block_size must be a positive int")
    if head_dim not in INT4_HEAD_DIMS:
        raise ValueError(_HEAD_DIM_MESSAGE)
    return (block_size * (head_dim // 2 + 4) + 15) // 16 * 16


def _check_pools(key_cache, value_cache, block_size, head_dim, fail=ValueError):
    """Shape and dtype checks shared by the operators over a pool; the pool's ``(num_blocks, kv_heads)``."""
    shape = key_cache.shape
    if (len(shape) != 3 or value_cache.shape != shape or key_cache.dtype is not torch.uint8
            or value_cache.dtype is not torch.uint8 or not key_cache.is_contiguous()
            or not value_cache.is_contiguous() or 0 in shape):
        raise fail("4-bit KV caches must be contiguous uint8 [pages, kv_heads, page_bytes]")
    if head_dim not in INT4_HEAD_DIMS:
        raise fail(_HEAD_DIM_MESSAGE)
    if type(block_size) is not int or block_size <= 0:
        raise fail("block size mismatch")
    if shape[2] != (block_size * (head_dim // 2 + 4) + 15) // 16 * 16:
        raise fail("block size mismatch: the pages are not int4_page_bytes(block_size, head_dim) long")
    return shape[0], shape[1]


def _device_of(tensors, fail, message):
    """The device that all of the tensors are on."""
    index = tensors[0].get_device()
    for tensor in tensors:
        if tensor.get_device() != index:
            raise fail(message)
    return tensors[0].device


def _source_rows(tensor):
    """(tensor, token stride) of a ``[tokens, kv_heads, head_dim]`` source whose heads are contiguous (copied if not)."""
    _, heads, dim = tensor.shape
    if tensor.is_contiguous():
        return tensor, heads * dim
    if tensor.stride(2) == 1 and (heads == 1 or tensor.stride(1) == dim) and tensor.stride(0) >= heads * dim:
        return tensor, tensor.stride(0)
    return tensor.contiguous(), heads * dim


def _extent(tensor):
    """(first byte, byte behind the last) of a tensor's elements."""
    last = sum((n - 1) * stride for n, stride in zip(tensor.shape, tensor.stride()))
    start = tensor.data_ptr()
    return start, start + (last + 1) * tensor.element_size() if tensor.numel() else start


def _overlaps(caches, sources):
    """Whether a cache shares bytes with the other one or with a source (views of one storage need not)."""
    held = [_extent(cache) for cache in caches]
    ranges = [*held[1:], *map(_extent, sources)]
    return any(a < d and c < b for i, (a, b) in enumerate(held) for c, d in ranges[i:])


def write_kv_cache_slots_int4(key_cache, value_cache, slot_mapping, key, value, block_size, *, backend="cuda",
                              validate=True):
    """Quantise packed K/V rows into 4-bit pools at ``slot_mapping`` (slots outside the capacity are skipped).

    ``key``/``value`` ``[tokens, kv_heads, head_dim]`` fp32/fp16/bf16 (token-strided
    views are read in place).  ``validate`` adds the host-synchronising slot checks
    of ``write_kv_cache_slots`` (data.py:109-119).
    """
    _backend(backend)
    shape = key.shape
    if len(shape) != 3 or value.shape != shape:
        raise ValueError("packed key/value must be [tokens, kv_heads, head_dim] matching the cache")
    tokens, heads, dim = shape
    num_blocks, kv_heads = _check_pools(key_cache, value_cache, block_size, dim)
    if heads != kv_heads:
        raise ValueError("packed key/value must be [tokens, kv_heads, head_dim] matching the cache")
    code = _lib.DTYPE_CODES.get(key.dtype)
    if code is None or value.dtype is not key.dtype:
        raise ValueError("packed KV requires FP32/FP16/BF16")
    if (slot_mapping.shape != (tokens,) or slot_mapping.dtype is not torch.int64
            or not slot_mapping.is_contiguous()):
        raise ValueError("slot_mapping must be contiguous int64 [tokens]")
    device = _device_of((key_cache, value_cache, slot_mapping, key, value), ValueError,
                        "packed KV tensors and slots must share the cache device")
    if validate:
        slots = slot_mapping.tolist()
        if any(slot < 0 or slot >= num_blocks * block_size for slot in slots):
            raise ValueError("KV slot is outside cache capacity")
        if len(set(slots)) != len(slots):
            raise ValueError("duplicate KV slots would race during scatter")
        if _overlaps((key_cache, value_cache), (key, value, slot_mapping)):
            raise ValueError("KV destinations and source tensors must not overlap")
    if device.type != "cuda":
        raise ValueError("CUDA packed KV writes require CUDA tensors")
    if tokens == 0:
        return
    key, key_stride = _source_rows(key)
    value, value_stride = _source_rows(value)
    lib = _lib.load()
    with _lib.on_device(device):
        status = lib.minikv_kv_scatter_slots_int4(
            key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.data_ptr(), key.data_ptr(), value.data_ptr(),
            tokens, num_blocks, block_size, kv_heads, dim, key_stride, value_stride, code, _lib.stream_of(device))
    if status:
        _lib.check(status, "write_kv_cache_slots_int4")


def write_kv_cache_batch_int4(key_cache, value_cache, block_tables, token_offsets, key, value, block_size, *,
                              backend="cuda", validate=True):
    """Quantise one new row per request at position ``token_offsets[b]`` of its page table (the decode append).

    ``key``/``value`` ``[batch, kv_heads, head_dim]``; rows whose position or page is
    out of range are skipped.  ``validate`` adds the host-synchronising checks of
    ``write_kv_cache_batch`` (data.py:67-81).
    """
    _backend(backend)
    if key.ndim != 3 or key.shape != value.shape:
        raise ValueError("batch key/value must be [batch, kv_heads, head_dim]")
    num_blocks, kv_heads = _check_pools(key_cache, value_cache, block_size, key.shape[2])
    if key.shape[1] != kv_heads:
        raise ValueError("batch K/V shape mismatch")
    if key.dtype not in _lib.DTYPE_CODES or value.dtype != key.dtype:
        raise ValueError("packed KV requires FP32/FP16/BF16")
    batch = key.shape[0]
    if (block_tables.ndim != 2 or token_offsets.ndim != 1 or block_tables.shape[0] != batch
            or token_offsets.shape[0] != batch or block_tables.dtype != torch.int64
            or token_offsets.dtype != torch.int64 or not block_tables.is_contiguous()
            or not token_offsets.is_contiguous()):
        raise ValueError("batch metadata must be contiguous int64 [batch, pages] and [batch]")
    device = _device_of((key_cache, value_cache, block_tables, token_offsets, key, value), ValueError,
                        "batch KV tensors must share the cache device")
    width = block_tables.shape[1]
    if validate and batch:
        if bool(((token_offsets < 0) | (token_offsets >= width * block_size)).any()):
            raise ValueError("batch KV offset out of range")
        pages = block_tables.gather(1, (token_offsets // block_size).unsqueeze(1)).squeeze(1)
        if bool(((pages < 0) | (pages >= num_blocks)).any()):
            raise ValueError("physical block id out of range")
        slots = pages * block_size + token_offsets % block_size
        if slots.unique().numel() != batch:
            raise ValueError("duplicate KV slots would race during scatter")
        if _overlaps((key_cache, value_cache), (key, value, block_tables, token_offsets)):
            raise ValueError("KV destinations and source tensors must not overlap")
    if device.type != "cuda":
        raise ValueError("CUDA batch KV writes require CUDA tensors")
    if batch == 0:
        return
    key, key_stride = _source_rows(key)
    value, value_stride = _source_rows(value)
    lib = _lib.load()
    with _lib.on_device(device):
        status = lib.minikv_kv_append_batch_int4(
            key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(), token_offsets.data_ptr(),
            key.data_ptr(), value.data_ptr(), batch, width, num_blocks, block_size, kv_heads, key.shape[2], key_stride,
            value_stride, _lib.DTYPE_CODES[key.dtype], _lib.stream_of(device))
    if status:
        _lib.check(status, "write_kv_cache_batch_int4")


def read_kv_cache_slots_int4(key_cache, value_cache, slot_mapping, block_size, head_dim, *, dtype=torch.float32,
                             backend="cuda", validate=True):
    """The values at ``slot_mapping``: ``(key, value)`` ``[tokens, kv_heads, head_dim]`` of ``dtype``.

    ``base + step * code`` in fp32, rounded once; a slot outside the capacity gives
    zeros (refused with ``validate``).
    """
    _backend(backend)
    num_blocks, kv_heads = _check_pools(key_cache, value_cache, block_size, head_dim)
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None:
        raise ValueError("packed KV requires FP32/FP16/BF16")
    if slot_mapping.ndim != 1 or slot_mapping.dtype is not torch.int64 or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 [tokens]")
    device = _device_of((key_cache, value_cache, slot_mapping), ValueError,
                        "packed KV tensors and slots must share the cache device")
    if validate and slot_mapping.numel():
        if bool(((slot_mapping < 0) | (slot_mapping >= num_blocks * block_size)).any()):
            raise ValueError("KV slot is outside cache capacity")
    if device.type != "cuda":
        raise ValueError("CUDA packed KV reads require CUDA tensors")
    tokens = slot_mapping.shape[0]
    key = torch.empty((tokens, kv_heads, head_dim), dtype=dtype, device=device)
    value = torch.empty_like(key)
    if tokens == 0:
        return key, value
    lib = _lib.load()
    with _lib.on_device(device):
        status = lib.minikv_kv_gather_slots_int4(
            key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.data_ptr(), key.data_ptr(), value.data_ptr(),
            tokens, num_blocks, block_size, kv_heads, head_dim, code, _lib.stream_of(device))
    if status:
        _lib.check(status, "read_kv_cache_slots_int4")
    return key, value


# ------------------------------------------------------------------ decode

_NEEDS: dict = {}
_SCRATCH: dict = {}
_OLD_SCRATCH: list = []
_CAPTURED: dict = {}
_CAPTURED_TICKETS = 1 << 22
_CAPTURED_LOCK = threading.Lock()


def _captured_tickets(device, count):
    """Counters of one captured call: zero, as every launch of it leaves them, and never another call's.

    They come from a buffer that the first eager call on the device zeroed, so that
    a replay need not; once that is used up (or before an eager call) the graph
    holds counters that it zeroes itself, about 2 us a call.
    """
    held = _CAPTURED.get(device.index)
    with _CAPTURED_LOCK:
        first = -1
        if held is not None and held[1] + count <= held[0].numel():
            first, held[1] = held[1], held[1] + count
    if first < 0:
        return torch.zeros(count, dtype=torch.int32, device=device)
    return held[0][first:first + count]


def _scratch(device, stream, tickets, need):
    """(ticket counters, workspace) of a page decode.

    Every launch leaves the counters zero, whatever its shape, and the workspace
    may hold anything, so the eager calls on one stream, which follow one another,
    share them.  A captured call may run beside other work of its stream: it gets
    counters of its own, and a workspace from the graph's memory.
    """
    if torch.cuda.is_current_stream_capturing():
        return _captured_tickets(device, tickets), torch.empty(need, dtype=torch.uint8, device=device)
    key = (device.index, stream)
    held = _SCRATCH.get(key)
    if held is None or held[0].numel() < tickets or held[1].numel() < need:
        if device.index not in _CAPTURED:
            zeros = torch.zeros(_CAPTURED_TICKETS, dtype=torch.int32, device=device)
            torch.cuda.current_stream(device).synchronize()  # once: a replay may run on any stream
            _CAPTURED[device.index] = [zeros, 0]
        if held is not None:
            _OLD_SCRATCH.append(held)  # a launch in flight may still use it
            tickets, need = max(tickets, 2 * held[0].numel()), max(need, 2 * held[1].numel())
        held = _SCRATCH[key] = (torch.zeros(max(tickets, 4096), dtype=torch.int32, device=device),
                                torch.empty(need, dtype=torch.uint8, device=device))
    return held


def _check_selected(selected, block_tables, context_lens, kv_heads, block_size, validate):
    if selected.dtype is not torch.int64 or not selected.is_contiguous():
        raise RuntimeError("selected must be contiguous int64")
    if selected.get_device() != block_tables.get_device():
        raise RuntimeError("all inputs must be on the same CUDA device")
    shape = selected.shape
    if len(shape) != 3 or shape[0] != block_tables.shape[0] or shape[1] != kv_heads or shape[2] <= 0:
        raise RuntimeError("selected must be [batch, kv_heads, blocks]")
    if validate:
        blocks = ((context_lens + block_size - 1) // block_size)[:, None, None]
        _require(not bool(((selected < -1) | (selected >= blocks)).any()), "selected block out of range")
        first, second = selected[..., :-1], selected[..., 1:]
        _require(not bool(((second <= first) & (second != -1)).any()) and
                 not bool(((first == -1) & (second != -1)).any()),
                 "selected blocks must be ascending, with -1 only behind the last")


def _decode_pages(entry, sizer, query, key_cache, value_cache, block_tables, context_lens, selected, block_size,
                  num_blocks, kv_heads, validate):
    """Metadata checks and launch shared by the decodes over page lists."""
    if not (query.is_contiguous() and key_cache.is_contiguous() and value_cache.is_contiguous()
            and block_tables.is_contiguous() and context_lens.is_contiguous()):
        raise RuntimeError("inputs must be contiguous")
    device = _device_of((query, key_cache, value_cache, block_tables, context_lens), RuntimeError,
                        "all inputs must be on the same CUDA device")
    if block_tables.dtype is not torch.int64 or context_lens.dtype is not torch.int64:
        raise RuntimeError("metadata must be int64")
    batch, heads, dim = query.shape
    if batch <= 0 or heads <= 0:
        raise RuntimeError("empty batch/heads/cache")
    if heads % kv_heads:
        raise RuntimeError("head dimension or GQA mismatch")
    table = block_tables.shape
    if len(table) != 2 or table[0] != batch or table[1] <= 0:
        raise RuntimeError("invalid block table")
    if context_lens.shape != (batch,):
        raise RuntimeError("invalid context lengths")
    width = table[1]
    if width * block_size > 1048576:
        raise RuntimeError("maximum table capacity is 1M tokens")
    if validate:
        _require(not bool(((context_lens <= 0) | (context_lens > width * block_size)).any()),
                 "invalid context length")
        positions = torch.arange(width, device=device, dtype=torch.int64) * block_size
        active = positions.unsqueeze(0) < context_lens.unsqueeze(1)
        _require(not bool((((block_tables < 0) | (block_tables >= num_blocks)) & active).any()),
                 "physical block id out of range")
    take, listed = 0, None
    if selected is not None:
        _check_selected(selected, block_tables, context_lens, kv_heads, block_size, validate)
        take, listed = selected.shape[2], selected.data_ptr()
    lib = _lib.load()
    code = _lib.DTYPE_CODES[query.dtype]
    with _lib.on_device(device):
        key = (sizer, device.index, batch, heads, kv_heads, dim, code)
        need = _NEEDS.get(key)
        if need is None:
            need = getattr(lib, sizer)(batch, heads, kv_heads, dim, num_blocks, block_size, width, code)
            if need < 0:
                _lib.check(_lib.EINVAL, entry)
            _NEEDS[key] = need
        stream = _lib.stream_of(device)
        tickets, workspace = _scratch(device, stream, batch * kv_heads * ((heads // kv_heads + 7) // 8), need)
        out = torch.empty_like(query)
        status = getattr(lib, entry)(
            query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
            context_lens.data_ptr(), listed, out.data_ptr(), tickets.data_ptr(), workspace.data_ptr(), need, batch,
            heads, kv_heads, dim, num_blocks, block_size, width, take, code, stream)
    if status:
        _lib.check(status, entry)
    return out


def paged_attention_int4(query, key_cache, value_cache, block_tables, context_lens, block_size, *, selected=None,
                         backend="cuda", validate=True):
    """Decode attention over 4-bit pools: ``softmax(q . K^T / sqrt(D)) V``.

    Arguments and guards as :func:`paged_attention` (``query [B, Hq, D]`` fp16 or
    bf16, ``block_tables [B, W]`` and ``context_lens [B]`` int64).  ``selected``
    (``[B, Hkv, K]`` int64, from :func:`select_blocks`) restricts each kv head to
    the listed logical blocks, ascending with -1 behind the last; the first
    ``min(K, blocks of the request)`` entries are read.  The codes enter the
    products exactly; Q is rounded to fp16 after a scaling by a power of two that
    fits its range.  Returns ``[B, Hq, D]`` in the query dtype.
    """
    check_backend(backend)
    if not query.is_cuda:
        raise RuntimeError("query must be CUDA")
    if query.dim() != 3:
        raise RuntimeError("invalid query/cache shapes")
    if query.dtype not in _QUERY_DTYPES:
        raise RuntimeError("a 4-bit KV pool needs an FP16/BF16 query")
    num_blocks, kv_heads = _check_pools(key_cache, value_cache, block_size, query.shape[2], RuntimeError)
    return _decode_pages("minikv_paged_decode_int4", "minikv_paged_decode_int4_workspace_bytes", query, key_cache,
                         value_cache, block_tables, context_lens, selected, block_size, num_blocks, kv_heads, validate)


def paged_prefill_attention_int4(q, key_cache, value_cache, cu_seqlens_q, query_starts, block_tables, context_lens,
                                 block_size, *, backend="cuda", validate=True, max_query_len=None):
    """Ragged causal prefill over 4-bit pools: :func:`paged_prefill_attention` with K/V read as ``base + step * code``.

    ``q`` is fp16 or bf16 ``[tokens, q_heads, head_dim]`` with up to 64 query heads
    a kv head.  Metadata, checks and messages as ``paged_prefill_attention``
    (``mini_engine/kernels/prefill.py:61-131``).  Packed tokens of no request, or
    past their context, get zeros.  The codes enter the products exactly.  A
    request's rows do not depend on the batch around it or on the table's width,
    and the call takes no workspace.
    """
    if backend != "cuda":
        raise ValueError("paged prefill backend must be cuda (this package has no torch/CPU path)")
    if q.ndim != 3 or q.shape[1] <= 0:
        raise ValueError("paged prefill Q must be [tokens, heads, head_dim] with divisible GQA heads")
    if q.dtype not in _QUERY_DTYPES:
        raise ValueError("a 4-bit KV pool needs an FP16/BF16 query")
    num_blocks, kv_heads = _check_pools(key_cache, value_cache, block_size, q.shape[2])
    if q.shape[1] % kv_heads:
        raise ValueError("paged prefill Q must be [tokens, heads, head_dim] with divisible GQA heads")
    metadata = (cu_seqlens_q, query_starts, block_tables, context_lens)
    requests = block_tables.shape[0]
    if (cu_seqlens_q.ndim != 1 or query_starts.ndim != 1 or context_lens.ndim != 1 or block_tables.ndim != 2
            or query_starts.shape[0] != requests or context_lens.shape[0] != requests
            or cu_seqlens_q.shape[0] != requests + 1):
        raise ValueError("paged prefill metadata shapes do not match request count")
    if any(t.dtype != torch.int64 or not t.is_contiguous() for t in metadata):
        raise ValueError("paged prefill metadata must be contiguous int64 tensors")
    if any(t.device != q.device for t in (key_cache, value_cache, *metadata)):
        raise ValueError("paged prefill tensors must share device")
    width = block_tables.shape[1]
    if validate:
        offsets, starts, tables, lengths = (t.tolist() for t in metadata)
        if offsets[0] != 0 or offsets[-1] != q.shape[0] or any(b < a for a, b in zip(offsets, offsets[1:])):
            raise ValueError("query offsets must be monotone and cover all packed queries")
        for index, (start, length, table) in enumerate(zip(starts, lengths, tables)):
            count = offsets[index + 1] - offsets[index]
            if start < 0 or length != start + count or length > len(table) * block_size:
                raise ValueError("query start/context length exceeds block table capacity or query range")
            used = (length + block_size - 1) // block_size
            if any(page < 0 or page >= num_blocks for page in table[:used]):
                raise ValueError("active block table contains an invalid physical page")
    if q.device.type != "cuda":
        raise ValueError("CUDA paged prefill requires CUDA tensors")
    q = q.contiguous()
    output = torch.empty_like(q)
    tokens = q.shape[0]
    if tokens == 0:
        return output
    bound = tokens if max_query_len is None else int(max_query_len)
    lib = _lib.load()
    _, heads, dim = q.shape
    code, device = _lib.DTYPE_CODES[q.dtype], q.device
    with _lib.on_device(device):
        status = lib.minikv_paged_prefill_int4(
            q.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), cu_seqlens_q.data_ptr(),
            query_starts.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), output.data_ptr(), None, 0,
            tokens, requests, heads, kv_heads, dim, num_blocks, block_size, width, bound, code, _lib.stream_of(device))
    if status:
        _lib.check(status, "paged_prefill_attention_int4")
    return output
