"""CPU oracle: the 4-bit KV pool.  Test infrastructure only (see oracle/__init__).

The reference has no 4-bit KV pool; its contract here is ours (include/minikv.h):
a page of one kv head holds ``block_size`` rows of ``head_dim / 2`` bytes, then
``block_size`` pairs of fp16 (step, base), padded to 16 bytes.  Rows are
quantised one by one; attention runs in 64 bits on the values.
"""

from __future__ import annotations

import math

import numpy as np
import torch

STEP_MIN = np.float32(2.0 ** -24)


def page_bytes(block_size, head_dim):
    return (block_size * (head_dim // 2 + 4) + 15) // 16 * 16


def quantize(x):
    """(codes, step fp16, base fp16) of the rows over the last axis of a float tensor."""
    x = x.detach().float().cpu().numpy().astype(np.float32)
    x = np.clip(np.where(np.isnan(x), np.float32(0), x), np.float32(-65504), np.float32(65504))
    low, high = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    base = low.astype(np.float16)
    step = np.maximum((high - low) / np.float32(15), STEP_MIN).astype(np.float16)
    # base + 15 step stays within 65504: else the largest fp16 with which it does (the step's least at least)
    wide = base.astype(np.float64)
    most = np.maximum((65504 - wide) / 15, float(STEP_MIN))
    down = most.astype(np.float16)
    down = np.where(down.astype(np.float64) > most, np.nextafter(down, np.float16(0)), down)
    over = (base.astype(np.float32) + np.float32(15) * step.astype(np.float32)) > np.float32(65504)
    step = np.where(over, down, step)
    d = x - base.astype(np.float32)
    codes = np.clip(np.rint(d / step.astype(np.float32)), 0, 15).astype(np.uint8)
    return codes, step[..., 0], base[..., 0]


def write_row(pool, block_size, slot, rows):
    """Put the quantised ``rows [kv_heads, head_dim]`` at ``slot`` of a uint8 numpy pool."""
    codes, step, base = quantize(rows)
    dim = codes.shape[-1]
    page, at = divmod(int(slot), block_size)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    pool[page, :, at * dim // 2:(at + 1) * dim // 2] = packed
    first = block_size * dim // 2 + at * 4
    pool[page, :, first:first + 4] = np.stack((step, base), -1).view(np.uint8)


def scatter(pool, block_size, slots, rows):
    """``write_kv_cache_slots_int4`` for one pool: slots outside the capacity are skipped."""
    capacity = pool.shape[0] * block_size
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < capacity:
            write_row(pool, block_size, slot, rows[t])


def values(pool, block_size, head_dim):
    """Values ``[blocks, block_size, kv_heads, head_dim]`` in 64 bits that a uint8 numpy pool stands for."""
    blocks, heads, _ = pool.shape
    rows = pool[..., :block_size * head_dim // 2].reshape(blocks, heads, block_size, head_dim // 2)
    codes = np.stack((rows & 15, rows >> 4), -1).reshape(blocks, heads, block_size, head_dim).astype(np.float64)
    first = block_size * head_dim // 2
    pairs = np.ascontiguousarray(pool[..., first:first + 4 * block_size]).view(np.float16)
    pairs = pairs.reshape(blocks, heads, block_size, 2).astype(np.float64)
    out = pairs[..., 1:] + np.maximum(pairs[..., :1], float(STEP_MIN)) * codes
    return torch.from_numpy(out.transpose(0, 2, 1, 3).copy())


def attend(q, keys, vals, keep):
    """Softmax attention in 64 bits of ``q [n, D]`` over ``keys/vals [t, D]``, ``keep [n, t]``; no key kept: zeros."""
    score = (q.double() @ keys.T) / math.sqrt(q.shape[-1])
    score = score.masked_fill(~keep, -math.inf)
    top = score.amax(-1, keepdim=True) if score.shape[1] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64)
    weight = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = weight.sum(-1, keepdim=True)
    safe = torch.where(keep.any(0)[:, None], vals, torch.zeros_like(vals))  # a row that no query keeps may hold anything
    out = (weight @ safe) / torch.where(total == 0, torch.ones_like(total), total)
    return out


def paged_decode(query, keys, vals, tables, lens, block_size, selected=None):
    """64-bit decode attention over value pools ``[blocks, block_size, kv_heads, D]`` with the kernels' guards."""
    batch, heads, dim = query.shape
    blocks, _, kv_heads, _ = keys.shape
    width, group = tables.shape[1], heads // kv_heads
    out = torch.zeros(query.shape, dtype=torch.float64)
    for b, length in enumerate(lens.tolist()):
        if length <= 0 or length > width * block_size:
            continue
        for h in range(kv_heads):
            have = -(-length // block_size)
            listed = torch.arange(have) if selected is None else selected[b, h, :have]
            listed = listed[(listed >= 0) & (listed < width)]
            pos = (listed[:, None] * block_size + torch.arange(block_size)).flatten()
            page = tables[b, listed].repeat_interleave(block_size)
            ok = (pos < length) & (page >= 0) & (page < blocks)
            page, off = page[ok], (pos % block_size)[ok]
            q = query[b, h * group:(h + 1) * group]
            out[b, h * group:(h + 1) * group] = attend(q, keys[page, off, h], vals[page, off, h],
                                                       torch.ones(group, len(page), dtype=torch.bool))
    return out


def paged_prefill(q, keys, vals, cu, starts, tables, lens, block_size):
    """64-bit ragged causal prefill over value pools, with the kernels' guards."""
    tokens, heads, dim = q.shape
    blocks, _, kv_heads, _ = keys.shape
    group, width = heads // kv_heads, tables.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    for r, (start, length) in enumerate(zip(starts.tolist(), lens.tolist())):
        lo, hi = int(cu[r]), int(cu[r + 1])
        reach = min(length, width * block_size)
        if hi <= lo or reach <= 0:
            continue
        pos = torch.arange(reach)
        page = tables[r, pos // block_size]
        ok = (page >= 0) & (page < blocks)
        safe = torch.where(ok, page, torch.zeros_like(page))
        seen = start + torch.arange(hi - lo)
        keep = (pos <= seen[:, None]) & ok & ((seen >= 0) & (seen < reach))[:, None]
        for h in range(heads):
            k, v = (x[safe, pos % block_size, h // group] for x in (keys, vals))
            out[lo:hi, h] = attend(q[lo:hi, h], k, v, keep)
    return out
