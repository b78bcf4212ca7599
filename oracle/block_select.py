"""CPU oracle: block bounds and block selection.  Test infrastructure only (see oracle/__init__).

No counterpart in the reference; the contract is that of include/minikv.h.
"""

from __future__ import annotations

import math

import numpy as np
import torch

LARGEST = float(np.finfo(np.float32).max)
NONE = 2.0 ** -100


def record(keys):
    """One block's record (uint8 ``[2 D + 16]``) from its key rows ``[rows, D]``."""
    x = np.asarray(keys, dtype=np.float64)
    x = np.clip(np.where(np.isnan(x), 0.0, x), -LARGEST, LARGEST)
    high, low = x.max(0), x.min(0)
    top = max(np.abs(high).max(), np.abs(low).max())
    dim = x.shape[1]
    out = np.zeros(2 * dim + 16, dtype=np.uint8)
    if top < NONE:
        return out
    out[:dim] = np.ceil(127.0 * high / top).astype(np.int8).view(np.uint8)
    out[dim:2 * dim] = np.floor(127.0 * low / top).astype(np.int8).view(np.uint8)
    out[2 * dim:2 * dim + 4] = np.array([np.float32(top) / np.float32(127)], dtype=np.float32).view(np.uint8)
    return out


def update(bounds, keys, tables, starts, lens, block_size):
    """In place on a uint8 numpy ``bounds``; ``keys`` values ``[blocks, block_size, kv_heads, D]``."""
    blocks, width = keys.shape[0], tables.shape[1]
    for r, (start, length) in enumerate(zip(starts.tolist(), lens.tolist())):
        if start < 0 or start >= length or length > width * block_size:
            continue
        for j in range(start // block_size, -(-length // block_size)):
            page = int(tables[r, j])
            if not 0 <= page < blocks:
                continue
            rows = min(block_size, length - j * block_size)
            for h in range(keys.shape[2]):
                bounds[page, h] = record(keys[page, :rows, h].double().numpy())


def read(bounds, ids, dim):
    up = bounds[ids][..., :dim].view(np.int8).astype(np.float32)
    down = bounds[ids][..., dim:2 * dim].view(np.int8).astype(np.float32)
    scale = np.ascontiguousarray(bounds[ids][..., 2 * dim:2 * dim + 4]).view(np.float32)
    return torch.from_numpy(down * scale), torch.from_numpy(up * scale)


def query_codes(q):
    """Codes ``[2 D]`` of one kv head's query heads ``[group, D]``."""
    x = q.detach().float().cpu().numpy()
    x = np.clip(np.where(np.isnan(x), np.float32(0), x), np.float32(-LARGEST), np.float32(LARGEST))
    total = np.zeros(2 * x.shape[1], dtype=np.float32)
    for row in x:  # in the order of the heads
        total = total + np.concatenate((np.maximum(row, 0), np.minimum(row, 0))).astype(np.float32)
    top = np.abs(total).max()
    if top < NONE:
        return np.zeros(total.shape, dtype=np.int64)
    return np.clip(np.rint(total * (np.float32(127) / top)), -127, 127).astype(np.int64)


def select(query, bounds, tables, lens, block_size, max_blocks, sink=1, recent=1):
    """``selected [B, Hkv, max_blocks]`` int64."""
    batch, heads, dim = query.shape
    blocks, kv_heads, _ = bounds.shape
    width = tables.shape[1]
    out = torch.full((batch, kv_heads, max_blocks), -1, dtype=torch.int64)
    for b, length in enumerate(lens.tolist()):
        if length <= 0 or length > width * block_size:
            continue
        n = -(-length // block_size)
        group = heads // kv_heads
        for h in range(kv_heads):
            codes = query_codes(query[b, h * group:(h + 1) * group])
            scored = []
            for j in range(n):
                page = int(tables[b, j])
                if not 0 <= page < blocks:
                    continue
                rec = bounds[page, h]
                dot = int((rec[:2 * dim].view(np.int8).astype(np.int64) * codes).sum())
                scale = rec[2 * dim:2 * dim + 4].view(np.float32)[0]
                score = float(np.float32(dot) * scale)
                if j < sink or j >= n - recent:
                    score = math.inf
                scored.append((-score, j))
            chosen = sorted(j for _, j in sorted(scored)[:max_blocks])
            out[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int64)
    return out
