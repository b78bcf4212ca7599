"""The Qwen3 decode step over a 4-bit pool and over selected blocks, and the pools' own methods.

Compared with the same step with its attention in plain PyTorch over the rows that it
reads back from its own copy of the pool (the writes, the bounds and the
selection have tests of their own against the 64-bit oracle).  Both steps round
the attention's result to bf16, so from the second layer on they differ by that
rounding, and a 4-bit code of the newest row may come out one step apart.

Bars: logits within the decode step's tolerance (tests/test_gpu_decode_step.py);
layer 0's appended rows and bounds, which both steps compute with the same
kernels from the same inputs, bit for bit; nothing else in the pools changed; a
captured step replays to the eager step's logits.
"""

import numpy as np
import pytest
import torch

import cases
from myvllm_mini_engine_b200 import _lib
from myvllm_mini_engine_b200.cache import INT4KVCachePool, PagedKVPool
from myvllm_mini_engine_b200.engine.qwen3 import Qwen3DecodeStep
from myvllm_mini_engine_b200.kernels import write_kv_cache_batch
from oracle import block_select, int4_kv
from test_gpu_decode_step import ATOL, RTOL, model_case

pytestmark = pytest.mark.gpu


class PlainAttention(Qwen3DecodeStep):
    """The step with the attention of every layer in plain PyTorch (selection by the oracle)."""

    def _attend(self, index, q, block_tables, positions):
        pool, bs = self.pool, self.pool.shape.block_size
        rows = (q.shape[0], self.config.num_key_value_heads, self.config.head_dim)
        stage = self._stage_k.view(rows), self._stage_v.view(rows)
        if self.int4:
            pool.write_batch(index, block_tables, positions, *stage)
        else:
            write_kv_cache_batch(pool.key[index], pool.value[index], block_tables, positions, *stage, bs,
                                 validate=False)
        selected = None
        if self.selected_blocks is not None:
            pool.update_bounds(index, block_tables, positions, positions + 1)
            selected = block_select.select(q.cpu(), pool.bounds[index].cpu().numpy(), block_tables.cpu(),
                                           (positions + 1).cpu(), bs, self.selected_blocks)
        out = torch.empty_like(q)
        group = q.shape[1] // rows[1]
        for b, length in enumerate((positions + 1).tolist()):
            ids = block_tables[b, :-(-length // bs)]
            if self.int4:
                keys, vals = pool.dequantized(index, ids, length)
            else:
                keys, vals = (p[index, ids].flatten(0, 1)[:length].float() for p in (pool.key, pool.value))
            keys, vals = (x.transpose(0, 1).repeat_interleave(group, 0) for x in (keys, vals))
            score = torch.einsum("hd,htd->ht", q[b].float(), keys) * q.shape[2] ** -0.5
            if selected is not None:
                block = torch.arange(length) // bs
                keep = (selected[b][:, :, None] == block).any(1).to(q.device).repeat_interleave(group, 0)
                score.masked_fill_(~keep, -torch.inf)
            out[b] = torch.einsum("ht,htd->hd", score.softmax(-1), vals).to(q.dtype)
        return out


def bounded_pool(pool, kind, tables, positions):
    """A pool of ``kind`` with bounds, holding ``pool``'s history."""
    s = pool.shape
    if kind == "int4":
        copy = INT4KVCachePool(s.num_layers, s.num_blocks, s.block_size, s.num_kv_heads, s.head_dim, block_bounds=True)
    else:
        copy = PagedKVPool(s.num_layers, s.num_blocks, s.block_size, s.num_kv_heads, s.head_dim, block_bounds=True)
    slots = torch.arange(s.num_blocks * s.block_size, device="cuda")
    rows = (-1, s.num_kv_heads, s.head_dim)
    for layer in range(s.num_layers):
        if kind == "int4":
            copy.write_slots(layer, slots, pool.key[layer].view(rows), pool.value[layer].view(rows), validate=False)
        else:
            copy.key[layer].copy_(pool.key[layer])
            copy.value[layer].copy_(pool.value[layer])
        copy.update_bounds(layer, tables, torch.zeros_like(positions), positions, validate=False)
    return copy


@pytest.mark.parametrize("kind,layers,selected,fused", [
    ("int4", 4, None, True), ("int4", 4, None, False),
    # one layer: both steps select by the same query, so by the same blocks
    ("int4", 1, 5, True), ("bf16", 1, 5, True), ("bf16", 1, 9, False)])
def test_step_matches_plain_attention_over_greedy_steps(cuda_device, kind, layers, selected, fused):
    contexts = (1, 15, 16, 17, 255, 256, 700, 1031)
    cfg, weights, pool, tables, ids, positions = model_case(contexts, seed=61, layers=layers)
    mine, theirs = (bounded_pool(pool, kind, tables, positions) for _ in range(2))
    step = Qwen3DecodeStep(cfg, weights, mine, fused_projections=fused, selected_blocks=selected)
    plain = PlainAttention(cfg, weights, theirs, fused_projections=fused, selected_blocks=selected)
    before = mine.key.clone(), mine.value.clone()
    bs = mine.shape.block_size
    pages = torch.cat([tables.gather(1, ((positions + i) // bs)[:, None]).flatten() for i in range(3)])
    for _ in range(3):
        logits, expected = (s.forward_decode_batch(ids, tables, positions) for s in (step, plain))
        torch.testing.assert_close(logits.float(), expected.float(), atol=ATOL, rtol=RTOL)
        ids, positions = expected.argmax(-1), positions + 1
    assert torch.equal(mine.key[0], theirs.key[0]) and torch.equal(mine.value[0], theirs.value[0])
    assert torch.equal(mine.bounds[0], theirs.bounds[0])
    for now, old in zip((mine.key, mine.value), before):
        now = now.clone()
        assert not torch.equal(now, old)
        now[:, pages] = old[:, pages]
        assert torch.equal(now, old)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("kind,selected", [("int4", None), ("int4", 6), ("bf16", 6)])
def test_step_replays_in_a_cuda_graph(cuda_device, kind, selected):
    cfg, weights, pool, tables, ids, positions = model_case((5, 64, 300, 999), seed=67, layers=4)
    held = bounded_pool(pool, kind, tables, positions)
    step = Qwen3DecodeStep(cfg, weights, held, selected_blocks=selected)
    start = held.storage.clone(), held.bounds.clone()

    def restore():
        held.storage.copy_(start[0])
        held.bounds.copy_(start[1])

    eager = step.forward_decode_batch(ids, tables, positions)
    restore()
    capture = torch.cuda.Stream()
    capture.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(capture):
        step.forward_decode_batch(ids, tables, positions)
    capture.synchronize()
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=capture):
        out = step.forward_decode_batch(ids, tables, positions)
    for _ in range(2):
        restore()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    assert _lib.device_status() == 0


def test_int4_pool_range_write_attend_prefill_read_and_copy_on_write(cuda_device):
    gen = torch.Generator().manual_seed(71)
    layers, blocks, bs, heads, dim = 2, 24, 16, 4, 64
    pool = INT4KVCachePool(layers, blocks, bs, heads, dim, block_bounds=True)
    assert pool.memory_bytes == 2 * layers * blocks * heads * bs * (dim // 2 + 4)
    ids, offset, tokens = [5, 17, 2, 9], 3, 50
    key, value = (torch.randn(tokens, heads, dim, generator=gen).to(torch.bfloat16) for _ in range(2))
    pool.write_range(1, ids, offset, key.cuda(), value.cuda())
    positions = torch.arange(tokens) + offset
    slots = torch.tensor(ids)[positions // bs] * bs + positions % bs
    plain = [np.zeros((blocks, heads, int4_kv.page_bytes(bs, dim)), dtype=np.uint8) for _ in range(2)]
    for bytes_, rows in zip(plain, (key, value)):
        int4_kv.scatter(bytes_, bs, slots, rows)
    assert np.array_equal(pool.key[1].cpu().numpy(), plain[0]) and np.array_equal(pool.value[1].cpu().numpy(), plain[1])
    assert not pool.storage[:, 0].any()
    keys, vals = (int4_kv.values(bytes_, bs, dim) for bytes_ in plain)
    table = torch.tensor([ids, ids])
    got = pool.dequantized(1, ids, offset + tokens)
    for mine, theirs in zip(got, (keys, vals)):
        assert torch.equal(mine[offset:].double().cpu(), theirs[slots // bs, slots % bs])
    lens = torch.tensor([offset + tokens, 20])
    query = torch.randn(2, 8, dim, generator=gen).to(torch.bfloat16)
    out = pool.attend(1, query.cuda(), table.cuda(), lens.cuda())
    expected = int4_kv.paged_decode(query, keys, vals, table, lens, bs)
    # the result's half step, and P' in one 16-bit term (2^-11)
    assert float((out.double().cpu() - expected).norm()) <= (2.0 ** -8 + 2.0 ** -11) * float(expected.norm())
    cu, starts = torch.tensor([0, 2, 3], dtype=torch.int64), lens - torch.tensor([2, 1])
    rows = torch.cat((query, query[:1]))
    out = pool.prefill(1, rows.cuda(), cu.cuda(), starts.cuda(), table.cuda(), lens.cuda())
    expected = int4_kv.paged_prefill(rows, keys, vals, cu, starts, table, lens, bs)
    assert float((out.double().cpu() - expected).norm()) <= (2.0 ** -8 + 2.0 ** -11) * float(expected.norm())
    pool.update_bounds(1, table[:1].cuda(), torch.zeros(1, dtype=torch.int64).cuda(), lens[:1].cuda())
    pool.copy_blocks([(17, 20)])
    torch.cuda.synchronize()
    for tensor in (pool.key, pool.value, pool.bounds):
        assert torch.equal(tensor[:, 20], tensor[:, 17]) and tensor[1, 17].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_paged_pool_with_bounds_selects_and_copies(cuda_device, dtype):
    gen = torch.Generator().manual_seed(73)
    blocks, bs, heads, dim = 12, 16, 2, 64
    pool = PagedKVPool(1, blocks, bs, heads, dim, dtype=dtype, block_bounds=True)
    ids = [7, 1, 9, 4, 3]
    rows = torch.randn(2, 70, heads, dim, generator=gen).to(dtype).cuda()
    pool.write_range(0, ids, 0, rows[0], rows[1])
    table, lens = torch.tensor([ids]), torch.tensor([70])
    pool.update_bounds(0, table.cuda(), torch.zeros(1, dtype=torch.int64).cuda(), lens.cuda())
    query = torch.randn(1, 4, dim, generator=gen).to(dtype)
    chosen = pool.select_blocks(0, query.cuda(), table.cuda(), lens.cuda(), 3)
    want = np.zeros((blocks, heads, 2 * dim + 16), dtype=np.uint8)
    block_select.update(want, pool.key[0].double().cpu(), table, torch.zeros(1, dtype=torch.int64), lens, bs)
    assert np.array_equal(pool.bounds[0].cpu().numpy(), want)
    assert torch.equal(chosen.cpu(), block_select.select(query, want, table, lens, bs, 3))
    pool.copy_blocks([(9, 0), (4, 11)])
    torch.cuda.synchronize()
    for tensor in (pool.key, pool.value, pool.bounds):
        assert torch.equal(tensor[:, 0], tensor[:, 9]) and torch.equal(tensor[:, 11], tensor[:, 4])
