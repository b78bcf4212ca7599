"""Block bounds, block selection and the attention over selected blocks, against the CPU oracle.

Bounds and selections match the oracle exactly.  The attention's bound is that of
tests/test_gpu_int4.py, with P in two terms of the pool's type (2^-16 for bf16).
"""

import math

import numpy as np
import pytest
import torch

from myvllm_mini_engine_b200 import _lib
from myvllm_mini_engine_b200.kernels import (block_bounds_bytes, paged_attention, paged_attention_int4,
                                             paged_attention_selected, read_block_bounds, select_blocks,
                                             update_block_bounds, write_kv_cache_batch_int4, write_kv_cache_slots_int4)
from oracle import block_select, int4_kv

pytestmark = pytest.mark.gpu


def randn(gen, *shape):
    return torch.from_numpy(gen.standard_normal(shape, dtype=np.float32))


def tables_for(gen, lens, block_size, spare=3):
    width = max(1, -(-max(lens) // block_size))
    blocks = len(lens) * width + spare
    table = torch.from_numpy(gen.permutation(blocks)[:len(lens) * width].astype(np.int64)).view(len(lens), width)
    return table, blocks


def int4_pool(gen, blocks, block_size, heads, dim):
    pool = np.zeros((blocks, heads, int4_kv.page_bytes(block_size, dim)), dtype=np.uint8)
    int4_kv.scatter(pool, block_size, torch.arange(blocks * block_size), randn(gen, blocks * block_size, heads, dim))
    return pool


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("pool", ["fp32", "fp16", "bf16", "int4"])
def test_bounds_match_the_oracle(cuda_device, pool, dim):
    gen = np.random.default_rng(dim)
    bs, heads = (16, 2) if dim != 96 else (7, 3)
    lens = (40, 16, 1, 33, 20)
    starts = torch.tensor([17, 0, 0, 33, 19])  # the fourth range is empty
    table, blocks = tables_for(gen, lens, bs)
    lens = torch.tensor(lens)
    if pool == "int4":
        cache = int4_pool(gen, blocks, bs, heads, dim)
        values, cache = int4_kv.values(cache, bs, dim), torch.from_numpy(cache)
    else:
        dtype = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[pool]
        cache = randn(gen, blocks, bs, heads, dim).to(dtype)
        first = int(table[0, 17 // bs])
        cache[first, 0, 0] = 0  # a block whose quotients fall on whole numbers
        cache[first, :, 0] = torch.arange(bs * dim).view(bs, dim) % 127 - 40
        cache[first, 0, 1, :3] = torch.tensor([float("nan"), float("inf"), -float("inf")])
        cache[int(table[1, 0])] = 0
        values = cache.double()
    init = gen.integers(0, 256, size=(blocks, heads, block_bounds_bytes(dim)), dtype=np.uint8)
    want = init.copy()
    block_select.update(want, values, table, starts, lens, bs)
    for longest in (None, 23):  # the second is the longest range
        got = torch.from_numpy(init.copy()).cuda()
        update_block_bounds(got, cache.cuda(), table.cuda(), starts.cuda(), lens.cuda(), bs, max_query_len=longest)
        assert np.array_equal(got.cpu().numpy(), want)
    touched = torch.tensor([int(table[0, 17 // bs]), int(table[2, 0]), -1, blocks])
    lower, upper = read_block_bounds(got, touched.cuda(), validate=False)
    ref_lower, ref_upper = block_select.read(want, touched[:2].numpy(), dim)
    assert torch.equal(lower[:2].cpu(), ref_lower) and torch.equal(upper[:2].cpu(), ref_upper)
    assert not lower[2:].any() and not upper[2:].any()


def test_bounds_bound_the_keys(cuda_device):
    gen = np.random.default_rng(1)
    cache = randn(gen, 6, 16, 2, 64).to(torch.bfloat16).cuda()
    bounds = torch.zeros(6, 2, block_bounds_bytes(64), dtype=torch.uint8, device="cuda")
    table, starts, lens = torch.arange(6).view(1, 6).cuda(), torch.tensor([0]).cuda(), torch.tensor([96]).cuda()
    update_block_bounds(bounds, cache, table, starts, lens, 16)
    lower, upper = read_block_bounds(bounds, torch.arange(6).cuda())
    keys = cache.float().transpose(1, 2)
    slack = keys.abs().amax((2, 3), keepdim=True) * 2.0 ** -22  # the scale and the product round once each
    assert bool((keys <= upper[:, :, None] + slack).all()) and bool((keys >= lower[:, :, None] - slack).all())


def test_bounds_guards(cuda_device):
    gen = np.random.default_rng(2)
    cache = randn(gen, 5, 16, 1, 32).to(torch.float16)
    table = torch.tensor([[0, -1, 9], [1, 2, 3], [1, 2, 3], [4, 4, 4]])
    starts, lens = torch.tensor([0, -5, 0, 40]), torch.tensor([48, 20, 49, 48])
    want = np.zeros((5, 1, block_bounds_bytes(32)), dtype=np.uint8)
    block_select.update(want, cache.double(), table, starts, lens, 16)
    got = torch.zeros(want.shape, dtype=torch.uint8, device="cuda")
    update_block_bounds(got, cache.cuda(), table.cuda(), starts.cuda(), lens.cuda(), 16, validate=False)
    assert np.array_equal(got.cpu().numpy(), want)


def test_bounds_refuse_what_depends_on_the_order(cuda_device):
    keys = torch.randn(4, 16, 2, 64, device="cuda").half()
    bounds = torch.zeros(4, 2, block_bounds_bytes(64), dtype=torch.uint8, device="cuda")
    table = torch.tensor([[0, 1], [0, 2]], device="cuda")
    starts = torch.zeros(2, dtype=torch.int64, device="cuda")
    update_block_bounds(bounds, keys, table, starts, torch.tensor([20, 32]).cuda(), 16)  # a full shared block
    with pytest.raises(RuntimeError, match="same rows"):
        update_block_bounds(bounds, keys, table, starts, torch.tensor([20, 9]).cuda(), 16)
    update_block_bounds(bounds, keys, table, starts, torch.tensor([20, 16]).cuda(), 16, max_query_len=20)
    with pytest.raises(RuntimeError, match="max_query_len"):
        update_block_bounds(bounds, keys, table, starts, torch.tensor([20, 16]).cuda(), 16, max_query_len=19)


def select_both(gen, lens, heads, kv_heads, dim, block_size, take, *, sink=1, recent=1, dtype=torch.bfloat16,
                levels=None, spoil=None, query=None, validate=True, pool_lens=None):
    table, blocks = tables_for(gen, pool_lens or lens, block_size)
    if spoil is not None:
        spoil(table)
    low = -np.abs(gen.standard_normal((blocks, kv_heads, dim))) - 0.5
    high = np.abs(gen.standard_normal((blocks, kv_heads, dim))) + 0.5
    if levels is not None:  # few distinct records, so that many scores are equal
        low, high = low[np.arange(blocks) % levels], high[np.arange(blocks) % levels]
    bounds = np.stack([np.stack([block_select.record(np.stack((low[i, h], high[i, h]))) for h in range(kv_heads)])
                       for i in range(blocks)])
    query = (randn(gen, len(lens), heads, dim) if query is None else query).to(dtype)
    lens = torch.tensor(lens)
    want = block_select.select(query, bounds, table, lens, block_size, take, sink, recent)
    got = select_blocks(query.cuda(), torch.from_numpy(bounds).cuda(), table.cuda(), lens.cuda(), block_size, take,
                        sink_blocks=sink, recent_blocks=recent, validate=validate)
    assert torch.equal(got.cpu(), want)
    return want


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_selection_matches_the_oracle(cuda_device, dtype, dim):
    select_both(np.random.default_rng(dim), (1000, 17, 160, 161, 1), 8, 4, dim, 16, 10, dtype=dtype)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (9, 9), (33, 11), (16, 2)])
def test_selection_head_groups(cuda_device, heads, kv_heads):
    select_both(np.random.default_rng(heads), (500, 301), heads, kv_heads, 64, 8, 12)


@pytest.mark.parametrize("take,sink,recent", [(1, 0, 0), (1, 1, 0), (2, 1, 1), (5, 2, 3), (40, 0, 1), (62, 1, 1), (63, 1, 1),
                                              (64, 1, 1), (200, 3, 3)])
def test_selection_sizes(cuda_device, take, sink, recent):
    select_both(np.random.default_rng(take), (1000, 999, 50), 4, 2, 64, 16, take, sink=sink, recent=recent)


def test_equal_scores_go_to_the_lowest_block(cuda_device):
    gen = np.random.default_rng(5)
    for levels, take in ((1, 7), (2, 30), (3, 64)):
        select_both(gen, (1600, 1111), 4, 2, 32, 16, take, levels=levels)
    # a zero query: every score is zero, of either sign
    want = select_both(gen, (1600,), 4, 2, 32, 16, 6, query=torch.zeros(1, 4, 32))
    assert want[0, 0].tolist() == [0, 1, 2, 3, 4, 99]


def test_selection_of_odd_queries(cuda_device):
    gen = np.random.default_rng(6)
    query = randn(gen, 1, 4, 64)
    query[0, 0, 3], query[0, 1, 5], query[0, 2, 7] = float("nan"), float("inf"), -float("inf")
    select_both(gen, (900,), 4, 2, 64, 16, 9, query=query, dtype=torch.float32)
    select_both(gen, (900,), 4, 2, 64, 16, 9, query=torch.full((1, 4, 64), 1e-35), dtype=torch.float32)


def test_selection_guards(cuda_device):
    def spoil(table):
        table[0, ::3] = -1
        table[1].fill_(1 << 40)
        table[3, 1:] = -1

    want = select_both(np.random.default_rng(7), (800, 800, 0, 700, 1 << 30), 4, 2, 64, 16, 20, spoil=spoil, validate=False,
                       pool_lens=(800, 800, 16, 700, 16))
    assert (want[1] == -1).all() and (want[2] == -1).all() and (want[4] == -1).all()
    assert (want[3, :, 0] == 0).all() and (want[3, :, 1:] == -1).all()


@pytest.mark.parametrize("blocks", [24576, 24577, 60000])
def test_selection_of_very_long_requests(cuda_device, blocks):
    """Around the number of keys that shared memory holds; against a sort of the same scores."""
    gen = torch.Generator("cuda").manual_seed(blocks)
    dim, pool = 32, 512
    bounds = torch.zeros(pool, 1, block_bounds_bytes(dim), dtype=torch.uint8, device="cuda")
    keys = torch.randn(pool, 2, 1, dim, generator=gen, device="cuda")
    update_block_bounds(bounds, keys, torch.arange(pool, device="cuda").view(1, pool), torch.tensor([0]).cuda(),
                        torch.tensor([2 * pool]).cuda(), 2)
    table = torch.randint(0, pool, (1, blocks), generator=gen, device="cuda")
    lens = torch.tensor([2 * blocks]).cuda()
    query = torch.randn(1, 2, dim, generator=gen, device="cuda")
    got = select_blocks(query, bounds, table, lens, 2, 300)
    codes = torch.from_numpy(block_select.query_codes(query[0])).cuda().double()
    score = bounds[:, 0, :2 * dim].view(torch.int8).double() @ codes
    score = (score.float() * bounds[:, 0, 2 * dim:2 * dim + 4].contiguous().view(torch.float32)[:, 0])[table[0]]
    score[0] = score[-1] = math.inf
    want = torch.sort(score, descending=True, stable=True).indices[:300].sort().values
    assert torch.equal(got[0, 0], want)


def attend_both(gen, dtype, lens, heads, kv_heads, dim, block_size, take, *, spoil=None, validate=True, pool_lens=None):
    table, blocks = tables_for(gen, pool_lens or lens, block_size)
    kc, vc = (randn(gen, blocks, block_size, kv_heads, dim).to(dtype) for _ in range(2))
    selected = torch.full((len(lens), kv_heads, take), -1, dtype=torch.int64)
    for b, n in enumerate(lens):
        have = min(table.shape[1], -(-max(0, n) // block_size))
        for h in range(kv_heads):
            chosen = np.sort(gen.permutation(have)[:gen.integers(1, take + 1) if have else 0])
            selected[b, h, :len(chosen)] = torch.from_numpy(chosen.astype(np.int64))
    if spoil is not None:
        spoil(table, selected, kc, vc)
    query, lens = randn(gen, len(lens), heads, dim).to(dtype), torch.tensor(lens)
    expected = int4_kv.paged_decode(query, kc.double(), vc.double(), table, lens, block_size, selected)
    actual = paged_attention_selected(query.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(), selected.cuda(),
                                      block_size, validate=validate)
    finite_k, finite_v = kc[torch.isfinite(kc)].double(), vc[torch.isfinite(vc)].double()
    spread = float(finite_v.max() - finite_v.min())
    terms = float(query.double().abs().sum(-1).max()) * float(finite_k.abs().max())
    ds = (dim + 8) * 2.0 ** -23 * terms * math.log2(math.e) / math.sqrt(dim)
    half = torch.finfo(dtype).eps / 2
    err = (actual.double().cpu() - expected).abs()
    assert bool((err <= half * expected.abs() + spread * (2.0 ** -16 + 2 * math.log(2) * ds) + 2.0 ** -25).all())
    assert float(err.norm()) <= (half + 2.0 ** -13) * float(expected.norm())
    return actual


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_attention_over_selected_blocks(cuda_device, dtype, dim):
    attend_both(np.random.default_rng(dim), dtype, (500, 33, 1), 8, 4, dim, 16, 9)


@pytest.mark.parametrize("heads,kv_heads,block_size,take", [(7, 1, 16, 30), (9, 1, 5, 40), (16, 16, 24, 6), (20, 2, 1, 77),
                                                            (4, 2, 256, 2), (8, 8, 8, 1)])
def test_selected_head_groups_and_block_sizes(cuda_device, heads, kv_heads, block_size, take):
    attend_both(np.random.default_rng(take), torch.bfloat16, (600, 301), heads, kv_heads, 64, block_size, take)


def test_selected_guards(cuda_device):
    def spoil(table, selected, kc, vc):
        table[0, 1::2] = -1
        selected[1, 0, 0], selected[1, 1] = 1 << 40, -5
        free = sorted(set(range(kc.shape[0])) - set(table.flatten().tolist()))
        kc[free] = float("nan")  # pages of nobody
        vc[free] = float("inf")
        page = int(table[3, 40 // 16])  # and the rows behind a request's last
        kc[page, 41 % 16:], vc[page, 41 % 16:] = float("nan"), float("nan")
        selected[3, :, 0], selected[3, :, 1], selected[3, :, 2:] = 0, 2, -1

    actual = attend_both(np.random.default_rng(8), torch.bfloat16, (300, 200, 0, 41, 1 << 33), 4, 2, 64, 16, 8, spoil=spoil,
                         validate=False, pool_lens=(300, 200, 16, 41, 16))
    assert torch.isfinite(actual).all() and not actual[1, 2:].any() and not actual[2].any() and not actual[4].any()
    assert _lib.device_status() == 0


def test_all_blocks_selected_is_the_plain_decode(cuda_device):
    gen = np.random.default_rng(9)
    table, blocks = tables_for(gen, (700,), 16)
    kc, vc = (randn(gen, blocks, 16, 2, 128).to(torch.bfloat16).cuda() for _ in range(2))
    query, lens = randn(gen, 1, 8, 128).to(torch.bfloat16).cuda(), torch.tensor([700]).cuda()
    everything = torch.arange(44).expand(1, 2, 44).contiguous().cuda()
    a = paged_attention_selected(query, kc, vc, table.cuda(), lens, everything, 16)
    b = paged_attention(query, kc, vc, table.cuda(), lens, 16)
    assert float((a.float() - b.float()).norm()) <= 2.0 ** -7 * float(b.float().norm())  # each half a step off


@pytest.mark.parametrize("graph", [False, True])
def test_a_run_of_steps_over_a_4bit_pool(cuda_device, graph):
    """Prompt write, bounds, then decode steps (append, bounds, selection, attention), each against the oracle."""
    gen = np.random.default_rng(10)
    bs, heads, kv_heads, dim, take = 16, 4, 2, 64, 4
    prompt = [130, 47]
    table, blocks = tables_for(gen, [n + 8 for n in prompt], bs)
    kp, vp = (torch.zeros(blocks, kv_heads, int4_kv.page_bytes(bs, dim), dtype=torch.uint8, device="cuda") for _ in range(2))
    bounds = torch.zeros(blocks, kv_heads, block_bounds_bytes(dim), dtype=torch.uint8, device="cuda")
    gpu_table = table.cuda()
    starts, lens = torch.zeros(2, dtype=torch.int64).cuda(), torch.tensor(prompt).cuda()
    for b, n in enumerate(prompt):
        pos = torch.arange(n)
        slots = (table[b, pos // bs] * bs + pos % bs).cuda()
        rows = randn(gen, 2, n, kv_heads, dim).to(torch.bfloat16).cuda()
        write_kv_cache_slots_int4(kp, vp, slots, rows[0], rows[1], bs)
    update_block_bounds(bounds, kp, gpu_table, starts, lens, bs)
    query = torch.zeros(2, heads, dim, dtype=torch.bfloat16, device="cuda")
    new = torch.zeros(2, 2, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    at = lens.clone()

    def step():
        write_kv_cache_batch_int4(kp, vp, gpu_table, at, new[0], new[1], bs, validate=False)
        after = at + 1
        update_block_bounds(bounds, kp, gpu_table, at, after, bs, validate=False, max_query_len=1)
        chosen = select_blocks(query, bounds, gpu_table, after, bs, take, validate=False)
        return chosen, paged_attention_int4(query, kp, vp, gpu_table, after, bs, selected=chosen, validate=False)

    if graph:
        keep = (kp.clone(), vp.clone(), bounds.clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            held = step()
        for tensor, old in zip((kp, vp, bounds), keep):
            tensor.copy_(old)

        def step():  # noqa: F811
            captured.replay()
            return held

    for i in range(6):
        query.copy_(randn(gen, 2, heads, dim))
        new.copy_(randn(gen, 2, 2, kv_heads, dim))
        chosen, out = step()
        torch.cuda.synchronize()
        after = (at + 1).cpu()
        keys, vals = (int4_kv.values(pool.cpu().numpy(), bs, dim) for pool in (kp, vp))
        want = bounds.cpu().numpy().copy()
        block_select.update(want, keys, table, torch.zeros(2, dtype=torch.int64), after, bs)
        assert np.array_equal(bounds.cpu().numpy(), want)
        assert torch.equal(chosen.cpu(), block_select.select(query.cpu(), want, table, after, bs, take))
        expected = int4_kv.paged_decode(query.cpu(), keys, vals, table, after, bs, chosen.cpu())
        assert float((out.double().cpu() - expected).norm()) <= (2.0 ** -8 + 2.0 ** -11) * float(expected.norm())
        at += 1
