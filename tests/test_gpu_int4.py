"""4-bit KV pool on the GPU against the CPU oracle (oracle/int4_kv.py, 64 bits).

Writes match the oracle byte for byte.  Attention: with V values in a range of
``spread`` an output is off by at most
  half a step of its type (eps / 2 of its value), plus
  spread * (2^-12 P' rounded to fp16 once, as bf16 outputs and the prefill have it; 2^-22 in two
  terms) plus spread * 2 ln 2 * ds for scores off by ds (log2), where an fp32 dot product of D
  terms is off by at most (D + 8) 2^-23 of the sum of its terms' magnitudes.
The bf16 prefill over an fp16 copy of the pages: half a step of fp16, 2^-11, of every K (in ds, of the
sum of the products' magnitudes) and V besides.
"""

import math

import numpy as np
import pytest
import torch

from myvllm_mini_engine_b200 import _lib
from myvllm_mini_engine_b200.kernels import (int4_page_bytes, paged_attention_int4, paged_prefill_attention_int4,
                                             read_kv_cache_slots_int4, write_kv_cache_batch_int4,
                                             write_kv_cache_slots_int4)
from oracle import int4_kv

pytestmark = pytest.mark.gpu


def randn(gen, *shape):
    return torch.from_numpy(gen.standard_normal(shape, dtype=np.float32))


def make_pool(gen, blocks, block_size, heads, dim, scale=1.0):
    """A uint8 numpy pool of quantised normal rows with channel offsets."""
    pool = np.zeros((blocks, heads, int4_kv.page_bytes(block_size, dim)), dtype=np.uint8)
    rows = (randn(gen, blocks * block_size, heads, dim) + randn(gen, heads, dim)) * scale
    int4_kv.scatter(pool, block_size, torch.arange(blocks * block_size), rows)
    return pool


def tables_for(gen, lens, block_size, spare=3):
    width = max(1, -(-max(lens) // block_size))
    blocks = len(lens) * width + spare
    table = torch.from_numpy(gen.permutation(blocks)[:len(lens) * width].astype(np.int64)).view(len(lens), width)
    return table, blocks


def assert_near(actual, expected, query, keys, vals, dtype, one_term, copied=False):
    """The bound of the module's docstring, element by element, and half a step of the type over the whole."""
    finite_k, finite_v = keys[torch.isfinite(keys)], vals[torch.isfinite(vals)]
    spread = float(finite_v.max() - finite_v.min())
    dim = query.shape[-1]
    terms = float(query.double().abs().sum(-1).max()) * float(finite_k.abs().max()) * 2  # codes and base apart
    ds = (dim + 8) * 2.0 ** -23 * terms * math.log2(math.e) / math.sqrt(dim)
    copy = 2.0 ** -11 * float(finite_v.abs().max()) if copied else 0.0
    if copied:
        ds += 2.0 ** -11 * terms / 2 * math.log2(math.e) / math.sqrt(dim)
    inner = spread * ((2.0 ** -12 if one_term else 2.0 ** -22) + 2 * math.log(2) * ds) + copy
    half = torch.finfo(dtype).eps / 2
    err = (actual.double().cpu() - expected).abs()
    assert bool((err <= half * expected.abs() + inner + 2.0 ** -25).all()), float(err.max())
    norm = float(expected.norm())
    if norm:  # (below 2^-14 an fp16's half step is 2^-25, whatever the value)
        least = 2.0 ** -25 * math.sqrt(expected.numel()) if dtype == torch.float16 else 0.0
        assert float((actual.double().cpu() - expected).norm()) <= (half + 2.0 ** -11) * norm + least


def decode(gen, dtype, lens, heads, kv_heads, dim, block_size, *, tables=None, scale=1.0, selected=None,
           validate=True, pool_lens=None, q_scale=1.0):
    table, blocks = tables_for(gen, pool_lens or [max(1, n) for n in lens], block_size)
    if tables is not None:
        table = tables(table)
    kp, vp = make_pool(gen, blocks, block_size, kv_heads, dim, scale), make_pool(gen, blocks, block_size, kv_heads, dim, scale)
    query = (randn(gen, len(lens), heads, dim) * q_scale).to(dtype)
    lens = torch.tensor(lens, dtype=torch.int64)
    keys, vals = int4_kv.values(kp, block_size, dim), int4_kv.values(vp, block_size, dim)
    expected = int4_kv.paged_decode(query, keys, vals, table, lens, block_size, selected)
    actual = paged_attention_int4(query.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), table.cuda(),
                                  lens.cuda(), block_size, validate=validate,
                                  selected=None if selected is None else selected.cuda())
    assert actual.dtype == dtype and actual.shape == query.shape
    assert_near(actual, expected, query, keys, vals, dtype, dtype == torch.bfloat16)
    return actual, expected


@pytest.mark.parametrize("src", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,block_size", [(32, 5), (64, 16), (96, 16), (128, 16), (128, 1), (192, 7), (256, 24)])
def test_writes_match_the_oracle_bytes(cuda_device, src, dim, block_size):
    gen = np.random.default_rng(3)
    blocks, heads = 9, 3
    tokens = min(40, blocks * block_size)
    sizes = torch.tensor([1e-6, 1.0, 30.0, 3e4])[torch.arange(2 * tokens) % 4]
    data = randn(gen, 2, 2 * tokens, heads, dim) * sizes[:, None, None]
    data[0, 0, 0, 0], data[0, 0, 1, 1] = float("nan"), float("inf")
    data[1, 2] = 0.25                      # a constant row: step at its least, codes zero
    data[1, 4, 0, :16] = torch.arange(16)  # codes on and between whole numbers
    data[1, 4, 0, 16:] = torch.arange(dim - 16) % 16 + 0.5
    data = data.to(src)
    key, value = data[0, ::2], data[1, ::2]  # token-strided views
    slots = torch.from_numpy(gen.permutation(blocks * block_size)[:tokens].astype(np.int64))
    slots[1], slots[3] = -1, blocks * block_size
    init = gen.integers(0, 256, size=(2, blocks, heads, int4_page_bytes(block_size, dim)), dtype=np.uint8)
    want = init.copy()
    int4_kv.scatter(want[0], block_size, slots, key)
    int4_kv.scatter(want[1], block_size, slots, value)
    got = torch.from_numpy(init.copy()).cuda()
    write_kv_cache_slots_int4(got[0], got[1], slots.cuda(), key.cuda(), value.cuda(), block_size, validate=False)
    assert np.array_equal(got.cpu().numpy(), want)
    # misaligned sources take the element loads
    odd = torch.zeros(data[0, ::2].numel() + 1, dtype=src, device="cuda")[1:].view(tokens, heads, dim)
    odd.copy_(key)
    got = torch.from_numpy(init.copy()).cuda()
    write_kv_cache_slots_int4(got[0], got[1], slots.cuda(), odd, value.cuda(), block_size, validate=False)
    assert np.array_equal(got.cpu().numpy(), want)
    # the values read back
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        k, v = read_kv_cache_slots_int4(got[0], got[1], slots.cuda(), block_size, dim, dtype=dtype, validate=False)
        for have, pool in ((k, want[0]), (v, want[1])):
            flat = int4_kv.values(pool, block_size, dim).float().view(-1, heads, dim)
            inside = (slots >= 0) & (slots < blocks * block_size)
            ref = torch.where(inside[:, None, None], flat[slots.clamp(0, blocks * block_size - 1)], torch.zeros(1))
            assert torch.equal(have.cpu(), ref.to(dtype))


def test_batch_append_matches_the_oracle(cuda_device):
    gen = np.random.default_rng(4)
    blocks, heads, dim, bs = 12, 2, 64, 16
    tables = torch.from_numpy(gen.permutation(blocks)[:10].astype(np.int64)).view(5, 2)
    tables[3, 1] = blocks + 4
    offsets = torch.tensor([0, 17, 31, 20, 40])  # the fourth meets an invalid page, the last is past its table
    rows = randn(gen, 2, 5, heads, dim).to(torch.bfloat16)
    want = np.zeros((2, blocks, heads, int4_page_bytes(bs, dim)), dtype=np.uint8)
    for b in range(3):
        slot = int(tables[b, offsets[b] // bs]) * bs + int(offsets[b]) % bs
        for i in range(2):
            int4_kv.write_row(want[i], bs, slot, rows[i, b])
    got = torch.zeros(want.shape, dtype=torch.uint8, device="cuda")
    write_kv_cache_batch_int4(got[0], got[1], tables.cuda(), offsets.cuda(), rows[0].cuda(), rows[1].cuda(), bs,
                              validate=False)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_decode_head_dims(cuda_device, dtype, dim):
    decode(np.random.default_rng(dim), dtype, (1, 33, 300), 8, 4, dim, 16)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (8, 1), (9, 1), (20, 1), (6, 2), (24, 8), (4, 4)])
def test_decode_head_groups(cuda_device, heads, kv_heads):
    decode(np.random.default_rng(heads), torch.bfloat16, (65, 2, 129), heads, kv_heads, 64, 16)


@pytest.mark.parametrize("block_size,lens", [(1, (7, 40)), (5, (64, 3)), (8, (100, 8)), (24, (70, 25)), (48, (96, 47)),
                                             (256, (513, 1, 300)), (1000, (999, 1001))])
def test_decode_block_sizes(cuda_device, block_size, lens):
    decode(np.random.default_rng(block_size), torch.float16, lens, 4, 2, 128, block_size)


@pytest.mark.parametrize("lens", [(5000,), (4097, 1, 16, 2500), (31, 32, 33, 63, 64, 65) * 6])
def test_decode_splits(cuda_device, lens):
    decode(np.random.default_rng(len(lens)), torch.bfloat16, lens, 16, 8, 64, 16)


def test_decode_of_more_requests_than_threads(cuda_device):
    """700 requests, some of them without a token, on few pages."""
    gen = np.random.default_rng(17)
    kp, vp = make_pool(gen, 30, 16, 2, 32), make_pool(gen, 30, 16, 2, 32)
    lens = torch.from_numpy(gen.integers(0, 90, size=700).astype(np.int64))
    lens[5:9] = 0
    lens[690:] = torch.tensor([0, 0, 1, 89, 1 << 40, -1, 33, 0, 0, 0])
    table = torch.from_numpy(gen.integers(0, 30, size=(700, 6)).astype(np.int64))
    query = randn(gen, 700, 4, 32).to(torch.float16)
    keys, vals = int4_kv.values(kp, 16, 32), int4_kv.values(vp, 16, 32)
    expected = int4_kv.paged_decode(query, keys, vals, table, lens, 16)
    actual = paged_attention_int4(query.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), table.cuda(),
                                  lens.cuda(), 16, validate=False)
    assert_near(actual, expected, query, keys, vals, torch.float16, False)
    assert not actual[lens <= 0].any()


@pytest.mark.parametrize("dtype,dim,block_size,select", [
    (torch.bfloat16, 32, 16, False), (torch.float16, 64, 16, True), (torch.float16, 32, 5, False),
    (torch.bfloat16, 128, 16, False), (torch.bfloat16, 256, 16, False)])
def test_decode_of_long_batches(cuda_device, dtype, dim, block_size, select):
    """Enough tiles that warps work on runs of their own, with partials of a unit in several CTAs."""
    gen = np.random.default_rng(dim + block_size)
    batch, heads, kv_heads, longest = 260, 8, 8, 600
    lens = torch.from_numpy(np.linspace(longest, 300, batch).round().astype(np.int64)[gen.permutation(batch)])
    lens[100:103] = 0
    lens[200] = 1
    width = -(-longest // block_size)
    kp, vp = make_pool(gen, 30, block_size, kv_heads, dim), make_pool(gen, 30, block_size, kv_heads, dim)
    table = torch.from_numpy(gen.integers(0, 30, size=(batch, width)).astype(np.int64))
    selected = None
    if select:  # all blocks but every third
        listed = torch.tensor([j for j in range(width) if j % 3])
        listed = listed.expand(batch, kv_heads, -1).clone()
        listed[listed * block_size >= lens[:, None, None]] = -1
        selected = listed.contiguous()
    tiles = lens if selected is None else (selected >= 0).sum(-1)[:, 0] * block_size
    warps = torch.cuda.get_device_properties(0).multi_processor_count * 16
    assert int((tiles // 32).sum()) * kv_heads >= 5 * warps
    query = randn(gen, batch, heads, dim).to(dtype)
    keys, vals = int4_kv.values(kp, block_size, dim), int4_kv.values(vp, block_size, dim)
    expected = int4_kv.paged_decode(query, keys, vals, table, lens, block_size, selected)
    args = [x.cuda() for x in (query, torch.from_numpy(kp), torch.from_numpy(vp), table, lens)]
    listed = None if selected is None else selected.cuda()
    actual = paged_attention_int4(*args, block_size, selected=listed, validate=False)
    assert_near(actual, expected, query, keys, vals, dtype, dtype == torch.bfloat16)
    assert not actual[100:103].any()
    for _ in range(3):  # partials are joined in one order
        assert torch.equal(paged_attention_int4(*args, block_size, selected=listed, validate=False), actual)


@pytest.mark.parametrize("scale,q_scale", [(2.0 ** -12, 1.0), (3000.0, 2.0 ** -8), (1.0, 2.0 ** -40), (2.0 ** -9, 2.0 ** 30)])
def test_decode_extreme_scales(cuda_device, scale, q_scale):
    decode(np.random.default_rng(9), torch.bfloat16, (40, 700), 8, 2, 64, 16, scale=scale, q_scale=q_scale)


def test_decode_of_values_of_very_different_sizes(cuda_device):
    """The token that takes the weight has tiny values, the others large ones."""
    gen = np.random.default_rng(10)
    bs, dim = 16, 64
    kp, vp = (np.zeros((6, 1, int4_kv.page_bytes(bs, dim)), dtype=np.uint8) for _ in range(2))
    k, v = randn(gen, 90, 1, dim), randn(gen, 90, 1, dim) * 200
    query = randn(gen, 1, 2, dim).to(torch.float16)
    k[3, 0] = query[0, 0].float() * 4
    v[3] *= 2.0 ** -18
    slots = torch.arange(90)
    int4_kv.scatter(kp, bs, slots, k)
    int4_kv.scatter(vp, bs, slots, v)
    table, lens = torch.arange(6).view(1, 6), torch.tensor([90])
    keys, vals = int4_kv.values(kp, bs, dim), int4_kv.values(vp, bs, dim)
    expected = int4_kv.paged_decode(query, keys, vals, table, lens, bs)
    actual = paged_attention_int4(query.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), table.cuda(),
                                  lens.cuda(), bs)
    assert_near(actual, expected, query, keys, vals, torch.float16, False)


def test_decode_guards(cuda_device):
    """Invalid pages and lengths: masked tokens, zero rows, nothing read outside."""
    def spoil(table):
        table[0].fill_(-1)
        table[1, 3] = 1 << 40
        table[3, 0] = -7
        return table

    actual, _ = decode(np.random.default_rng(11), torch.bfloat16, (65, 300, 0, 17, 1 << 40, -3), 8, 2, 64, 16,
                       tables=spoil, validate=False, pool_lens=[65, 300, 16, 17, 16, 16])
    assert torch.isfinite(actual).all() and not actual[0].any() and not actual[2].any()
    assert not actual[4].any() and not actual[5].any()
    assert _lib.device_status() == 0


def test_decode_ignores_what_lies_behind_the_length(cuda_device):
    gen = np.random.default_rng(12)
    bs, dim = 16, 128
    kp, vp = make_pool(gen, 4, bs, 2, dim), make_pool(gen, 4, bs, 2, dim)
    query = randn(gen, 1, 4, dim).to(torch.bfloat16).cuda()
    table, lens = torch.tensor([[2, 0]]).cuda(), torch.tensor([21]).cuda()
    first = paged_attention_int4(query, torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), table, lens, bs)
    for pool in (kp, vp):  # NaN and infinite pairs, other codes, behind position 21 and in unused pages
        pairs = pool[..., bs * dim // 2:bs * (dim // 2 + 4)].view(np.float16).reshape(4, 2, bs, 2)
        pairs[0, :, 5:] = np.nan
        pairs[1], pairs[3] = np.inf, np.nan
        pool[0, :, 5 * dim // 2:bs * dim // 2] = 0xff
    again = paged_attention_int4(query, torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), table, lens, bs)
    assert torch.equal(first, again)


def test_decode_of_a_zeroed_pool_is_zero(cuda_device):
    pool = torch.zeros(3, 2, int4_page_bytes(16, 64), dtype=torch.uint8, device="cuda")
    query = torch.ones(1, 4, 64, dtype=torch.float16, device="cuda")
    out = paged_attention_int4(query, pool, pool.clone(), torch.tensor([[1, 2]]).cuda(), torch.tensor([20]).cuda(), 16)
    assert not out.any()


def test_decode_with_selected_blocks(cuda_device):
    gen = np.random.default_rng(13)
    lens = (300, 40, 17)
    selected = torch.full((3, 2, 6), -1, dtype=torch.int64)
    selected[0, 0, :4] = torch.tensor([0, 5, 9, 18])
    selected[0, 1, :6] = torch.tensor([1, 2, 3, 16, 17, 18])
    selected[1, 0, :3] = torch.tensor([0, 1, 2])
    selected[1, 1, :1] = torch.tensor([2])
    selected[2, 0, :1] = torch.tensor([1])  # the other head of request 2 attends nothing
    actual, _ = decode(gen, torch.bfloat16, lens, 6, 2, 128, 16, selected=selected)
    assert not actual[2, 3:].any()
    # every block listed: the attention over the whole table
    full, blocks = tables_for(gen, [70], 24)
    kp, vp = make_pool(gen, blocks, 24, 2, 64), make_pool(gen, blocks, 24, 2, 64)
    args = [randn(gen, 1, 4, 64).to(torch.float16).cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(),
            full.cuda(), torch.tensor([70]).cuda(), 24]
    all_blocks = torch.arange(3).expand(1, 2, 3).contiguous().cuda()
    assert torch.equal(paged_attention_int4(*args), paged_attention_int4(*args, selected=all_blocks))


def test_decode_is_repeatable_and_independent_of_the_batch(cuda_device):
    gen = np.random.default_rng(14)
    table, blocks = tables_for(gen, [2000] * 4, 16)
    kp, vp = (torch.from_numpy(make_pool(gen, blocks, 16, 2, 64)).cuda() for _ in range(2))
    query = randn(gen, 4, 8, 64).to(torch.float16).cuda()
    lens = torch.tensor([2000, 1500, 3, 900]).cuda()
    first = paged_attention_int4(query, kp, vp, table.cuda(), lens, 16)
    for _ in range(5):
        assert torch.equal(first, paged_attention_int4(query, kp, vp, table.cuda(), lens, 16))


def test_calls_of_other_shapes_between(cuda_device):
    """The ticket counters are zero after every call, whatever came before on the stream."""
    gen = np.random.default_rng(15)
    cases = []
    for batch, n in ((2, 3000), (300, 40), (1, 5000), (64, 200), (2, 3000)):
        table, blocks = tables_for(gen, [n] * batch, 16)
        pools = [torch.from_numpy(make_pool(gen, min(blocks, 40), 16, 1, 32)).cuda() for _ in range(2)]
        table = (table % min(blocks, 40)).cuda()
        cases.append((randn(gen, batch, 2, 32).to(torch.bfloat16).cuda(), *pools, table,
                      torch.full((batch,), n).cuda(), 16))
    alone = [paged_attention_int4(*c) for c in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, want in zip(cases, alone):
            assert torch.equal(paged_attention_int4(*c, validate=False), want)


def test_decode_on_other_streams_and_in_graphs(cuda_device):
    """Two graphs captured on one stream are replayed at once on two others, beside eager calls."""
    gen = np.random.default_rng(16)
    table, blocks = tables_for(gen, [4000] * 2, 16)
    kp, vp = (torch.from_numpy(make_pool(gen, blocks, 16, 2, 64)).cuda() for _ in range(2))
    table = table.cuda()
    lens = [torch.tensor(x).cuda() for x in ([4000, 3000], [100, 3999])]
    query = [randn(gen, 2, 8, 64).to(torch.bfloat16).cuda() for _ in range(2)]
    want = [paged_attention_int4(q, kp, vp, table, n, 16) for q, n in zip(query, lens)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for q, n in zip(query, lens):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(paged_attention_int4(q, kp, vp, table, n, 16, validate=False))
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        eager = paged_attention_int4(query[0], kp, vp, table, lens[0], 16, validate=False)
        for side, graph in zip(sides, graphs):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    # new lengths in a captured graph
    lens[0].copy_(torch.tensor([5, 4000]))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], paged_attention_int4(query[0], kp, vp, table, lens[0], 16))


# ------------------------------------------------------------------ prefill

@pytest.mark.parametrize("left", [0, 20, 1 << 20])
def test_captured_calls_have_counters_of_their_own(cuda_device, monkeypatch, left):
    """Graphs of several decodes that run at the same time, with kept counters or with the graph's own."""
    from myvllm_mini_engine_b200.kernels import int4

    gen = np.random.default_rng(31)
    table, blocks = tables_for(gen, [3000, 900], 16)
    kp, vp = (torch.from_numpy(make_pool(gen, blocks, 16, 2, 64)).cuda() for _ in range(2))
    lens, table = torch.tensor([3000, 900]).cuda(), table.cuda()
    query = [randn(gen, 2, 4, 64).to(torch.float16).cuda() for _ in range(6)]
    run = lambda q: paged_attention_int4(q, kp, vp, table, lens, 16, validate=False)  # noqa: E731
    expected = [run(q) for q in query]
    counters, used = int4._CAPTURED[torch.cuda.current_device()]
    monkeypatch.setitem(int4._CAPTURED, torch.cuda.current_device(), [counters, max(used, counters.numel() - left)])
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for part in (query[:3], query[3:]):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs += [run(q) for q in part]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, expected):
        assert torch.equal(out, want)
    assert not counters.any()


def prefill(gen, dtype, counts, starts, heads, kv_heads, dim, block_size, *, tables=None, lens=None, extra=0,
            validate=True, scale=1.0, max_query_len=None):
    full = [s + c for s, c in zip(starts, counts)]
    table, blocks = tables_for(gen, [max(1, n) for n in full], block_size)
    if tables is not None:
        table = tables(table)
    kp, vp = make_pool(gen, blocks, block_size, kv_heads, dim, scale), make_pool(gen, blocks, block_size, kv_heads, dim, scale)
    cu = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int64)
    starts = torch.tensor(starts, dtype=torch.int64)
    lens = torch.tensor(full if lens is None else lens, dtype=torch.int64)
    q = randn(gen, int(cu[-1]) + extra, heads, dim).to(dtype)
    keys, vals = int4_kv.values(kp, block_size, dim), int4_kv.values(vp, block_size, dim)
    expected = int4_kv.paged_prefill(q, keys, vals, cu, starts, table, lens, block_size)
    actual = paged_prefill_attention_int4(q.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), cu.cuda(),
                                          starts.cuda(), table.cuda(), lens.cuda(), block_size, validate=validate,
                                          max_query_len=max_query_len)
    assert actual.dtype == dtype and actual.shape == q.shape
    # the rule of the two routes: bf16, head_dim 64 or 128, enough rows a request, the tcgen05 kernel's pages
    copied = (dtype == torch.bfloat16 and dim in (64, 128) and block_size % 8 == 0 and 128 % (heads // kv_heads) == 0
              and q.shape[0] * (heads // kv_heads) >= 128 * len(counts))
    assert_near(actual, expected, q, keys, vals, dtype, True, copied)
    return actual


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_prefill_head_dims(cuda_device, dtype, dim):
    prefill(np.random.default_rng(dim), dtype, (1, 70, 33), (0, 37, 200), 8, 4, dim, 16)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (7, 1), (14, 2), (64, 1), (4, 4)])
def test_prefill_head_groups(cuda_device, heads, kv_heads):
    prefill(np.random.default_rng(heads), torch.bfloat16, (40, 5), (100, 0), heads, kv_heads, 64, 16)


@pytest.mark.parametrize("block_size,counts,starts", [(1, (9, 20), (3, 0)), (5, (30,), (64,)), (24, (65, 64, 63), (0, 1, 127)),
                                                      (256, (300, 2), (255, 256)), (16, (0, 17, 0), (5, 1, 9))])
def test_prefill_block_sizes_and_lengths(cuda_device, block_size, counts, starts):
    prefill(np.random.default_rng(block_size), torch.float16, counts, starts, 4, 2, 128, block_size)


@pytest.mark.parametrize("scale", [2.0 ** -12, 2000.0])
def test_prefill_extreme_scales(cuda_device, scale):
    prefill(np.random.default_rng(21), torch.bfloat16, (50,), (90,), 4, 2, 64, 16, scale=scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_growing_steps(cuda_device, dtype):
    """Values whose steps grow along the keys by far more than fp16's range."""
    gen = np.random.default_rng(22)
    bs, dim, n = 16, 64, 400
    kp, vp = (np.zeros((25, 1, int4_kv.page_bytes(bs, dim)), dtype=np.uint8) for _ in range(2))
    v = randn(gen, n, 1, dim) * torch.exp2(torch.linspace(-16, 13, n))[:, None, None]
    int4_kv.scatter(kp, bs, torch.arange(n), randn(gen, n, 1, dim))
    int4_kv.scatter(vp, bs, torch.arange(n), v)
    keys, vals = int4_kv.values(kp, bs, dim), int4_kv.values(vp, bs, dim)
    q = randn(gen, n, 2, dim).to(dtype)
    cu, starts, lens = torch.tensor([0, n]), torch.tensor([0]), torch.tensor([n])
    table = torch.arange(25).view(1, 25)
    expected = int4_kv.paged_prefill(q, keys, vals, cu, starts, table, lens, bs)
    actual = paged_prefill_attention_int4(q.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), cu.cuda(),
                                          starts.cuda(), table.cuda(), lens.cuda(), bs)
    # row by row: each has its own range of values (those it sees)
    for i in range(0, n, 7):
        assert_near(actual[i:i + 1], expected[i:i + 1], q[i:i + 1], keys, vals.view(-1, 1, dim)[:i + 1],
                    dtype, True, dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("more", [0, 100])
def test_prefill_guards(cuda_device, dtype, more):
    """Invalid pages, contexts that end early, tokens of no request, a bound below a request's length."""
    def spoil(table):
        table[0, 1] = -1
        table[1].fill_(1 << 33)
        return table

    first = 60 + more  # long chunks take the other route of bf16
    actual = prefill(np.random.default_rng(23), dtype, (first, 20, 50), (0, 7, 30), 4, 2, 64, 16, tables=spoil,
                     lens=(first, 27, 60), extra=9, validate=False, max_query_len=200 if more else 10)
    actual = actual[more:]
    assert not actual[60:80].any()          # every page of request 1 is invalid
    assert not actual[110:130].any()        # positions 60..79 of request 2 lie past its context
    assert not actual[130:].any()           # tokens of no request


@pytest.mark.parametrize("dim,heads,kv_heads,block_size,counts,starts", [
    (128, 8, 4, 16, (200, 64, 130), (37, 0, 500)), (64, 4, 4, 8, (300, 1), (5, 700)), (128, 16, 1, 24, (20, 9), (0, 90)),
    (64, 32, 1, 256, (33,), (255,)), (128, 2, 2, 64, (128, 128), (0, 0))])
def test_prefill_over_a_copy(cuda_device, dim, heads, kv_heads, block_size, counts, starts):
    """bf16 batches of enough queries a request, on the tcgen05 prefill."""
    prefill(np.random.default_rng(dim + heads), torch.bfloat16, counts, starts, heads, kv_heads, dim, block_size)


def test_prefill_in_a_graph(cuda_device):
    """Both routes, captured with one split of the queries and replayed with another."""
    gen = np.random.default_rng(25)
    table, blocks = tables_for(gen, [400, 400], 16)
    kp, vp = make_pool(gen, blocks, 16, 2, 64), make_pool(gen, blocks, 16, 2, 64)
    keys, vals = int4_kv.values(kp, 16, 64), int4_kv.values(vp, 16, 64)
    kp, vp, gpu_table = torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), table.cuda()
    for dtype in (torch.float16, torch.bfloat16):
        q = randn(gen, 200, 4, 64).to(dtype)
        cu, starts, lens = torch.tensor([0, 120, 200]), torch.tensor([10, 20]), torch.tensor([130, 100])
        gpu = [x.cuda() for x in (q, cu, starts, lens)]
        run = lambda: paged_prefill_attention_int4(gpu[0], kp, vp, gpu[1], gpu[2], gpu_table, gpu[3], 16,  # noqa: E731
                                                   validate=False)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        cu, starts, lens = torch.tensor([0, 50, 200]), torch.tensor([300, 0]), torch.tensor([350, 150])
        for held, new in zip(gpu[1:], (cu, starts, lens)):
            held.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        expected = int4_kv.paged_prefill(q, keys, vals, cu, starts, table, lens, 16)
        assert_near(out, expected, q, keys, vals, dtype, True, dtype == torch.bfloat16)


def test_prefill_matches_decode(cuda_device):
    """The last token of a prefill and the decode at its position agree to their roundings."""
    gen = np.random.default_rng(24)
    table, blocks = tables_for(gen, [200], 16)
    kp, vp = (torch.from_numpy(make_pool(gen, blocks, 16, 2, 128)).cuda() for _ in range(2))
    q = randn(gen, 50, 8, 128).to(torch.bfloat16).cuda()
    cu, starts, lens = (torch.tensor(x).cuda() for x in ([0, 50], [150], [200]))
    pre = paged_prefill_attention_int4(q, kp, vp, cu, starts, table.cuda(), lens, 16)
    dec = paged_attention_int4(q[-1:].contiguous(), kp, vp, table.cuda(), lens, 16)
    assert float((pre[-1:].float() - dec.float()).norm()) <= 2 * 2.0 ** -8 * float(dec.float().norm())
