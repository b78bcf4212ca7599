"""Bits that the 4-bit pool's attention and the selected decode have to keep, against the 64-bit oracle.

An output is the 64-bit value rounded once, off by half a step of its type at that value, plus 2 ``inner`` (twice, for
values at the border of two binades), where ``inner`` is what is lost before the rounding:
  weights: lg2.approx is off by 2^-22 relative, so of a step in [2^-6, 2^2] by at most 6 * 2^-22 (log2), which is
    4.2 * 2^-22 of a weight; ex2.approx by 2^-22, rcp.approx by 2^-23, the two fp16 terms of P' by 2^-22 (hi is
    nearest, the rest has 11 bits of its own): under 7 * 2^-22; scores of |s| < 3 (log2) that are one product (keys of
    one value each, a query of one power of two) have three roundings, 9 * 2^-24 ln 2: under 9 * 2^-22 of a weight in
    all, and twice that of a quotient of two sums;
  sums: fp32, of a few hundred tokens in at most 16 dependent additions of 2^-23 a warp, and the odd codes' sums are
    1/16 of a difference of sums 17 times as large, 2^-23 each: under 20 * 2^-23;
  together under 28 * 2^-22 of the spread of the values, taken as 2^-17;
  other scores, off by ds (log2): 2 ln 2 ds of the spread, ds = (D + 8) 2^-23 of the sum of the products' magnitudes.
"""

import math

import numpy as np
import pytest
import torch

from myvllm_mini_engine_b200.kernels import (int4_page_bytes, paged_attention_int4, paged_attention_selected,
                                             paged_prefill_attention_int4)
from oracle import int4_kv

pytestmark = pytest.mark.gpu


def randn(gen, *shape):
    return torch.from_numpy(gen.standard_normal(shape, dtype=np.float32))


def pool_of(rows, block_size):
    """A uint8 pool that holds ``rows [tokens, heads, dim]`` in the order of its slots."""
    tokens, heads, dim = rows.shape
    pool = np.zeros((-(-tokens // block_size), heads, int4_page_bytes(block_size, dim)), dtype=np.uint8)
    int4_kv.scatter(pool, block_size, torch.arange(tokens), rows)
    return pool


def half_step(x, dtype):
    bits, least = (10, -14) if dtype == torch.float16 else (7, -126)
    exponent = torch.frexp(x.abs()).exponent.double() - 1
    return torch.exp2(exponent.clamp(min=least) - bits - 1)


def assert_rounded_once(actual, expected, inner, dtype):
    err = (actual.double().cpu() - expected).abs()
    over = err - half_step(expected, dtype) - 2 * inner
    assert bool((over <= 0).all()), (int((over > 0).sum()), float(over.max()), float(err.max()))


def rows_of_many_steps(gen, tokens, heads, dim):
    """Normal rows, each times a factor of its own."""
    return (randn(gen, tokens, heads, dim) + randn(gen, heads, dim)) * (0.5 + 1.5 * torch.from_numpy(
        gen.random((tokens, heads, 1), dtype=np.float32)))


def keys_of_one_value(gen, tokens, heads, dim):
    """Rows of one fp16 value in (-1, 1) each: with a query of 1/8 everywhere a score is that value times sqrt(dim) / 8."""
    return torch.from_numpy(gen.uniform(-1, 1, (tokens, heads, 1)).astype(np.float16)).float().expand(-1, -1, dim)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,select,heads,kv_heads", [(32, False, 8, 4), (64, True, 12, 2), (128, False, 8, 4),
                                                       (128, True, 14, 2), (128, False, 9, 1), (256, False, 4, 1)])
def test_decode_weights_keep_their_bits(cuda_device, dtype, dim, select, heads, kv_heads):
    gen = np.random.default_rng(dim)
    bs, lens = 16, torch.tensor([1, 2, 3, 5, 17, 40, 130])
    width = 9
    rows = len(lens) * width * bs, kv_heads, dim
    kp, vp = pool_of(keys_of_one_value(gen, *rows), bs), pool_of(rows_of_many_steps(gen, *rows), bs)
    table = torch.from_numpy(gen.permutation(len(lens) * width).astype(np.int64)).view(len(lens), width)
    keys, vals = int4_kv.values(kp, bs, dim), int4_kv.values(vp, bs, dim)
    query = torch.full((len(lens), heads, dim), 0.125, dtype=dtype)
    selected = torch.arange(width).expand(len(lens), kv_heads, width).contiguous() if select else None
    expected = int4_kv.paged_decode(query, keys, vals, table, lens, bs)
    actual = paged_attention_int4(query.cuda(), *(torch.from_numpy(p).cuda() for p in (kp, vp)), table.cuda(), lens.cuda(),
                                  bs, validate=False, selected=None if selected is None else selected.cuda())
    assert_rounded_once(actual, expected, float(vals.max() - vals.min()) * 2.0 ** -17, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,count", [(32, 2, 9), (64, 4, 200), (128, 4, 20), (128, 4, 200), (256, 2, 30)])
def test_prefill_weights_keep_their_bits(cuda_device, dtype, dim, heads, count):
    gen = np.random.default_rng(dim + count)
    bs, kv_heads, start = 16, 2, 3
    rows = -(-(start + count) // bs) * bs, kv_heads, dim
    kp, vp = pool_of(keys_of_one_value(gen, *rows), bs), pool_of(rows_of_many_steps(gen, *rows), bs)
    keys, vals = int4_kv.values(kp, bs, dim), int4_kv.values(vp, bs, dim)
    q = torch.full((count, heads, dim), 0.125, dtype=dtype)
    meta = torch.tensor([0, count]), torch.tensor([start]), torch.arange(len(kp))[None], torch.tensor([start + count])
    expected = int4_kv.paged_prefill(q, keys, vals, *meta, bs)
    actual = paged_prefill_attention_int4(q.cuda(), *(torch.from_numpy(p).cuda() for p in (kp, vp)),
                                          *(m.cuda() for m in meta), bs)
    assert_rounded_once(actual, expected, float(vals.max() - vals.min()) * 2.0 ** -17, dtype)


@pytest.mark.parametrize("dtype,top,small", [
    # next to a largest element of 1024, two odd elements of 2^-4 that differ by 2^-9 of themselves
    (torch.float16, 1024.0, (1 + 33 / 1024, 1 + 31 / 1024)),
    (torch.bfloat16, 8192.0, (1 + 9 / 128, 1 + 7 / 128))])
@pytest.mark.parametrize("prefill", [False, True])
def test_small_query_elements_keep_their_bits(cuda_device, dtype, top, small, prefill):
    gen = np.random.default_rng(2)
    bs, dim = 16, 64
    keys, vals = torch.zeros(16, 1, dim), randn(gen, 16, 1, dim)
    keys[0, 0, 1] = keys[1, 0, 3] = 8192.0
    kp, vp = pool_of(keys, bs), pool_of(vals, bs)
    keys, vals = int4_kv.values(kp, bs, dim), int4_kv.values(vp, bs, dim)
    q = torch.zeros(1, 1, dim)
    q[0, 0, 0], q[0, 0, 1], q[0, 0, 3] = top, small[0] / 16, small[1] / 16
    assert torch.equal(q.to(dtype).float(), q)
    q = q.to(dtype)
    pools = [torch.from_numpy(p).cuda() for p in (kp, vp)]
    table, lens = torch.tensor([[0]]), torch.tensor([2])
    if prefill:
        meta = torch.tensor([0, 1]), torch.tensor([1]), table, lens
        expected = int4_kv.paged_prefill(q, keys, vals, *meta, bs)
        actual = paged_prefill_attention_int4(q.cuda(), *pools, *(m.cuda() for m in meta), bs)
    else:
        expected = int4_kv.paged_decode(q, keys, vals, table, lens, bs)
        actual = paged_attention_int4(q.cuda(), *pools, table.cuda(), lens.cuda(), bs)
    spread = float(vals[0, :2].max() - vals[0, :2].min())
    ds = (dim + 8) * 2.0 ** -23 * float(keys.max()) * small[0] / 16 * math.log2(math.e) / math.sqrt(dim)
    assert_rounded_once(actual, expected, spread * (2.0 ** -17 + 2 * math.log(2) * ds), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_rows_do_not_feel_a_value_they_do_not_weigh(cuda_device, dtype):
    """One value row 2^22 times the others': behind it, for the rows before; of no weight, for the rows after."""
    gen = np.random.default_rng(6)
    bs, dim, n, at = 16, 64, 64, 40
    keys, vals = randn(gen, n, 1, dim), randn(gen, n, 1, dim) * 2.0 ** -9
    keys[at] = -40.0  # with queries of 0.5: a score of -160
    q = torch.full((n, 1, dim), 0.5, dtype=dtype)
    meta = torch.tensor([0, n]), torch.tensor([0]), torch.arange(n // bs)[None], torch.tensor([n])
    large = vals.clone()
    large[at] = randn(gen, 1, dim) * 2.0 ** 13
    kp, vp, lp = pool_of(keys, bs), pool_of(vals, bs), pool_of(large, bs)

    def run(vp):
        return paged_prefill_attention_int4(q.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(),
                                            *(m.cuda() for m in meta), bs).cpu()

    without, actual = run(vp), run(lp)
    assert torch.equal(actual[:at], without[:at])
    k, v = int4_kv.values(kp, bs, dim), int4_kv.values(lp, bs, dim)
    expected = int4_kv.paged_prefill(q, k, v, *meta, bs)
    others = vals[torch.arange(n) != at]
    spread = float(others.max() - others.min())
    terms = 2 * dim * 0.5 * float(k.abs().max())
    ds = (dim + 8) * 2.0 ** -23 * terms * math.log2(math.e) / math.sqrt(dim)
    assert_rounded_once(actual[at + 1:], expected[at + 1:], spread * (2.0 ** -17 + 2 * math.log(2) * ds), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", ["decode", "prefill", "selected"])
def test_many_light_tokens_keep_their_values(cuda_device, dtype, form):
    """One token takes the weight; 131071 others, 2^-25.05 of it each, alone have values in the odd dims.

    Those dims hold the light tokens' sum, 2^-8 of their value, on two pages that the table repeats.  P' of a light
    token keeps 2^-11 at least (fp16, of which it is above the subnormals); the sum of the weights may miss the light
    ones, 2^-8 (a term below half a step of the sum it is added to).
    """
    bs, dim, n = 256, 64, 131072
    batch, kv_heads = (1, 1) if form == "prefill" else (64, 8)  # so that a warp of a decode has many of the tokens
    keys, vals = torch.zeros(2 * bs, kv_heads, dim), torch.ones(2 * bs, kv_heads, dim) * 15
    vals[:, :, 0] = 0.0  # base 0, step 1, codes 0 and 15
    keys[0] = 25.05 / (math.log2(math.e) * math.sqrt(dim))
    vals[0, :, 1::2] = 0.0
    table = torch.ones(batch, n // bs, dtype=torch.int64)
    table[:, 0] = 0
    lens = torch.full((batch,), n)
    q = torch.ones(batch, kv_heads, dim, dtype=dtype)
    if form == "selected":
        k16, v16 = (x.view(2, bs, kv_heads, dim).to(dtype) for x in (keys, vals))
        k, v = k16.double(), v16.double()
        listed = torch.arange(n // bs).expand(batch, kv_heads, -1).contiguous()
        actual = paged_attention_selected(q.cuda(), k16.cuda(), v16.cuda(), table.cuda(), lens.cuda(), listed.cuda(), bs)
    else:
        kp, vp = pool_of(keys, bs), pool_of(vals, bs)
        k, v = int4_kv.values(kp, bs, dim), int4_kv.values(vp, bs, dim)
        pools = [torch.from_numpy(p).cuda() for p in (kp, vp)]
        if form == "decode":
            actual = paged_attention_int4(q.cuda(), *pools, table.cuda(), lens.cuda(), bs)
        else:
            meta = torch.tensor([0, 1]), torch.tensor([n - 1]), table, lens
            actual = paged_prefill_attention_int4(q.cuda(), *pools, *(m.cuda() for m in meta), bs)
    weight = torch.exp(float(k[0, 0, 0].sum()) / math.sqrt(dim) * torch.tensor([1.0, 0.0], dtype=torch.float64))
    weight[1] *= n - 1
    weight /= weight.sum()
    odd = (weight[0] * v[0, 0, 0] + weight[1] * v[1, 0, 0])[1::2].expand(batch, kv_heads, -1)
    assert 0.02 < float(odd.min()) < 0.1
    ds = (dim + 8) * 2.0 ** -23 * 25.05
    bound = half_step(odd, dtype) + odd * (2.0 ** -7.9 + 2.0 ** -11 + 2 * math.log(2) * ds)
    assert bool(((actual.double().cpu()[..., 1::2] - odd).abs() <= bound).all()), actual[0, 0, :8]


def test_prefill_does_not_depend_on_its_neighbours(cuda_device):
    """bf16: a request alone, in batches of short and of long chunks, and on a wider table gives the same bytes."""
    gen = np.random.default_rng(8)
    bs, dim, heads, kv_heads, count, start = 16, 128, 4, 2, 40, 70
    blocks = 60
    pools = [torch.from_numpy(pool_of(rows_of_many_steps(gen, blocks * bs, kv_heads, dim), bs)).cuda() for _ in range(2)]
    table = torch.from_numpy(gen.permutation(blocks).astype(np.int64))
    q = randn(gen, 400, heads, dim).to(torch.bfloat16).cuda()

    def run(counts, starts, width):
        cu = torch.tensor([0, *np.cumsum(counts)])
        tables = torch.full((len(counts), width), -1)
        for r, (c, s) in enumerate(zip(counts, starts)):
            used = -(-(c + s) // bs)
            tables[r, :used] = table[20 * r:20 * r + used]
        lens = torch.tensor([c + s for c, s in zip(counts, starts)])
        return paged_prefill_attention_int4(q[:int(cu[-1])].contiguous(), *pools, cu.cuda(), torch.tensor(starts).cuda(),
                                            tables.cuda(), lens.cuda(), bs)[:count]

    alone = run([count], [start], 7)
    for counts, starts, width in (([count, 1, 1], [start, 5, 90], 7), ([count, 200], [start, 11], 14), ([count], [start], 60000)):
        assert torch.equal(run(counts, starts, width), alone)


def saturating_rows(gen, dim):
    """Rows whose largest element, or what it is rounded to, lies at the end of fp16's range (65504)."""
    x = randn(gen, 24, 2, dim) * torch.tensor([3e4, 2e4, 1.0])[torch.arange(24) % 3][:, None, None]
    x[0, 0, 0], x[0, 0, 1] = -65504.0, 65504.0   # step 8733.87, nearest fp16 8736: 15 of them reach 65536
    x[3, 0, 2], x[6, 1, 5], x[6, 1, 6] = math.inf, -math.inf, 1e30
    x[9] = -50.0
    x[9, :, 7] = 65504.0                          # step 4370.27, nearest 4372: 65530
    x[12], x[15] = 65504.0, 65500.0               # constant rows
    x[18], x[18, :, 3] = 65504.0, 65489.0         # the least element rounds up to the largest
    x[21], x[21, :, 0] = 60010.0, 65504.0
    return x


@pytest.mark.parametrize("src", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 96, 128])
def test_rows_at_the_end_of_the_range_read_back_finite(cuda_device, src, dim):
    from myvllm_mini_engine_b200.kernels import read_kv_cache_slots_int4, write_kv_cache_slots_int4

    bs = 16
    x = saturating_rows(np.random.default_rng(dim), dim).to(src)
    slots = torch.arange(24)
    got = torch.zeros(2, 2, 2, int4_page_bytes(bs, dim), dtype=torch.uint8, device="cuda")
    write_kv_cache_slots_int4(got[0], got[1], slots.cuda(), x.cuda(), x.cuda(), bs)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        key, value = read_kv_cache_slots_int4(got[0], got[1], slots.cuda(), bs, dim, dtype=dtype)
        assert bool(torch.isfinite(key).all()) and torch.equal(key, value)
        if dtype != torch.bfloat16:  # (65504 rounds to 65536 in bf16)
            assert float(key.abs().max()) <= 65504.0
    assert np.array_equal(got[0].cpu().numpy(), pool_of(x, bs))
    assert np.array_equal(got[1].cpu().numpy(), pool_of(x, bs))
    # an output that is one such value
    query = torch.zeros(24, 2, dim, dtype=torch.float16)
    table, lens = torch.arange(2)[None], torch.tensor([1])
    out = paged_attention_int4(query[:1].cuda(), got[0], got[1], table.cuda(), lens.cuda(), bs)
    assert bool(torch.isfinite(out).all())
    meta = torch.tensor([0, 24]), torch.tensor([0]), table, torch.tensor([24])
    assert bool(torch.isfinite(paged_prefill_attention_int4(query.cuda(), got[0], got[1], *(m.cuda() for m in meta), bs)).all())


@pytest.mark.parametrize("heads", [2, 8])
def test_warps_that_share_a_unit_join_all_of_its_parts(cuda_device, heads):
    """Every call gives the 64-bit answer's bytes again: units cut among the warps of several CTAs, many times over."""
    gen = np.random.default_rng(11)
    bs, dim, kv_heads, batch, n = 16, 64, 1, 600, 1500
    rows = 40 * bs, kv_heads, dim
    kp, vp = pool_of(keys_of_one_value(gen, *rows), bs), pool_of(rows_of_many_steps(gen, *rows), bs)
    keys, vals = int4_kv.values(kp, bs, dim), int4_kv.values(vp, bs, dim)
    table = torch.from_numpy(gen.integers(0, 40, (batch, -(-n // bs))).astype(np.int64))
    lens = torch.from_numpy(gen.integers(n // 2, n, batch).astype(np.int64))
    warps = torch.cuda.get_device_properties(0).multi_processor_count * 16
    assert 5 * warps <= int(((lens + 31) // 32).sum()) and -(-n // 32) * warps <= 8 * int(((lens + 31) // 32).sum())
    query = torch.full((batch, heads, dim), 0.125, dtype=torch.float16)
    args = query.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), table.cuda(), lens.cuda(), bs
    first = paged_attention_int4(*args)
    expected = int4_kv.paged_decode(query, keys, vals, table, lens, bs)
    # (partials: up to ten more sums, and sums of up to 1500 tokens)
    assert_rounded_once(first, expected, float(vals.max() - vals.min()) * 2.0 ** -15, torch.float16)
    for _ in range(50):
        assert torch.equal(paged_attention_int4(*args, validate=False), first)


@pytest.mark.parametrize("form", ["decode", "twin", "prefill"])
def test_sums_of_many_tokens_have_no_bias(cuda_device, form):
    """The mean of (output - 64-bit value) / (the codes' part of it), over outputs of thousands of tokens each.

    Sums of a tile lose at most 8 truncations of 2^-23, of which the mean is half; the tiles are added with rounding,
    as likely up as down. The outputs' own roundings, under 2^-11 / sqrt(12) of a value that is no larger than twice
    the codes' part, are independent: four deviations of their mean are added.
    """
    gen = np.random.default_rng(12)
    bs, dim, n = 16, 64, 16384 if form == "prefill" else 32768
    batch, kv_heads = (32, 2) if form == "prefill" else (512, 2)
    heads = kv_heads * (2 if form == "twin" else 6)
    rows = 64 * bs, kv_heads, dim
    kp, vp = pool_of(keys_of_one_value(gen, *rows), bs), pool_of(rows_of_many_steps(gen, *rows), bs)
    keys, vals = (int4_kv.values(p, bs, dim).view(-1, kv_heads, dim) for p in (kp, vp))
    table = torch.from_numpy(gen.integers(0, 64, (batch, n // bs)).astype(np.int64))
    query = torch.full((batch, heads, dim), 0.125, dtype=torch.float16)
    args = query.cuda(), torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda()
    lens = torch.full((batch,), n)
    if form == "prefill":
        cu = torch.arange(batch + 1)
        actual = paged_prefill_attention_int4(*args, cu.cuda(), (lens - 1).cuda(), table.cuda(), lens.cuda(), bs)
    else:
        actual = paged_attention_int4(*args, table.cuda(), lens.cuda(), bs)
    weight = torch.exp(keys[..., 0] * math.sqrt(dim) / 8)           # [slots, kv_heads]
    count = torch.stack([torch.bincount(t, minlength=64) for t in table]).double()
    page = torch.einsum("pshd,psh->phd", vals.view(64, bs, kv_heads, dim), weight.view(64, bs, kv_heads))
    low = torch.einsum("psh,psh->ph", vals.amin(-1).view(64, bs, kv_heads), weight.view(64, bs, kv_heads))
    total = (count @ weight.view(64, bs, kv_heads).sum(1))[..., None]
    expected = torch.einsum("bp,phd->bhd", count, page) / total
    codes = expected - (count @ low)[..., None] / total
    err = actual.double().cpu().view(batch, kv_heads, -1, dim) - expected[:, :, None]
    bias = float((err / codes[:, :, None]).mean())
    used = codes > 0.5 * expected.abs()
    assert float(used.double().mean()) > 0.9
    # the query heads of a kv head are alike, and so are their roundings
    chance = 4 * 2.0 ** -11 / math.sqrt(12) * 2 / math.sqrt(batch * kv_heads * dim)
    assert abs(bias) <= 4 * 2.0 ** -23 + chance, bias
