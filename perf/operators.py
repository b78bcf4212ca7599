"""Cases of the 4-bit KV cache and of the attention over selected blocks, with their plain forms.

Six operators, each as its plain form (elementary torch operations in 32 bits, rounded once at the end) and, where
``own`` is true, as the calls a user makes of the framework:

* ``write``    quantise K/V rows into a 4-bit pool at their slots and read the same slots back;
* ``decode``   attention of one query token per request over a 4-bit pool;
* ``prefill``  ragged causal attention over a 4-bit pool;
* ``bounds``   per-block key bounds of the blocks that newly written rows touch;
* ``select``   the blocks of highest score for each request and kv head;
* ``attend``   decode attention over selected blocks, of a 16-bit pool or of a 4-bit pool.

Formats (the framework's):

* 4-bit pool ``[blocks, kv_heads, page_bytes]`` uint8.  A page of one kv head holds ``block_size`` rows of
  ``head_dim / 2`` bytes (element 2i in the low half of byte i), then ``block_size`` pairs of fp16 (step, base); an
  element reads as ``base + step * code``.  Rows are quantised one by one: base = fp16(min), step = fp16((max - min) / 15),
  at least 2^-24, code = round((x - base) / step) in 0..15, all quotients true ones.
* block bounds ``[blocks, kv_heads, 2 * head_dim + 16]`` uint8: ``head_dim`` int8 codes of the keys' elementwise
  maximum, ``head_dim`` of their minimum, one fp32 scale = top / 127 with top the largest magnitude of the 2 * head_dim
  bounds; the codes are ceil(127 * max / top) and floor(127 * min / top), and a bound reads as ``code * scale``.
* a block's score for a kv head bounds the sum of its query heads' dot products with any key of the block:
  ``sum_d max_d * qp_d + min_d * qn_d`` with qp / qn the summed positive / negative parts of the heads' queries, held in
  8 bits.  The sum of the codes' products is a whole number, so a score has one value whatever the order of its sum.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
F32_MAX = 3.4028234663852886e38
STEP_MIN = 2.0 ** -24


def listed():
    return [
        # a decode step's append: one new row for each of 32 requests (latency)
        {"name": "write_step_b32", "op": "write", "dtype": "bf16", "tokens": 32, "kv_heads": 8, "dim": 128, "bs": 16},
        # a prompt chunk's rows, 64-wide heads
        {"name": "write_chunk_16k", "op": "write", "dtype": "fp16", "tokens": 16384, "kv_heads": 8, "dim": 64, "bs": 32},
        # a small interactive batch on large pages
        {"name": "decode_b8_ctx513", "op": "decode", "dtype": "fp16", "batch": 8, "lo": 513, "hi": 513, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "bs": 256},
        # a full serving batch at long contexts
        {"name": "decode_b256_ctx4096", "op": "decode", "dtype": "bf16", "batch": 256, "lo": 4096, "hi": 4096,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "bs": 16},
        # chunked prefill: short chunks behind ragged cached prefixes
        {"name": "prefill_16x128", "op": "prefill", "dtype": "bf16", "requests": 16, "new_lo": 128, "new_hi": 128,
         "past": 1024, "q_heads": 16, "kv_heads": 8, "dim": 128, "bs": 16},
        # long chunks of ragged lengths deep in a long prompt
        {"name": "prefill_4x1000_past4k", "op": "prefill", "dtype": "fp16", "requests": 4, "new_lo": 500, "new_hi": 1000,
         "past": 4096, "q_heads": 32, "kv_heads": 8, "dim": 128, "bs": 16},
        # the bounds after one decode step, read from the 4-bit pool
        {"name": "bounds_step_b32", "op": "bounds", "pool": "int4", "dtype": "bf16", "batch": 32, "lo": 1024, "hi": 4096,
         "new": 1, "kv_heads": 8, "dim": 128, "bs": 16},
        # the bounds after a prompt chunk, read from a 16-bit pool
        {"name": "bounds_chunk_16x1024", "op": "bounds", "pool": "16bit", "dtype": "bf16", "batch": 16, "lo": 2048,
         "hi": 4096, "new": 1024, "kv_heads": 8, "dim": 128, "bs": 16},
        # one long conversation
        {"name": "select_b1_ctx8k", "op": "select", "dtype": "fp16", "batch": 1, "lo": 8000, "hi": 8192, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "bs": 16, "take": 64},
        # a batch of very long contexts
        {"name": "select_b32_ctx32k", "op": "select", "dtype": "bf16", "batch": 32, "lo": 24000, "hi": 32768,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "bs": 16, "take": 256},
        # the blocks so chosen, attended in a 16-bit pool
        {"name": "attend_b4_top128", "op": "attend", "pool": "16bit", "dtype": "bf16", "batch": 4, "lo": 24000,
         "hi": 32768, "q_heads": 16, "kv_heads": 8, "dim": 128, "bs": 16, "take": 128},
        # and in a 4-bit pool
        {"name": "attend_int4_b32_top256", "op": "attend", "pool": "int4", "dtype": "bf16", "batch": 32, "lo": 8192,
         "hi": 16384, "q_heads": 32, "kv_heads": 8, "dim": 128, "bs": 16, "take": 256},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "decode", "decode", "prefill", "bounds", "select", "attend", "attend"])
    case = {"op": op, "dtype": rng.choice(["fp16", "bf16"]), "kv_heads": rng.choice([1, 2, 4, 8]),
            "dim": rng.choice([64, 128, 128, 256]), "bs": rng.choice([8, 16, 16, 24, 32, 64, 256])}
    group = rng.choice([1, 2, 3, 4, 7, 8])
    # the largest drawn case costs about an eighth of the largest listed one
    if op == "write":
        case["tokens"] = _between(rng, 1, 16384)
        return case
    if op == "prefill":
        case |= {"requests": rng.randint(1, 8), "new_lo": 1, "new_hi": _between(rng, 2, 400), "past": _between(rng, 1, 2048),
                 "q_heads": case["kv_heads"] * group}
        return case
    hi = _between(rng, 2, 16384)
    case |= {"batch": _between(rng, 1, max(1, min(64, 262144 // hi))), "lo": max(1, hi // rng.choice([1, 2, 8])), "hi": hi}
    if op == "bounds":
        return case | {"pool": rng.choice(["int4", "16bit"]), "new": _between(rng, 1, case["lo"])}
    case["q_heads"] = case["kv_heads"] * group
    if op in ("select", "attend"):
        case["take"] = _between(rng, 2, 256)
    if op == "attend":
        case["pool"] = rng.choice(["int4", "16bit"])
    return case


# ------------------------------------------------------------------ formats, in plain operations

def _page_bytes(bs, dim):
    return (bs * (dim // 2 + 4) + 15) // 16 * 16


def _over(a, b):
    """a / b, rounded once (a division by a Python number multiplies by its rounded inverse, and so does one of it)."""
    a, b = (torch.as_tensor(v, dtype=torch.float32, device="cuda") for v in (a, b))
    return a / b


def _quantize(x):
    """(codes uint8, step fp16, base fp16) of rows over the last axis."""
    x = x.float().nan_to_num(nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    base = low.half()
    step = _over(high - low, 15.0).clamp(min=STEP_MIN).half()
    codes = torch.round(_over(x - base.float(), step.float())).clamp(0.0, 15.0).to(torch.uint8)
    return codes, step[..., 0], base[..., 0]


def _pack_rows(codes, step, base):
    """Bytes of the rows and of their (step, base) pairs."""
    rows = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return rows, torch.stack((step, base), -1).view(torch.uint8)


def _values(pages, bs, dim, wide=torch.float32):
    """Values ``[..., bs, dim]`` that pages ``[..., page_bytes]`` of a 4-bit pool stand for."""
    rows = pages[..., : bs * dim // 2].unflatten(-1, (bs, dim // 2))
    codes = torch.stack((rows & 15, rows >> 4), -1).flatten(-2).to(wide)
    pairs = pages[..., bs * dim // 2: bs * (dim // 2 + 4)].contiguous().view(torch.float16).unflatten(-1, (bs, 2)).to(wide)
    return pairs[..., 1:] + pairs[..., :1].clamp(min=STEP_MIN) * codes


def _bound_codes(low, high):
    """(high codes, low codes, scale) of elementwise bounds over the last axis."""
    top = torch.maximum(low.abs(), high.abs()).amax(-1, keepdim=True)
    none = top < 2.0 ** -100
    scale = torch.where(none, torch.zeros_like(top), _over(top, 127.0))
    # in 64 bits: a quotient next to a whole number must not be rounded across it
    high, low, wide = high.double() * 127.0, low.double() * 127.0, torch.where(none, math.inf, top.double())
    up = torch.ceil(high / wide).clamp(-127.0, 127.0)
    down = torch.floor(low / wide).clamp(-127.0, 127.0)
    return up.to(torch.int8), down.to(torch.int8), scale


def _pack_bounds(low, high):
    up, down, scale = _bound_codes(low, high)
    pad = torch.zeros((*scale.shape[:-1], 12), dtype=torch.uint8, device=scale.device)
    return torch.cat((up.view(torch.uint8), down.view(torch.uint8), scale.contiguous().view(torch.uint8), pad), -1)


# ------------------------------------------------------------------ inputs

def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _rows_like_keys(gen, n, heads, dim, dtype):
    """Rows with the channel offsets and the spread that keys have."""
    x = _randn(gen, n, heads, dim, dtype=dtype)
    return x * (0.5 + torch.rand(heads, dim, generator=gen, device="cuda")).to(dtype) + _randn(gen, heads, dim, dtype=dtype)


def _int4_pool(gen, blocks, heads, bs, dim):
    pool = torch.zeros(blocks, heads, _page_bytes(bs, dim), dtype=torch.uint8, device="cuda")
    at, piece = 0, max(1, (1 << 26) // (heads * bs * dim))
    while at < blocks:
        n = min(piece, blocks - at)
        rows, pairs = _pack_rows(*_quantize(_rows_like_keys(gen, n * bs, heads, dim, torch.float32)))
        pool[at:at + n, :, : bs * dim // 2] = rows.view(n, bs, heads, -1).transpose(1, 2).flatten(-2)
        pool[at:at + n, :, bs * dim // 2: bs * (dim // 2 + 4)] = pairs.view(n, bs, heads, -1).transpose(1, 2).flatten(-2)
        at += n
    return pool


def _pool16(gen, blocks, heads, bs, dim, dtype):
    return _rows_like_keys(gen, blocks * bs, heads, dim, dtype).view(blocks, bs, heads, dim)


def _lengths(gen, n, lo, hi):
    """n lengths spread over [lo, hi]: the same ones for every seed, so that outputs keep their sizes, in another order."""
    return torch.linspace(hi, lo, n, device="cuda").round().long()[torch.randperm(n, generator=gen, device="cuda")]


def _tables(gen, lens, bs, longest):
    """Pages of every request out of a shuffled pool, -1 behind the last, and the pool's number of pages."""
    width = -(-longest // bs)
    pages = (lens + bs - 1) // bs
    total = int(pages.sum())
    blocks = total + total // 16 + 1
    perm = torch.randperm(blocks, generator=gen, device="cuda")
    start = pages.cumsum(0) - pages
    column = torch.arange(width, device="cuda")
    held = column < pages[:, None]
    return torch.where(held, perm[(start[:, None] + column).clamp(max=blocks - 1)], -1), blocks


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    op, bs, dim, heads, dtype = case["op"], case["bs"], case["dim"], case["kv_heads"], DTYPES[case["dtype"]]
    state = dict(case)
    if op == "write":
        n = case["tokens"]
        blocks = -(-n // bs) + 8
        state["key_cache"] = torch.zeros(blocks, heads, _page_bytes(bs, dim), dtype=torch.uint8, device="cuda")
        state["value_cache"] = torch.zeros_like(state["key_cache"])
        state["slots"] = torch.randperm(blocks * bs, generator=gen, device="cuda")[:n].contiguous()
        state["key"] = _rows_like_keys(gen, n, heads, dim, dtype)
        state["value"] = _randn(gen, n, heads, dim, dtype=dtype)
        return state
    if op == "prefill":
        n = case["requests"]
        new = _lengths(gen, n, case["new_lo"], case["new_hi"])
        past = torch.randint(0, case["past"] + 1, (n,), generator=gen, device="cuda") // bs * bs
        lens = past + new
        state["cu"] = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)))
        state["starts"], state["lens"] = past, lens
        state["longest_new"] = case["new_hi"]
        state["tables"], blocks = _tables(gen, lens, bs, case["past"] + case["new_hi"])
        state["query"] = _randn(gen, int(new.sum()), case["q_heads"], dim, dtype=dtype)
        state["key_cache"], state["value_cache"] = (_int4_pool(gen, blocks, heads, bs, dim) for _ in range(2))
        return state
    lens = _lengths(gen, case["batch"], case["lo"], case["hi"])
    state["lens"] = lens
    state["tables"], blocks = _tables(gen, lens, bs, case["hi"])
    if op == "bounds":
        state["starts"] = lens - case["new"]
        state["key_cache"] = (_int4_pool(gen, blocks, heads, bs, dim) if case["pool"] == "int4"
                              else _pool16(gen, blocks, heads, bs, dim, dtype))
        state["bounds"] = torch.zeros(blocks, heads, 2 * dim + 16, dtype=torch.uint8, device="cuda")
        width = state["tables"].shape[1]
        column = torch.arange(width, device="cuda")
        touched = (column >= (state["starts"] // bs)[:, None]) & (column < ((lens + bs - 1) // bs)[:, None])
        state["touched"] = state["tables"][touched].contiguous()  # the pages whose bounds the pass returns
        return state
    state["query"] = _randn(gen, case["batch"], case["q_heads"], dim, dtype=dtype)
    if op == "select":
        middle = _randn(gen, 1, heads, dim)
        high = middle + _randn(gen, blocks, heads, dim).abs() * 0.5 + 1.0
        low = middle - _randn(gen, blocks, heads, dim).abs() * 0.5 - 1.0
        state["bounds"] = _pack_bounds(low, high)
        return state
    if case.get("pool") == "16bit":
        state["key_cache"], state["value_cache"] = (_pool16(gen, blocks, heads, bs, dim, dtype) for _ in range(2))
    else:
        state["key_cache"], state["value_cache"] = (_int4_pool(gen, blocks, heads, bs, dim) for _ in range(2))
    if op == "attend":  # blocks as select_blocks gives them: ascending, -1 behind the last
        take, width = case["take"], state["tables"].shape[1]
        pages = ((lens + bs - 1) // bs)[:, None, None]
        score = torch.rand(case["batch"], heads, width, generator=gen, device="cuda")
        column = torch.arange(width, device="cuda")
        score = score.masked_fill(column == pages - 1, 2.0).masked_fill(column >= pages, -1.0)
        kept, at = score.sort(-1, descending=True)
        at = at.masked_fill(kept < 0, width)[..., :take].sort(-1).values
        selected = torch.full((case["batch"], heads, take), -1, dtype=torch.int64, device="cuda")
        selected[..., : at.shape[-1]] = at.masked_fill(at == width, -1)
        state["selected"] = selected
    return state


# ------------------------------------------------------------------ one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from myvllm_mini_engine_b200 import kernels as k

    op, bs = s["op"], s["bs"]
    if op == "write":
        k.write_kv_cache_slots_int4(s["key_cache"], s["value_cache"], s["slots"], s["key"], s["value"], bs, validate=False)
        return k.read_kv_cache_slots_int4(s["key_cache"], s["value_cache"], s["slots"], bs, s["dim"], dtype=s["key"].dtype,
                                          validate=False)
    if op == "decode":
        return k.paged_attention_int4(s["query"], s["key_cache"], s["value_cache"], s["tables"], s["lens"], bs, validate=False)
    if op == "prefill":
        return k.paged_prefill_attention_int4(s["query"], s["key_cache"], s["value_cache"], s["cu"], s["starts"], s["tables"],
                                              s["lens"], bs, validate=False, max_query_len=s["longest_new"])
    if op == "bounds":
        k.update_block_bounds(s["bounds"], s["key_cache"], s["tables"], s["starts"], s["lens"], bs, validate=False,
                              max_query_len=s["new"])
        return k.read_block_bounds(s["bounds"], s["touched"], validate=False)
    if op == "select":
        return k.select_blocks(s["query"], s["bounds"], s["tables"], s["lens"], bs, s["take"], validate=False)
    if s["pool"] == "int4":
        return k.paged_attention_int4(s["query"], s["key_cache"], s["value_cache"], s["tables"], s["lens"], bs,
                                      selected=s["selected"], validate=False)
    return k.paged_attention_selected(s["query"], s["key_cache"], s["value_cache"], s["tables"], s["lens"], s["selected"], bs,
                                      validate=False)


def _attention(q, keys, values, keep):
    """Softmax attention ``[..., queries, keys]`` in the arguments' precision; a row that keeps no key gives zeros."""
    score = (q @ keys.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    score = score.masked_fill(~keep, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    return (weight @ values) / weight.sum(-1, keepdim=True).clamp(min=1e-300 if q.dtype == torch.float64 else 1e-30)


def _run_plain(s):
    return globals()["_plain_" + s["op"]](s)


def _plain_write(s):
    bs, dim, out = s["bs"], s["dim"], []
    page, at = s["slots"] // bs, s["slots"] % bs
    head = torch.arange(s["kv_heads"], device="cuda")
    for cache, x in ((s["key_cache"], s["key"]), (s["value_cache"], s["value"])):
        rows, pairs = _pack_rows(*_quantize(x))
        for size, first, data in ((dim // 2, 0, rows), (4, bs * dim // 2, pairs)):
            byte = first + at[:, None] * size + torch.arange(size, device="cuda")
            cache[page[:, None, None], head[:, None], byte[:, None, :]] = data
        pages = [cache[page[:, None, None], head[:, None], (first + at[:, None] * size + torch.arange(size, device="cuda"))[:, None, :]]
                 for size, first in ((dim // 2, 0), (4, bs * dim // 2))]
        out.append(_values(torch.cat(pages, -1), 1, dim)[..., 0, :].to(x.dtype))
    return tuple(out)


def _plain_decode(s):
    bs, dim, heads = s["bs"], s["dim"], s["kv_heads"]
    tables = s["tables"].clamp(min=0)
    keys, values = (_values(s[name][tables].transpose(1, 2), bs, dim).flatten(2, 3) for name in ("key_cache", "value_cache"))
    keep = torch.arange(keys.shape[2], device="cuda") < s["lens"][:, None]
    q = s["query"].float().unflatten(1, (heads, -1))
    return _attention(q, keys, values, keep[:, None, None]).flatten(1, 2).to(s["query"].dtype)


def _plain_prefill(s):
    bs, dim, heads, longest = s["bs"], s["dim"], s["kv_heads"], s["longest_new"]
    tables = s["tables"].clamp(min=0)
    keys, values = (_values(s[name][tables].transpose(1, 2), bs, dim).flatten(2, 3) for name in ("key_cache", "value_cache"))
    at = torch.arange(longest, device="cuda")
    row = s["cu"][:-1, None] + at
    real = row < s["cu"][1:, None]
    q = s["query"].float()[row.clamp(max=s["query"].shape[0] - 1)].unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4)
    keep = torch.arange(keys.shape[2], device="cuda") <= (s["starts"][:, None] + at)[..., None]
    out = _attention(q, keys[:, :, None], values[:, :, None], keep[:, None, None])
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[real].to(s["query"].dtype)


def _touched_rows(s):
    """For the touched pages, in order: how many rows of each are written."""
    bs, width = s["bs"], s["tables"].shape[1]
    column = torch.arange(width, device="cuda")
    touched = (column >= (s["starts"] // bs)[:, None]) & (column < ((s["lens"] + bs - 1) // bs)[:, None])
    return (s["lens"][:, None] - column * bs).clamp(max=bs)[touched]


def _page_keys(s, wide):
    if s["pool"] == "int4":
        return _values(s["key_cache"][s["touched"]], s["bs"], s["dim"], wide)
    return s["key_cache"][s["touched"]].to(wide).transpose(1, 2)


def _plain_bounds(s):
    keys = _page_keys(s, torch.float32).nan_to_num(nan=0.0, posinf=F32_MAX, neginf=-F32_MAX)
    keep = (torch.arange(s["bs"], device="cuda") < _touched_rows(s)[:, None])[:, None, :, None]
    low, high = keys.masked_fill(~keep, math.inf).amin(2), keys.masked_fill(~keep, -math.inf).amax(2)
    records = _pack_bounds(low, high)
    s["bounds"][s["touched"]] = records
    up, down = (records[..., i * s["dim"]:(i + 1) * s["dim"]].view(torch.int8).float() for i in range(2))
    scale = records[..., 2 * s["dim"]: 2 * s["dim"] + 4].contiguous().view(torch.float32)
    return down * scale, up * scale


def _plain_select(s):
    bs, dim, heads, take = s["bs"], s["dim"], s["kv_heads"], s["take"]
    q = s["query"].float().unflatten(1, (heads, -1))
    parts = torch.cat((q.clamp(min=0.0), q.clamp(max=0.0)), -1)
    total = parts[:, :, 0]
    for h in range(1, parts.shape[2]):  # in the order of the heads: a sum of 32-bit numbers has one value only so
        total = total + parts[:, :, h]
    top = total.abs().amax(-1, keepdim=True)
    codes = torch.round(total * torch.where(top < 2.0 ** -100, torch.zeros_like(top), _over(127.0, top))).clamp(-127.0, 127.0)
    pages = ((s["lens"] + bs - 1) // bs)[:, None, None]
    width = s["tables"].shape[1]
    records = s["bounds"][s["tables"].clamp(min=0)]
    bound = records[..., : 2 * dim].view(torch.int8).float()
    scale = records[..., 2 * dim: 2 * dim + 4].contiguous().view(torch.float32)[..., 0]
    # below 2^24: exact in any order.  The maximum meets the positive parts, the minimum the negative ones.
    score = (torch.einsum("bwhd,bhd->bhw", bound, codes) * scale.transpose(1, 2)) + 0.0
    column = torch.arange(width, device="cuda")
    score = score.masked_fill((column < 1) | (column == pages - 1), math.inf)
    score = score.masked_fill(column >= pages, -math.inf)
    at = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :take]
    at = at.masked_fill(at >= pages, width).sort(-1).values
    selected = torch.full((*at.shape[:2], take), -1, dtype=torch.int64, device="cuda")
    selected[..., : at.shape[-1]] = at.masked_fill(at == width, -1)
    return selected


def _chosen(s, wide):
    """Keys and values ``[batch, kv_heads, rows, dim]`` of the selected blocks, and which rows are kept."""
    bs, dim, heads = s["bs"], s["dim"], s["kv_heads"]
    chosen = s["selected"]
    page = s["tables"].gather(1, chosen.clamp(min=0).flatten(1)).view_as(chosen).clamp(min=0)
    head = torch.arange(heads, device="cuda")[None, :, None]
    off = torch.arange(bs, device="cuda")
    keep = (chosen[..., None] >= 0) & (chosen[..., None] * bs + off < s["lens"][:, None, None, None])
    if s["pool"] == "int4":
        kv = [_values(s[name][page, head], bs, dim, wide) for name in ("key_cache", "value_cache")]
    else:
        kv = [s[name][page[..., None], off, head[..., None]].to(wide) for name in ("key_cache", "value_cache")]
    return kv[0].flatten(2, 3), kv[1].flatten(2, 3), keep.flatten(2, 3)


def _plain_attend(s):
    keys, values, keep = _chosen(s, torch.float32)
    q = s["query"].float().unflatten(1, (s["kv_heads"], -1))
    return _attention(q, keys, values, keep[:, :, None]).flatten(1, 2).to(s["query"].dtype)


# ------------------------------------------------------------------ 64 bits

def _exact_rows(x):
    """Values in 64 bits that the quantised rows stand for."""
    x = x.double()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    base, step = low.half().double(), ((high - low) / 15.0).clamp(min=STEP_MIN).half().double()
    return base + step * torch.round((x - base) / step).clamp(0, 15)


def exact(case, seed):
    s = prepare(case, seed)
    op, bs, dim, heads, wide = s["op"], s["bs"], s["dim"], s["kv_heads"], torch.float64
    if op == "write":
        return _exact_rows(s["key"]), _exact_rows(s["value"])
    if op == "select":
        return None
    if op == "bounds":
        keys, rows, found = _page_keys(s, wide), _touched_rows(s).tolist(), [[], []]
        for i, n in enumerate(rows):
            low, high = keys[i, :, :n].amin(1), keys[i, :, :n].amax(1)
            top = torch.maximum(low.abs(), high.abs()).amax(-1, keepdim=True)
            found[0].append(torch.floor(low * 127.0 / top) * top / 127.0)
            found[1].append(torch.ceil(high * 127.0 / top) * top / 127.0)
        return tuple(torch.stack(f) for f in found)
    out = []
    for b, length in enumerate(s["lens"].tolist()):
        table = s["tables"][b, : -(-length // bs)]
        if op == "prefill":
            q = s["query"][int(s["cu"][b]): int(s["cu"][b + 1])].double().unflatten(1, (heads, -1)).permute(1, 2, 0, 3)
            last = int(s["starts"][b]) + torch.arange(q.shape[2], device="cuda")
        else:
            q = s["query"][b].double().unflatten(0, (heads, -1))[:, :, None]
            last = torch.full((1,), length - 1, device="cuda")
        each = []
        for h in range(heads):
            pages, position = table, torch.arange(len(table) * bs, device="cuda")
            if op == "attend":
                chosen = s["selected"][b, h]
                chosen = chosen[chosen >= 0]
                pages = table[chosen]
                position = (chosen[:, None] * bs + torch.arange(bs, device="cuda")).flatten()
            if s.get("pool") == "16bit":
                k, v = (s[name][pages, :, h].double().flatten(0, 1) for name in ("key_cache", "value_cache"))
            else:
                k, v = (_values(s[name][pages, h], bs, dim, wide).flatten(0, 1) for name in ("key_cache", "value_cache"))
            weight = torch.einsum("gqd,td->gqt", q[h], k) / math.sqrt(dim)
            weight = weight.masked_fill(position > last[:, None], -math.inf).softmax(-1)
            each.append(torch.einsum("gqt,td->gqd", weight, v))
        out.append(torch.stack(each).flatten(0, 1).transpose(0, 1))
    return torch.cat(out)


# ------------------------------------------------------------------ work

def work(case):
    """Bytes and operations of one pass; ragged lengths count at their mean."""
    op, bs, dim, heads = case["op"], case["bs"], case["dim"], case["kv_heads"]
    size = 2
    row4 = heads * (dim // 2 + 4)
    if op == "write":
        n = case["tokens"]
        return {"bytes": n * (2 * heads * dim * size * 2 + 2 * row4 + 16), "flops": n * heads * dim * 2 * 6}
    if op == "prefill":
        n, new, past = case["requests"], (case["new_lo"] + case["new_hi"]) / 2, case["past"] / 2
        pairs = n * new * (past + (new + 1) / 2)
        return {"bytes": n * ((past + new) * 2 * row4 + 2 * new * case["q_heads"] * dim * size),
                "flops": 4 * pairs * case["q_heads"] * dim}
    mean, n = (case["lo"] + case["hi"]) / 2, case["batch"]
    if op == "bounds":
        touched = case["new"] / bs + 1
        row = heads * dim * size if case["pool"] == "16bit" else row4
        rows = min(mean, case["new"] + bs / 2)
        return {"bytes": n * (rows * row + touched * heads * (2 * dim + 4 + 2 * dim * 4)), "flops": n * rows * heads * dim * 2}
    io = 2 * n * case["q_heads"] * dim * size
    if op == "select":
        pages = n * mean / bs
        return {"bytes": pages * (heads * (2 * dim + 4) + 8) + io / 2 + n * heads * case["take"] * 8,
                "flops": pages * heads * 2 * dim * 2}
    rows = n * (mean if op == "decode" else min(mean, case["take"] * bs))
    row = heads * dim * size if case.get("pool") == "16bit" else row4
    return {"bytes": rows * 2 * row + io, "flops": 4 * rows * case["q_heads"] * dim}
