"""Refusals of the 4-bit pool's and the block selection's operators (no GPU), and the oracle's own checks."""

import ctypes

import numpy as np
import pytest
import torch

from myvllm_mini_engine_b200 import _lib, kernels as k
from oracle import block_select, int4_kv

BS, HKV, DIM = 16, 2, 64


def pools(blocks=4, dim=DIM, bs=BS, heads=HKV):
    return tuple(torch.zeros(blocks, heads, k.int4_page_bytes(bs, dim), dtype=torch.uint8) for _ in range(2))


def rows(tokens=3, heads=HKV, dim=DIM, dtype=torch.bfloat16):
    return torch.zeros(tokens, heads, dim, dtype=dtype)


def test_page_bytes_agree_and_refuse_other_shapes():
    lib = _lib.load()
    for bs in (1, 3, 5, 16, 24, 256):
        for dim in (32, 64, 96, 128, 192, 256):
            assert k.int4_page_bytes(bs, dim) == lib.minikv_int4_page_bytes(bs, dim) == int4_kv.page_bytes(bs, dim)
    assert k.int4_page_bytes(16, 128) == 16 * 68
    for bs, dim in ((16, 80), (16, 16), (0, 64), (-1, 64), (16, 512)):
        with pytest.raises(ValueError):
            k.int4_page_bytes(bs, dim)
        assert lib.minikv_int4_page_bytes(bs, dim) == -1


def bad_writes():
    kc, vc = pools()
    key, slots = rows(), torch.arange(3)
    return {
        "backend": ((kc, vc, slots, key, key, BS), {"backend": "torch"}, "backend"),
        "page bytes": ((kc, vc, slots, key, key, 8), {}, "block size"),
        "block size type": ((kc, vc, slots, key, key, 16.0), {}, "block size"),
        "head dim": ((kc, vc, slots, rows(dim=80), rows(dim=80), BS), {}, "head_dim"),
        "heads": ((kc, vc, slots, rows(heads=3), rows(heads=3), BS), {}, "matching the cache"),
        "pool dtype": ((kc.float(), vc.float(), slots, key, key, BS), {}, "uint8"),
        "pool stride": ((kc[:, :, ::2], vc[:, :, ::2], slots, key, key, BS), {}, "contiguous"),
        "row dtype": ((kc, vc, slots, key.double(), key.double(), BS), {}, "FP32/FP16/BF16"),
        "mixed dtype": ((kc, vc, slots, key, key.float(), BS), {}, "FP32/FP16/BF16"),
        "slots dtype": ((kc, vc, slots.int(), key, key, BS), {}, "int64"),
        "slots count": ((kc, vc, torch.arange(2), key, key, BS), {}, "int64"),
        "slot range": ((kc, vc, torch.tensor([0, 1, 64]), key, key, BS), {}, "capacity"),
        "slot twice": ((kc, vc, torch.tensor([0, 1, 0]), key, key, BS), {}, "duplicate"),
        "same pool": ((kc, kc, slots, key, key, BS), {}, "overlap"),
        "cpu": ((kc, vc, slots, key, key, BS), {}, "CUDA"),
    }


@pytest.mark.parametrize("name", list(bad_writes()))
def test_slot_writes_refuse(name):
    args, kwargs, message = bad_writes()[name]
    with pytest.raises(ValueError, match=message):
        k.write_kv_cache_slots_int4(*args, **kwargs)


def test_batch_writes_and_reads_refuse():
    kc, vc = pools()
    key, offsets, tables = rows(), torch.tensor([0, 5, 20]), torch.tensor([[0, 1], [2, 3], [1, 0]])
    for bad, message in (((tables, torch.tensor([0, 5, 32])), "offset"), ((tables, torch.tensor([0, 5, -1])), "offset"),
                         ((tables + 2, offsets), "physical block"), ((torch.zeros_like(tables), torch.tensor([3, 3, 1])), "duplicate"),
                         ((tables.int(), offsets), "int64"), ((tables[:2], offsets), "int64"), ((tables, offsets), "CUDA")):
        with pytest.raises(ValueError, match=message):
            k.write_kv_cache_batch_int4(kc, vc, *bad, key, key, BS)
    with pytest.raises(ValueError, match="capacity"):
        k.read_kv_cache_slots_int4(kc, vc, torch.tensor([64]), BS, DIM)
    with pytest.raises(ValueError, match="FP32"):
        k.read_kv_cache_slots_int4(kc, vc, torch.tensor([0]), BS, DIM, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        k.read_kv_cache_slots_int4(kc, vc, torch.tensor([0]), BS, DIM)


def test_prefill_refuses():
    kc, vc = pools()
    q = torch.zeros(5, 4, DIM, dtype=torch.bfloat16)
    meta = [torch.tensor([0, 5]), torch.tensor([0]), torch.tensor([[0, 1]]), torch.tensor([5])]

    def call(q=q, pool=(kc, vc), bs=BS, **change):
        m = list(meta)
        for i, value in change.items():
            m[int(i[1:])] = value
        return k.paged_prefill_attention_int4(q, *pool, *m, bs)

    for kwargs, message in (({"q": q.float()}, "FP16/BF16"), ({"q": q[:, :3]}, "GQA"), ({"q": q[0]}, "heads"),
                            ({"bs": 8}, "block size"), ({"m0": torch.tensor([0, 4])}, "monotone"),
                            ({"m1": torch.tensor([1])}, "query start"), ({"m2": torch.tensor([[7, 1]])}, "physical page"),
                            ({"m3": torch.tensor([5], dtype=torch.int32)}, "int64"), ({"m3": torch.tensor([5, 5])}, "request count"),
                            ({}, "CUDA")):
        with pytest.raises(ValueError, match=message):
            call(**kwargs)


def test_decodes_and_selection_need_cuda_tensors_and_known_backends():
    kc, vc = pools()
    q, tables, lens = torch.zeros(1, 4, DIM, dtype=torch.bfloat16), torch.tensor([[0, 1]]), torch.tensor([5])
    bounds = torch.zeros(4, HKV, k.block_bounds_bytes(DIM), dtype=torch.uint8)
    wide = torch.zeros(4, BS, HKV, DIM, dtype=torch.bfloat16)
    selected = torch.zeros(1, HKV, 1, dtype=torch.int64)
    calls = {
        "decode": lambda **kw: k.paged_attention_int4(q, kc, vc, tables, lens, BS, **kw),
        "attend": lambda **kw: k.paged_attention_selected(q, wide, wide, tables, lens, selected, BS, **kw),
        "select": lambda **kw: k.select_blocks(q, bounds, tables, lens, BS, 4, **kw),
        "bounds": lambda **kw: k.update_block_bounds(bounds, wide, tables, torch.tensor([0]), lens, BS, **kw),
    }
    for call in calls.values():
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
        with pytest.raises(ValueError, match="backend"):
            call(backend="torch")
    with pytest.raises(RuntimeError, match="CUDA"):
        k.read_block_bounds(bounds, torch.tensor([0]))
    with pytest.raises(ValueError, match="head_dim"):
        k.block_bounds_bytes(80)
    for bad in (bounds[:, :, :-1].contiguous(), bounds.int(), bounds[:, :, ::2]):
        with pytest.raises(RuntimeError, match="bounds"):
            k.read_block_bounds(bad, torch.tensor([0]))
    with pytest.raises(RuntimeError, match="matching the bounds"):
        k.update_block_bounds(bounds, wide[:, :8].contiguous(), tables, torch.tensor([0]), lens, BS)
    with pytest.raises(RuntimeError, match="matching the bounds"):
        k.update_block_bounds(bounds, kc, tables, torch.tensor([0]), lens, 8)


def test_c_entry_points_refuse():
    """Codes and messages, never an exception or an abort; null pointers and bad sizes reach no launch."""
    lib, p = _lib.load(), ctypes.c_void_p(16)

    def refused(rc, word):
        assert rc == _lib.EINVAL and word in lib.minikv_last_error().decode(), lib.minikv_last_error()

    decode = [p] * 8 + [p, 1 << 30]
    for entry in (lib.minikv_paged_decode_int4, lib.minikv_paged_decode_selected):
        refused(entry(*decode, 2, 6, 4, 64, 10, 16, 4, 2, _lib.BF16, None), "GQA")
        refused(entry(*decode, 2, 8, 4, 80, 10, 16, 4, 2, _lib.BF16, None), "head_dim")
        refused(entry(*decode, 2, 8, 4, 64, 10, 16, 1 << 17, 2, _lib.BF16, None), "1M tokens")
        refused(entry(*decode, 2, 8, 4, 64, 10, 16, 4, 0, _lib.BF16, None), "selected")
        refused(entry(*decode, 2, 8, 4, 64, 10, 16, 4, 1 << 20, _lib.BF16, None), "selected")
        refused(entry(*decode, 0, 8, 4, 64, 10, 16, 4, 2, _lib.BF16, None), "empty")
        refused(entry(*decode, 2, 8, 4, 64, 10, 16, 4, 2, _lib.F32, None), "FP16/BF16")
        refused(entry(*decode, 2, 8, 4, 64, 1 << 31, 16, 4, 2, _lib.BF16, None), "2^31")
        refused(entry(None, *decode[1:], 2, 8, 4, 64, 10, 16, 4, 2, _lib.BF16, None), "null")
        refused(entry(ctypes.c_void_p(8), *decode[1:], 2, 8, 4, 64, 10, 16, 4, 2, _lib.BF16, None), "aligned")
        refused(entry(*decode[:9], 16, 2, 8, 4, 64, 10, 16, 4, 2, _lib.BF16, None), "workspace")
    refused(lib.minikv_paged_decode_selected(*decode[:5], None, *decode[6:], 2, 8, 4, 64, 10, 16, 4, 2, _lib.BF16, None), "null")
    assert lib.minikv_paged_decode_int4_workspace_bytes(2, 8, 4, 64, 10, 16, 4, _lib.BF16) > 0
    assert lib.minikv_paged_decode_selected_workspace_bytes(2, 8, 4, 80, 10, 16, 4, _lib.BF16) == -1
    refused(lib.minikv_kv_scatter_slots_int4(p, p, p, p, p, 3, 8, 16, 2, 64, 127, 128, _lib.BF16, None), "stride")
    refused(lib.minikv_kv_scatter_slots_int4(p, p, p, p, p, 3, 8, 16, 2, 64, 128, 128, 5, None), "FP32")
    refused(lib.minikv_kv_scatter_slots_int4(p, p, None, p, p, 3, 8, 16, 2, 64, 128, 128, _lib.BF16, None), "null")
    refused(lib.minikv_kv_append_batch_int4(p, p, p, None, p, p, 3, 2, 8, 16, 2, 64, 128, 128, _lib.BF16, None), "null")
    refused(lib.minikv_kv_gather_slots_int4(p, p, p, p, None, 3, 8, 16, 2, 64, _lib.BF16, None), "null")
    for rc in (lib.minikv_kv_scatter_slots_int4(*[None] * 5, 0, 8, 16, 2, 64, 128, 128, _lib.BF16, None),
               lib.minikv_kv_append_batch_int4(*[None] * 6, 0, 2, 8, 16, 2, 64, 128, 128, _lib.BF16, None),
               lib.minikv_kv_gather_slots_int4(*[None] * 5, 0, 8, 16, 2, 64, _lib.BF16, None),
               lib.minikv_paged_prefill_int4(*[None] * 9, 0, 0, 1, 4, 2, 64, 8, 16, 4, 1, _lib.BF16, None),
               lib.minikv_block_bounds_update(*[None] * 5, 0, 4, 8, 16, 2, 64, 1, _lib.BF16, None),
               lib.minikv_block_bounds_read(None, None, 0, None, None, 8, 2, 64, None)):
        assert rc == _lib.OK  # empty calls touch nothing
    refused(lib.minikv_paged_prefill_int4(*[p] * 9, 0, 5, 70000, 4, 2, 64, 8, 16, 4, 1, _lib.BF16, None), "requests")
    assert lib.minikv_paged_prefill_int4(*[p] * 9, 0, 5, 1, 65, 1, 64, 8, 16, 4, 1, _lib.BF16, None) == _lib.EUNSUPPORTED
    refused(lib.minikv_block_bounds_update(*[p] * 5, 1, 4, 8, 16, 2, 64, 1, 7, None), "4-bit")
    select = [p] * 6 + [1 << 20]
    refused(lib.minikv_select_blocks(*select, 2, 8, 4, 64, 10, 16, 4, 3, 2, 2, _lib.BF16, None), "max_blocks")
    refused(lib.minikv_select_blocks(*select, 2, 8, 4, 64, 10, 16, 4, 0, 0, 0, _lib.BF16, None), "max_blocks")
    refused(lib.minikv_select_blocks(*select, 2, 8, 4, 64, 10, 16, 4, 3, 1, 1, 9, None), "FP32")
    refused(lib.minikv_select_blocks(*select[:6], 4, 2, 8, 4, 64, 10, 16, 4, 3, 1, 1, _lib.BF16, None), "workspace")


def test_oracle_round_trip():
    """Values lie within half a step of the inputs (plus the pair's own fp16 rounding)."""
    gen = np.random.default_rng(0)
    x = torch.from_numpy(gen.standard_normal((32, 2, 64), dtype=np.float32))
    pool = np.zeros((2, 2, int4_kv.page_bytes(16, 64)), dtype=np.uint8)
    int4_kv.scatter(pool, 16, torch.arange(32), x)
    back = int4_kv.values(pool, 16, 64).reshape(32, 2, 64)
    spread = x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)
    # half a step; the base is off by half a step of fp16, the step by 2^-11 of itself, at most 15 times
    bound = spread / 30 + x.abs().amax() * 2.0 ** -11 + spread * 2.0 ** -11
    assert bool(((back - x.double()).abs() <= bound).all())


def test_oracle_scores_bound_the_products():
    gen = np.random.default_rng(1)
    keys = torch.from_numpy(gen.standard_normal((16, 64)))
    query = torch.from_numpy(gen.standard_normal((3, 64), dtype=np.float32))
    rec = block_select.record(keys.numpy())
    lower, upper = block_select.read(rec[None, None], [0], 64)
    pos, neg = query.clamp(min=0).sum(0).double(), query.clamp(max=0).sum(0).double()
    bound = float((upper[0, 0].double() * pos + lower[0, 0].double() * neg).sum())
    assert bound >= float((keys @ query.double().T).sum(1).max()) - 1e-5
    codes = block_select.query_codes(query)
    assert codes.shape == (128,) and int(np.abs(codes).max()) == 127


def test_overlap_is_of_bytes_not_of_storages():
    from myvllm_mini_engine_b200.kernels.int4 import _overlaps

    both = torch.zeros(2, 64, dtype=torch.uint8)
    other = torch.zeros(4, 2, 8, dtype=torch.bfloat16)
    assert not _overlaps((both[0], both[1]), (other, other[:, 1]))
    assert _overlaps((both[0], both.view(-1)[63:]), (other,))
    assert not _overlaps((both[0], both[1]), (both[1, :0],))
    halves = torch.zeros(4, 2, 8, dtype=torch.bfloat16).view(torch.uint8)
    for i in range(2):  # a source that lies in either cache, strided too
        caches = [both[0], both[1]]
        caches[i] = halves.view(-1)[:64]
        assert _overlaps(caches, (halves.view(torch.bfloat16)[1:, 1],))


def test_pools_check_their_arguments():
    from myvllm_mini_engine_b200.cache import INT4KVCachePool, PagedKVPool

    with pytest.raises(ValueError, match="head_dim"):
        INT4KVCachePool(1, 4, 16, 2, 80, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        INT4KVCachePool(1, 0, 16, 2, 64, device="cpu")
    pool = INT4KVCachePool(2, 4, 16, 2, 64, device="cpu")
    assert pool.memory_bytes == 2 * 2 * 4 * 2 * 16 * 36 and pool.bounds is None
    one = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="block bounds"):
        pool.update_bounds(0, one[None], one, one)
    with pytest.raises(IndexError, match="layer"):
        pool.write_range(2, [0], 0, rows(), rows())
    with pytest.raises(IndexError, match="block id"):
        pool.write_range(0, [7], 0, rows(), rows())
    with pytest.raises(ValueError, match="capacity"):
        pool.write_range(0, [0], 15, rows(), rows())
    with pytest.raises(ValueError, match="CUDA"):  # no CPU path
        pool.write_slots(0, torch.arange(3), rows(), rows())
    with pytest.raises(ValueError, match="16-bit and 4-bit"):
        PagedKVPool(1, 4, 16, 2, 64, dtype=torch.float32, device="cpu", block_bounds=True)
    with pytest.raises(ValueError, match="head_dim"):
        PagedKVPool(1, 4, 16, 2, 80, device="cpu", block_bounds=True)
    held = PagedKVPool(3, 4, 16, 2, 64, device="cpu", block_bounds=True)
    assert held.bounds.shape == (3, 4, 2, k.block_bounds_bytes(64))


def test_decode_step_checks_its_pool():
    from myvllm_mini_engine_b200.cache import FP8KVCachePool, INT4KVCachePool, PagedKVPool
    from myvllm_mini_engine_b200.engine.qwen3 import Qwen3Config, Qwen3DecodeStep, Qwen3Weights

    cfg = Qwen3Config.qwen3_0_6b(num_hidden_layers=1, vocab_size=64)
    weights = Qwen3Weights.random(cfg, dtype=torch.bfloat16, device="cpu", seed=0)
    shape = (1, 4, 16, cfg.num_key_value_heads, cfg.head_dim)
    for pool in (PagedKVPool(*shape, device="cpu"), INT4KVCachePool(*shape, device="cpu"),
                 FP8KVCachePool(*shape, k_scale=1.0, v_scale=1.0, device="cpu")):
        with pytest.raises(ValueError, match="block bounds"):
            Qwen3DecodeStep(cfg, weights, pool, selected_blocks=4)
    with pytest.raises(ValueError, match="2 blocks"):
        Qwen3DecodeStep(cfg, weights, INT4KVCachePool(*shape, device="cpu", block_bounds=True), selected_blocks=1)


def test_decode_refuses_lists_of_more_tiles_than_it_counts():
    lib = _lib.load()
    for args in ((40000, 1, 1, 32, 1, 1048576, 1), (1, 65535, 65535, 32, 1, 1, 1048576),
                 (16384, 1024, 1, 32, 1, 1048576, 1)):
        for sizer in (lib.minikv_paged_decode_int4_workspace_bytes, lib.minikv_paged_decode_selected_workspace_bytes):
            assert sizer(*args, _lib.BF16) == -1
            assert "too large" in lib.minikv_last_error().decode()
    assert lib.minikv_paged_decode_int4_workspace_bytes(1024, 64, 8, 128, 1 << 20, 16, 65536, _lib.BF16) > 0
