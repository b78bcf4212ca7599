"""What the 4-bit pool promises, as far as it shows without a GPU."""

import numpy as np
import pytest
import torch

from myvllm_mini_engine_b200 import _lib
from oracle import int4_kv


@pytest.mark.parametrize("tokens,requests,width", [(1, 1, 1), (2048, 16, 72), (16384, 16, 65536), (200, 16, 65536)])
@pytest.mark.parametrize("dtype", [_lib.F16, _lib.BF16])
def test_a_prefill_takes_no_workspace(tokens, requests, width, dtype):
    """Whatever its table could hold: 16 requests on tables of a million tokens take none."""
    for heads, kv_heads, dim in ((16, 8, 128), (4, 2, 64), (32, 1, 64), (2, 2, 256)):
        size = _lib.load().minikv_paged_prefill_int4_workspace_bytes(tokens, requests, heads, kv_heads, dim, 1 << 20, 16,
                                                                     width, dtype)
        assert size == 0


def test_the_oracle_reads_rows_at_the_end_of_the_range_back_finite():
    """Rows from -65504, and from values that round up, to 65504; half a step of the value away at most."""
    gen = np.random.default_rng(3)
    x = torch.from_numpy(gen.uniform(-65504, 65504, (400, 64)).astype(np.float32))
    x[:, 1] = 65504.0
    low = torch.from_numpy(gen.uniform(-65504, 65504, 400).astype(np.float32))
    x = torch.maximum(x, low[:, None])  # rows of every width up to the whole range
    x[0, 0], x[1], x[2] = -65504.0, 65504.0, 65489.0
    x[2, 3] = 65504.0
    codes, step, base = (torch.from_numpy(np.asarray(v, dtype=np.float64)) for v in int4_kv.quantize(x))
    back = base[:, None] + step[:, None] * codes
    assert float(back.max()) <= 65504.0 and bool(torch.isfinite(back.half()).all())
    # half a step; base and step were rounded (2^-11 of base, 2^-10 of 15 steps rounded down)
    bound = step / 2 + base.abs() * 2.0 ** -11 + 15 * step * 2.0 ** -10
    assert bool(((back - x.double()).abs() <= bound[:, None]).all())


def test_pools_tell_the_bytes_of_their_bounds():
    from myvllm_mini_engine_b200.cache import INT4KVCachePool, PagedKVPool

    for make, share in ((INT4KVCachePool, 8), (PagedKVPool, 30)):
        plain, held = (make(2, 5, 16, 3, 128, device="cpu", block_bounds=b) for b in (False, True))
        assert plain.bounds_bytes == 0 and held.memory_bytes == plain.memory_bytes
        assert held.bounds_bytes == 2 * 5 * 3 * (2 * 128 + 16) == held.bounds.nbytes
        assert held.memory_bytes // held.bounds_bytes == share


def test_captures_of_two_threads_where_the_kept_counters_end(monkeypatch):
    """A second capture that comes in between the first one's look at what is left and its taking it."""
    import threading

    from myvllm_mini_engine_b200.kernels import int4

    device, count, got = torch.device("cpu", 0), 3, []

    class Kept:
        """Counters for one call more."""

        def __init__(self):
            self.data, self.other = torch.zeros(count, dtype=torch.int32), None

        def numel(self):
            if self.other is None:
                self.other = threading.Thread(target=lambda: got.append(int4._captured_tickets(device, count)))
                self.other.start()
                self.other.join(0.3)
            return self.data.numel()

        def __getitem__(self, part):
            return self.data[part]

    kept = Kept()
    monkeypatch.setattr(int4, "_CAPTURED", {0: [kept, 0]})
    got.append(int4._captured_tickets(device, count))
    kept.other.join(5)
    assert len(got) == 2 and all(t.numel() == count for t in got)
    assert got[0].data_ptr() != got[1].data_ptr()
