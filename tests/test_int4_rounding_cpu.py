"""What the 4-bit pool promises, as far as it shows without a GPU."""

import pytest

from myvllm_mini_engine_b200 import _lib


@pytest.mark.parametrize("tokens,requests,width", [(1, 1, 1), (2048, 16, 72), (16384, 16, 65536), (200, 16, 65536)])
@pytest.mark.parametrize("dtype", [_lib.F16, _lib.BF16])
def test_a_prefill_takes_no_workspace(tokens, requests, width, dtype):
    """Whatever its table could hold: 16 requests on tables of a million tokens take none."""
    for heads, kv_heads, dim in ((16, 8, 128), (4, 2, 64), (32, 1, 64), (2, 2, 256)):
        size = _lib.load().minikv_paged_prefill_int4_workspace_bytes(tokens, requests, heads, kv_heads, dim, 1 << 20, 16,
                                                                     width, dtype)
        assert size == 0
