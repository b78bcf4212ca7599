"""A selection's query codes are scaled by the largest element, whichever lane holds it."""

import numpy as np
import pytest
import torch

from myvllm_mini_engine_b200.kernels import block_bounds_bytes, select_blocks
from oracle import block_select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,heads,kv_heads", [(32, 3, 3), (64, 16, 8), (96, 5, 5), (256, 9, 9)])
def test_the_largest_element_in_any_place(cuda_device, dim, heads, kv_heads):
    gen = np.random.default_rng(dim)
    batch, bs, width, take = dim, 16, 40, 7
    query = torch.from_numpy(gen.uniform(-1, 1, (batch, heads, dim)).astype(np.float32))
    at = torch.arange(batch)
    query[at, :, at] = torch.where(at % 2 == 0, 30.0, -30.0)[:, None]  # request b's largest element is at dim b
    bounds = np.zeros((width, kv_heads, block_bounds_bytes(dim)), dtype=np.uint8)
    for page in range(width):
        for h in range(kv_heads):
            bounds[page, h] = block_select.record(gen.standard_normal((4, dim)))
    table = torch.from_numpy(np.stack([gen.permutation(width) for _ in range(batch)]).astype(np.int64))
    lens = torch.full((batch,), width * bs)
    expected = block_select.select(query, bounds, table, lens, bs, take)
    actual = select_blocks(query.cuda(), torch.from_numpy(bounds).cuda(), table.cuda(), lens.cuda(), bs, take)
    assert torch.equal(actual.cpu(), expected)
