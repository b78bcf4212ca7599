"""Decodes of different batches on one stream share a workspace: none may find another's sums where its counters lie."""

import pytest
import torch

from myvllm_mini_engine_b200.kernels import paged_attention, paged_attention_fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
def test_batches_of_other_sizes_between(cuda_device, fp8):
    gen = torch.Generator("cuda").manual_seed(4)
    heads, kv_heads, dim, bs, blocks = 8, 2, 64, 16, 200

    def pool():
        x = torch.randn(blocks, bs, kv_heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
        return x.to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else x

    k, v = pool(), pool()

    def case(batch, length):
        q = torch.randn(batch, heads, dim, generator=gen, device="cuda").to(torch.bfloat16)
        table = torch.randint(blocks, (batch, length // bs), generator=gen, device="cuda")
        lens = torch.full((batch,), length, device="cuda")
        if fp8:
            return lambda: paged_attention_fp8(q, k, v, table, lens, bs, 1.0, 1.0, validate=False)
        return lambda: paged_attention(q, k, v, table, lens, bs, validate=False)

    # (the counters of 17000 requests do not fit the first 64 KB of a workspace)
    calls = [case(*x) for x in ((128, 2048), (32, 4096), (128, 2048), (512, 1024), (3, 8192), (512, 1024),
                                (17000, 16), (16600, 32), (300, 2048), (17000, 48))]
    # the first answers, each on a stream (and so with a workspace) of its own
    streams, want = [torch.cuda.Stream() for _ in calls], []
    torch.cuda.synchronize()
    for stream, call in zip(streams, calls):
        with torch.cuda.stream(stream):
            want.append(call())
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(3):
            got = [call() for call in calls]
            torch.cuda.synchronize()
            for g, w in zip(got, want):
                assert torch.equal(g, w)
