"""Attention gives the same bits whatever the calls before it left on the SMs: rows of a tile that no
query has, and keys of a block that are not read, take no part."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len,kv_len,heads,kv_heads,dim,page,window,sinks", [
    (6, 3180, 28, 4, 80, 8, 2442, 216),
    (210, 6923, 16, 16, 128, 8, 2442, 216),
    (300, 9000, 16, 16, 64, 16, 1111, 70),
    (33, 1500, 32, 8, 128, 16, 333, 5),
    (210, 6923, 16, 16, 128, 8, 2442, 0),
    (300, 9000, 16, 16, 64, 16, 1111, 0),
    (75, 2000, 32, 8, 96, 8, 0, 0),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_calls_before_left_behind(cuda, q_len, kv_len, heads, kv_heads, dim, page, window, sinks, dtype):
    from freemoe_b200 import attention

    g = torch.Generator(device="cuda").manual_seed(q_len)
    pages = -(-kv_len // page)
    q = torch.randn(q_len, heads, dim, generator=g, device="cuda").to(dtype)
    caches = [torch.randn(pages, kv_heads, page, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None]
    q_start, length = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, q_len], [kv_len]))

    def call(k, v):
        return attention.paged_attention(q, k, v, table, q_start, length, max_q_len=q_len, max_kv_len=kv_len,
                                         window=window, sinks=sinks)

    outs = []
    for left in (0.0, float("nan"), float("inf"), 1.0):
        filled = torch.full_like(caches[0], left)
        for _ in range(3):
            call(filled, filled)
        outs.append(call(*caches))
    assert torch.isfinite(outs[0].float()).all()
    for out in outs[1:]:
        assert torch.equal(out, outs[0])
