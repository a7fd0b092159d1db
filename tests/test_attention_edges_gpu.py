"""The attention side where values, lengths and launches are at their edges.

Tolerances are those of tests/test_attention_gpu.py and tests/test_norm_rope_gpu.py; what has to be
the same row in another call is compared bit by bit."""
from __future__ import annotations

import pytest
import torch

from test_attention_gpu import Batch

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")

# decoding whose units are cut over the warps of the GPU: one unit and two (32 warps join a row, in
# halves and whole), some hundred (4 warps), and more units than warps
CUT = [([(1, 20000)], 8, 1), ([(1, 3000), (1, 9000)], 8, 8), ([(4, 6000 + 500 * b) for b in range(8)], 8, 2),
       ([(1, 2000 + 37 * b) for b in range(50)], 4, 2), ([(1, 300 + (37 * b) % 600) for b in range(700)], 4, 2)]


@pytest.mark.parametrize("lens,heads,kv_heads", CUT)
@pytest.mark.parametrize("dim", [64, 128])
def test_not_a_number_of_a_query_outlives_the_join(cuda, lens, heads, kv_heads, dim):
    b = Batch(lens, heads, kv_heads, dim, 64, seed=51)
    want, want_lse = b.run()
    b.q[::7, 1, 5] = NAN
    got, lse = b.run()
    assert torch.isnan(got[::7, 1]).all() and torch.isnan(lse[::7, 1]).all()
    got[::7, 1], lse[::7, 1] = want[::7, 1], want_lse[::7, 1]
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("lens,heads,kv_heads", CUT[:4])
def test_not_a_number_of_many_keys_outlives_the_join(cuda, lens, heads, kv_heads):
    """Whole fragments whose scores are all NaN, beside others that are finite.  (The first sequence's
    ranges begin 32 keys behind a multiple of 64, a unit's cost before them: none is NaN in part.)"""
    b = Batch(lens, heads, kv_heads, 128, 32, seed=52, causal=False)
    want, want_lse = b.run()
    for page in range(11, 41):
        b.k_cache[b.table[0, page], 0] = NAN
    got, lse = b.run()
    rows, group = lens[0][0], heads // kv_heads
    assert torch.isnan(got[:rows, :group]).all() and torch.isnan(lse[:rows, :group]).all()
    got[:rows, :group], lse[:rows, :group] = want[:rows, :group], want_lse[:rows, :group]
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
