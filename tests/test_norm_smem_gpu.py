"""Norms of rows whose weights take all the shared memory that a launch has without asking for more."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [5888, 6001, 6144, 6152, 11784, 12288, 12289])
@pytest.mark.parametrize("tokens", [2, 150, 900])
def test_rows_of_48_kilobytes_of_weights(cuda, d, tokens):
    from freemoe_b200 import attention

    g = torch.Generator(device="cuda").manual_seed(d)
    x, res = (torch.randn(tokens, d, generator=g, device="cuda") for _ in range(2))
    w1, w2 = (torch.randn(d, generator=g, device="cuda") for _ in range(2))

    def norm(v, w):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w.double()

    # E = 2^-24.  A sum of d squares is off by 44 E (32 values in turn, then a tree), half of it in the root;
    # the root, the division and the products add 5 E
    near = dict(rtol=64 * 2.0 ** -24, atol=64 * 2.0 ** -24)
    y, h = attention.add_rms_norm(x, w1, residual=res)
    torch.testing.assert_close(h, x + res, rtol=0, atol=0)
    torch.testing.assert_close(y.double(), norm(h.double(), w1), **near)
    y, h = attention.norm_add_norm(x, w1, res, w2)
    # the normed x is off by 35 E, h by 2 E more of both terms; y by 40 E of its own, by what h is off, and
    # by the root's share, at most 37 E sqrt(sum size^2 / sum h^2), a factor of 1.3 here
    want = res.double() + norm(x.double(), w1)
    size = (res.abs() + (want - res).abs()).double()
    assert ((h - want).abs() <= 64 * 2.0 ** -24 * size).all()
    off = (y - norm(want, w2)).abs()
    scale = w2.abs().double() * size / torch.sqrt((want * want).mean(-1, keepdim=True))
    assert (off <= 128 * 2.0 ** -24 * (scale + norm(want, w2).abs())).all()
