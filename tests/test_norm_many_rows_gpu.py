"""Norms of as many rows as a call can have: 2^32 - 1, in teams of four a CTA.

Rows of one value, without epsilon: y = sign(x) w, here +-1.5, and h = r + y.  The root is within 2
units of f32 and the two products within half a unit each, so that y is within 2^-21 of +-1.5 and h of
1.75 and -1, which round to just these in bf16: equal, no tolerance.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS = (1 << 32) - 1
MARKED = [0, 1, 5, (1 << 31) - 1, 1 << 31, ROWS - 5, ROWS - 2, ROWS - 1]


def rows(value, marked):
    x = torch.full((ROWS, 1), value, dtype=torch.bfloat16, device="cuda")
    x[MARKED] = marked
    return x


def hold(got, value, marked):
    at = torch.tensor(MARKED, device="cuda")
    assert (got[at] == marked).all()
    got[at] = value
    for part in got.split(1 << 28):
        assert (part == value).all()


def test_norm(cuda):
    from freemoe_b200 import attention

    x, w = rows(0.5, -2.0), torch.tensor([1.5], device="cuda")
    y, _ = attention.add_rms_norm(x, w, epsilon=0.0)
    hold(y, 1.5, -1.5)


def test_norms_around_a_block(cuda):
    from freemoe_b200 import attention

    x, r, w = rows(0.5, -2.0), rows(0.25, 0.5), torch.tensor([1.5], device="cuda")
    y, h = attention.norm_add_norm(x, w, r, w, epsilon=0.0)
    hold(h, 1.75, -1.0)
    hold(y, 1.5, -1.5)
