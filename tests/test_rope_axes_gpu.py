"""Rotary positions of several axes, with the write into a paged cache, against a plain
implementation in 64 bits.

Tolerance, derived before the first run: cos and sin are f32 (two ulp), products and one sum
in f32: |error| <= u |y| + 6 * 2^-24 (|a| + |b|) factor, u half a unit in the last place of
the output; f16 results add half of their smallest step, 2^-25.
"""
from __future__ import annotations

import pytest
import torch

from freemoe_b200._lib import FmError

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def tensor(*shape, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def hold(got, x, positions, axis, inv_freq, factor, interleaved):
    half = inv_freq.shape[0]
    first = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    angle = torch.stack([positions[a].double() * f for a, f in zip(axis, inv_freq.double().tolist())], -1)
    cos, sin = (torch.cos(angle) * factor)[:, None], (torch.sin(angle) * factor)[:, None]
    want = x.double().clone()
    a, b = want[..., first].clone(), want[..., second].clone()
    want[..., first], want[..., second] = a * cos - b * sin, a * sin + b * cos
    size = torch.zeros_like(want)
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * factor
    assert ((got.double() - want).abs() <= ULP[got.dtype] * want.abs() + 6 * 2.0 ** -24 * size + FLOOR[got.dtype]).all()


def case(tokens, heads, kv_heads, dim, axis, in_dtype, out_dtype, page, interleaved, layout="hnd", seed=0, far=1 << 20):
    from freemoe_b200 import attention

    axes = max(axis) + 1
    q, k, v = (tensor(tokens, h, dim, dtype=in_dtype, seed=seed + i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    g = torch.Generator(device="cuda").manual_seed(seed)
    positions = torch.randint(0, far, (axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    inv_freq, factor = attention.rope_frequencies(2 * len(axis), 1e6)
    pages = -(-tokens // page) + 2
    shape = (pages, kv_heads, page, dim) if layout == "hnd" else (pages, page, kv_heads, dim)
    kc, vc = (torch.full(shape, 7.0, dtype=out_dtype, device="cuda") for _ in range(2))
    if layout == "nhd":
        kc, vc = kc.permute(0, 2, 1, 3), vc.permute(0, 2, 1, 3)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    if tokens > 2:
        slots[1] = -1
    got = attention.rope_append(q, k, v, positions, inv_freq, kc, vc, slots, interleaved=interleaved,
                                attention_factor=1.25, axes=torch.tensor(axis, dtype=torch.uint8, device="cuda"))
    assert got.dtype == out_dtype
    hold(got, q, positions, axis, inv_freq, 1.25, interleaved)
    kf, vf = (c.transpose(1, 2).reshape(-1, kv_heads, dim) for c in (kc, vc))
    live = slots >= 0
    hold(kf[slots[live]], k[live], positions[:, live], axis, inv_freq, 1.25, interleaved)
    assert torch.equal(vf[slots[live]], v[live].to(out_dtype))
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots[live]] = False
    assert (kf[rest] == 7).all() and (vf[rest] == 7).all()


@pytest.mark.parametrize("sections,dim", [((64,), 128), ((16, 24, 24), 128), ((8, 12, 12), 64), ((1, 2, 0, 1), 80),
                                          ((20, 20), 80), ((24, 24), 96), ((1, 1, 1, 1, 1, 1, 1, 1), 17), ((3, 5, 7, 1), 64),
                                          ((200, 56), 512)])
@pytest.mark.parametrize("order", ["blocks", "turn"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 5, 700])
def test_sections(cuda, sections, dim, order, interleaved, tokens):
    from freemoe_b200 import attention

    axis = attention.rope_axes(sections, order).tolist()
    assert [axis.count(a) for a in range(len(sections))] == list(sections)
    case(tokens, 6, 2, dim, axis, F32, BF16, 16, interleaved)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("in_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (1, 1)])
def test_types_and_layouts(cuda, in_dtype, out_dtype, layout, heads, kv_heads):
    case(37, heads, kv_heads, 128, [0] * 16 + [1] * 24 + [2] * 24, in_dtype, out_dtype, 24, False, layout=layout)
    case(2000, heads, kv_heads, 64, [0, 1, 2, 3] * 4, in_dtype, out_dtype, 7, True, layout=layout)
    assert cuda.device_status() == 0


def test_far_positions_keep_their_angle(cuda):
    case(9, 4, 4, 64, [2, 1, 0] * 8, F32, F32, 8, False, far=(1 << 31) - 1)


def test_text_stands_at_one_position_on_all_axes(cuda):
    """Where the axes agree the rotation is that of one axis, bit for bit."""
    from freemoe_b200 import attention

    q, at = tensor(77, 5, 96, dtype=BF16), torch.arange(5000, 5077, dtype=torch.int32, device="cuda")
    inv_freq, _ = attention.rope_frequencies(96)
    axes = attention.rope_axes((16, 20, 12), "turn")
    got = attention.rope_append(q, None, None, at.expand(3, -1).contiguous(), inv_freq, None, None, None, axes=axes)
    assert torch.equal(got, attention.rope_append(q, None, None, at, inv_freq, None, None, None))
    # rows of a wider table of positions
    table = torch.full((3, 200), -5, dtype=torch.int32, device="cuda")
    table[:, 20:97] = at
    assert torch.equal(attention.rope_append(q, None, None, table[:, 20:97], inv_freq, None, None, None, axes=axes), got)


def test_an_unknown_axis_is_reported(cuda):
    from freemoe_b200 import attention

    q, at = tensor(3, 2, 64), torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
    inv_freq, _ = attention.rope_frequencies(64)
    axes = attention.rope_axes((16, 16))
    axes[9] = 2
    got = attention.rope_append(q, None, None, at, inv_freq, None, None, None, axes=axes)
    assert cuda.device_status() == 26
    axes[9] = 0
    assert torch.equal(got, attention.rope_append(q, None, None, at, inv_freq, None, None, None, axes=axes))
    assert cuda.device_status() == 0


def test_captured_and_replayed(cuda):
    from freemoe_b200 import attention

    q, at = tensor(30, 4, 128, dtype=BF16), torch.randint(0, 9000, (3, 30), dtype=torch.int32, device="cuda")
    inv_freq, _ = attention.rope_frequencies(128)
    axes = attention.rope_axes((16, 24, 24))

    def call():
        return attention.rope_append(q, None, None, at, inv_freq, None, None, None, axes=axes)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(2):
        at.random_(0, 100000)
        graph.replay()
        assert torch.equal(got, call())


def test_refusals(cuda):
    from freemoe_b200 import attention

    q = tensor(3, 2, 64)
    at = torch.zeros(3, 3, dtype=torch.int32, device="cuda")
    inv_freq, _ = attention.rope_frequencies(64)
    axes = attention.rope_axes((8, 12, 12))
    ok = dict(q=q, k=None, v=None, positions=at, inv_freq=inv_freq, k_cache=None, v_cache=None, slots=None, axes=axes)

    def refused(code, **change):
        with pytest.raises(FmError) as e:
            attention.rope_append(**{**ok, **change})
        assert e.value.code == code

    refused(8, axes=None)
    refused(8, positions=at[0])
    refused(8, positions=at[:, :2])
    refused(8, positions=at.long())
    refused(8, positions=at.t().contiguous().t())
    refused(8, positions=at[:1].expand(3, 3))
    refused(8, positions=torch.zeros(9, 3, dtype=torch.int32, device="cuda"))
    refused(8, positions=at[:0])
    refused(8, axes=axes[:31])
    refused(8, axes=axes.int())
    refused(26, axes=axes.cpu())
    none = attention.rope_append(q[:0], None, None, at[:, :0], inv_freq, None, None, None, axes=axes)
    assert none.shape == (0, 2, 64)
