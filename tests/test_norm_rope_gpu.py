"""RMS norm with the residual's addition, and rotary positions with the write
into a paged cache, against plain implementations in 64 bits.

Tolerances, derived before the first run.  u: half a unit in the last place of
the output (2^-24 f32, 2^-8 bf16, 2^-11 f16).
Norm: h is one f32 addition, the sum of d squares has a relative error below
(32 + 10 + 2) 2^-24 (32 values a thread in turn, then a tree), half of it in the root, and three
f32 roundings follow: |error| <= (u + 40 * 2^-24) |y|, plus 2^-24 max|h| w / rms where x and
residual cancel.
Scales of the 8-bit form: relative 45 * 2^-24.  A code is the e4m3 value nearest
to y / scale, or, where rounding moved y / scale across a boundary, its neighbour:
|code * scale - y| <= half a step of the code's binade (1 + 1e-4).
Rotation: cos and sin are f32 (two ulp), products and one sum in f32:
|error| <= u |y| + 6 * 2^-24 (|a| + |b|) factor.
f16 results add its smallest step 2^-25 (half of 2^-24).
"""
from __future__ import annotations

import math

import pytest
import torch

from freemoe_b200._lib import FmError

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def norm_exact(x, w, res, eps):
    h = x.double() + (0.0 if res is None else res.double())
    root = torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, h / root * w.double(), root


def hold_norm(y, x, w, res, eps, dtype):
    h, want, root = norm_exact(x, w, res, eps)
    tol = (ULP[dtype] + 40 * 2.0 ** -24) * want.abs() + FLOOR[dtype]
    if res is not None:
        tol = tol + 2.0 ** -24 * (x.double().abs() + res.double().abs()) * w.double().abs() / root
    assert ((y.double() - want).abs() <= tol).all()
    return h


def tensor(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("d", [1, 7, 8, 128, 130, 256, 264, 1000, 1024, 1032, 2048, 2050, 4096, 5000, 8192, 8200, 16384,
                               16392, 20001, 40000])
@pytest.mark.parametrize("tokens", [1, 3, 700])
def test_norm_widths(cuda, d, tokens):
    from freemoe_b200 import attention

    x, w, res = tensor(tokens, d, seed=d), tensor(d, seed=1) + 1, tensor(tokens, d, seed=2)
    y, none = attention.add_rms_norm(x, w)
    assert none is None
    hold_norm(y, x, w, None, 1e-5, F32)
    y, h = attention.add_rms_norm(x, w, residual=res, epsilon=1e-6)
    want = hold_norm(y, x, w, res, 1e-6, F32)
    assert torch.equal(h, (x + res)) and torch.allclose(h.double(), want, atol=1e-5)


@pytest.mark.parametrize("x_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("res_dtype", [None, F32, BF16, F16])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("w_dtype", [F32, BF16])
@pytest.mark.parametrize("d", [514, 2048])
def test_norm_types(cuda, x_dtype, res_dtype, out, w_dtype, d):
    from freemoe_b200 import attention

    x, w = tensor(5, d, dtype=x_dtype, seed=3), tensor(d, dtype=w_dtype, seed=4)
    res = None if res_dtype is None else tensor(5, d, dtype=res_dtype, seed=5)
    y, h = attention.add_rms_norm(x, w, residual=res, out_dtype=out)
    assert y.dtype == out
    hold_norm(y, x, w, res, 1e-5, out)
    if res is not None:
        assert h.dtype == res_dtype and torch.equal(h, (x.float() + res.float()).to(res_dtype))


def e4m3_step(v):
    """The step of e4m3 at |v| (v in code units)."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)


@pytest.mark.parametrize("d", [1, 100, 128, 130, 1000, 1024, 2050, 4096, 8192, 16384, 20000, 20001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_norm_to_8_bits(cuda, d, dtype):
    from freemoe_b200 import attention

    x, w, res = tensor(9, d, dtype=dtype, seed=d, scale=3.0), tensor(d, seed=1), tensor(9, d, dtype=dtype, seed=2)
    codes, scales, h = attention.add_rms_norm_fp8(x, w, residual=res)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == (9, d)
    groups = -(-d // 128)
    assert scales.shape == (9, groups)
    _, want, root = norm_exact(x, w, res, 1e-5)
    pad = torch.zeros(9, groups * 128, dtype=torch.float64, device="cuda")
    pad[:, :d] = want
    top = pad.view(9, groups, 128).abs().amax(-1).clamp(min=1e-10) / 448
    # x + residual may cancel in the largest value of a group: one f32 rounding of h
    assert ((scales.double() - top).abs() <= 60 * 2.0 ** -24 * top).all()
    scale = scales.double().repeat_interleave(128, 1)[:, :d]
    c = codes.float().double()
    assert (c.abs() <= 448).all()
    slack = 2.0 ** -22 * (x.double().abs() + res.double().abs()) * w.double().abs() / root
    z = want / scale
    assert ((c * scale - want).abs() <= 0.5 * (1 + 1e-4) * torch.maximum(e4m3_step(c), e4m3_step(z)) * scale + slack).all()
    assert torch.equal(h, (x.float() + res.float()).to(dtype))


def test_norm_edges(cuda):
    """Zero rows, huge and tiny rows, NaN and infinity stay in their rows."""
    from freemoe_b200 import attention

    x = tensor(6, 512)
    x[0] = 0
    x[1] *= 1e15
    x[2] *= 1e-18
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    w = tensor(512, seed=1)
    y, _ = attention.add_rms_norm(x, w, epsilon=0.0, out_dtype=F32)
    assert torch.isnan(y[0]).all()  # 0 / 0 with no epsilon
    hold_norm(y[1:3], x[1:3], w, None, 0.0, F32)
    assert torch.isnan(y[3]).all() and torch.isnan(y[4, 9]) and torch.isfinite(y[5]).all()
    codes, scales, _ = attention.add_rms_norm_fp8(x, w)
    assert (codes[0].float() == 0).all() and (scales[0] > 0).all()
    assert torch.isfinite(codes[5].float()).all()


def test_norm_strides_streams_and_in_place(cuda):
    from freemoe_b200 import attention
    from freemoe_b200._lib import RmsNormArgs, check, load
    import ctypes as C

    wide = tensor(33, 700, dtype=BF16)
    x, w = wide[:, 40:552], tensor(512, seed=1)
    want, _ = attention.add_rms_norm(x.contiguous(), w)
    assert torch.equal(attention.add_rms_norm(x, w)[0], want)
    assert torch.equal(attention.add_rms_norm(wide[:, 41:553], w)[0],
                       attention.add_rms_norm(wide[:, 41:553].contiguous(), w)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, _ = attention.add_rms_norm(x, w, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # y on x and residual_out on residual, as the C entry allows
    res = tensor(33, 512, dtype=BF16, seed=3)
    want, h = attention.add_rms_norm(x, w, residual=res)
    y, r = x.contiguous(), res.clone()
    a = RmsNormArgs(y.data_ptr(), r.data_ptr(), w.data_ptr(), y.data_ptr(), r.data_ptr(), None, 512, 512, 512, 1, 1, 0, 1,
                    33, 512, 1e-5)
    check(load().fmcuda_add_rms_norm(C.byref(a), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(y, want) and torch.equal(r, h)


def test_norm_refusals(cuda):
    from freemoe_b200 import attention

    x, w = tensor(4, 64), tensor(64)

    def refused(code, call):
        with pytest.raises(FmError) as e:
            call()
        assert e.value.code == code

    refused(26, lambda: attention.add_rms_norm(x.double(), w))
    refused(26, lambda: attention.add_rms_norm(x, w, out_dtype=torch.int8))
    refused(8, lambda: attention.add_rms_norm(x, w[:32]))
    refused(8, lambda: attention.add_rms_norm(x, w, residual=x[:2]))
    refused(26, lambda: attention.add_rms_norm(x, w, epsilon=-1.0))
    refused(26, lambda: attention.add_rms_norm(x, w, epsilon=float("nan")))
    refused(26, lambda: attention.add_rms_norm(x.cpu(), w))
    refused(8, lambda: attention.add_rms_norm(x.t(), tensor(4)))
    y, _ = attention.add_rms_norm(x[:0], w)
    assert y.shape == (0, 64)


# ---------------------------------------------------------------------------------------- rotary


def rope_exact(x, positions, inv_freq, factor, interleaved):
    half = inv_freq.shape[0]
    first = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = (torch.cos(angle) * factor)[:, None], (torch.sin(angle) * factor)[:, None]
    y = x.double().clone()
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    size = torch.zeros_like(y)
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(factor)
    return y, size


def hold_rope(got, x, positions, inv_freq, factor, interleaved):
    want, size = rope_exact(x, positions, inv_freq, factor, interleaved)
    u = ULP[got.dtype]
    assert ((got.double() - want).abs() <= u * want.abs() + 6 * 2.0 ** -24 * size + FLOOR[got.dtype]).all()


def rope_case(tokens, heads, kv_heads, dim, rot, in_dtype, out_dtype, page, interleaved, far=True, layout="hnd", seed=0):
    from freemoe_b200 import attention

    q, k, v = (tensor(tokens, h, dim, dtype=in_dtype, seed=seed + i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    g = torch.Generator(device="cuda").manual_seed(seed)
    positions = torch.randint(0, 1 << 20 if far else 100, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    inv_freq, factor = attention.rope_frequencies(rot, 10000.0, kind="ramp", factor=4.0, trained_context=4096, fast=32,
                                                  slow=1)
    pages = -(-tokens // page) + 2
    shape = (pages, kv_heads, page, dim) if layout == "hnd" else (pages, page, kv_heads, dim)
    kc, vc = (torch.full(shape, 7.0, dtype=out_dtype, device="cuda") for _ in range(2))
    if layout == "nhd":
        kc, vc = kc.permute(0, 2, 1, 3), vc.permute(0, 2, 1, 3)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    if tokens > 2:
        slots[1] = -1
    got = attention.rope_append(q, k, v, positions, inv_freq, kc, vc, slots, interleaved=interleaved,
                                attention_factor=factor)
    assert got.dtype == out_dtype
    hold_rope(got, q, positions, inv_freq, factor, interleaved)
    kf, vf = (c.transpose(1, 2).reshape(-1, kv_heads, dim) for c in (kc, vc))
    live = slots >= 0
    hold_rope(kf[slots[live]], k[live], positions[live], inv_freq, factor, interleaved)
    assert torch.equal(vf[slots[live]], v[live].to(out_dtype))
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots[live]] = False
    assert (kf[rest] == 7).all() and (vf[rest] == 7).all()


@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (80, 32), (96, 96), (96, 20), (48, 6), (17, 16),
                                     (2, 2), (256, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_rope_widths(cuda, dim, rot, interleaved, tokens):
    rope_case(tokens, 6, 2, dim, rot, F32, BF16, 16, interleaved)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("in_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (1, 1)])
def test_rope_types_and_layouts(cuda, in_dtype, out_dtype, layout, heads, kv_heads):
    rope_case(37, heads, kv_heads, 128, 128, in_dtype, out_dtype, 24, False, layout=layout)
    rope_case(37, heads, kv_heads, 64, 32, in_dtype, out_dtype, 7, True, layout=layout)
    assert cuda.device_status() == 0


def test_rope_alone_strided_and_zero_position(cuda):
    from freemoe_b200 import attention

    fused = tensor(50, 12, 64, dtype=BF16)
    positions = torch.zeros(50, dtype=torch.int32, device="cuda")
    inv_freq, factor = attention.rope_frequencies(64)
    assert factor == 1.0
    got = attention.rope_append(fused[:, 2:9], None, None, positions, inv_freq, None, None, None)
    assert torch.equal(got, fused[:, 2:9])  # position 0 turns nothing
    positions += 77
    got = attention.rope_append(fused[:, 2:9], None, None, positions, inv_freq, None, None, None, out_dtype=F32)
    hold_rope(got, fused[:, 2:9], positions, inv_freq, 1.0, False)
    none = torch.empty(0, dtype=torch.float32, device="cuda")
    assert torch.equal(attention.rope_append(fused, None, None, positions, none, None, None, None), fused)


def test_rope_keeps_relative_angles(cuda):
    """q . k after rotation depends on the distance of the positions alone, far out too."""
    from freemoe_b200 import attention

    inv_freq, _ = attention.rope_frequencies(128, 500000.0)
    q, k = tensor(1, 1, 128), tensor(1, 1, 128, seed=1)
    dots = []
    for base in (0, 1000, 131071, 1 << 22):
        at = [torch.tensor([base + d], dtype=torch.int32, device="cuda") for d in (9, 0)]
        a, b = (attention.rope_append(x, None, None, p, inv_freq, None, None, None) for x, p in zip((q, k), at))
        dots.append(float((a.double() * b.double()).sum()))
    size = float(q.double().norm() * k.double().norm())
    assert max(dots) - min(dots) <= 2 * 6 * 2.0 ** -24 * 2 * size


def test_rope_bad_slot_is_reported(cuda):
    from freemoe_b200 import attention

    q, k = tensor(3, 2, 64, dtype=BF16), tensor(3, 1, 64, dtype=BF16)
    kc = torch.zeros(2, 1, 8, 64, dtype=BF16, device="cuda")
    inv_freq, _ = attention.rope_frequencies(64)
    positions = torch.arange(3, dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 16, 1], device="cuda")
    attention.rope_append(q, k, k, positions, inv_freq, kc, kc.clone(), slots)
    assert cuda.device_status() == 26
    assert (kc[0, 0, 0] != 0).any() and (kc[0, 0, 1] != 0).any() and (kc[0, 0, 2:] == 0).all()


def test_rope_refusals(cuda):
    from freemoe_b200 import attention

    q, k = tensor(3, 2, 64, dtype=BF16), tensor(3, 1, 64, dtype=BF16)
    kc = torch.zeros(2, 1, 8, 64, dtype=BF16, device="cuda")
    inv_freq, _ = attention.rope_frequencies(64)
    positions = torch.arange(3, dtype=torch.int32, device="cuda")
    slots = torch.arange(3, device="cuda")
    ok = dict(q=q, k=k, v=k, positions=positions, inv_freq=inv_freq, k_cache=kc, v_cache=kc.clone(), slots=slots)

    def refused(code, **change):
        with pytest.raises(FmError) as e:
            attention.rope_append(**{**ok, **change})
        assert e.value.code == code

    refused(26, k=None)
    refused(26, slots=None)
    refused(8, slots=slots.int())
    refused(8, positions=positions.long())
    refused(8, inv_freq=torch.ones(40, device="cuda"))
    refused(26, q=q.float())
    refused(8, k=tensor(3, 2, 64, dtype=BF16))
    refused(8, k_cache=kc[..., :32])
    refused(26, out_dtype=F32)
    refused(26, q=q.cpu())


def test_a_layer_of_steps_matches_one_prompt(cuda):
    """A prompt in one chunk, in ragged chunks and token by token: the same rows, within the rounding of 16-bit weights."""
    from freemoe_b200 import attention

    heads, kv_heads, dim, page, n = 8, 2, 64, 16, 90
    q, k, v = (tensor(n, h, dim, seed=i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    inv_freq, factor = attention.rope_frequencies(dim)
    table = torch.tensor([[3, 0, 5, 1, 4, 2]], dtype=torch.int32, device="cuda")
    outs = []
    for chunks in ([90], [1, 40, 33, 16], [1] * 90):
        kc, vc = (torch.full((6, kv_heads, page, dim), float("nan"), dtype=BF16, device="cuda") for _ in range(2))
        at, rows = 0, []
        for c in chunks:
            pos = torch.arange(at, at + c, dtype=torch.int32, device="cuda")
            slots = table[0].long()[(pos // page).long()] * page + pos % page
            qr = attention.rope_append(q[at:at + c], k[at:at + c], v[at:at + c], pos, inv_freq, kc, vc, slots,
                                       attention_factor=factor)
            at += c
            rows.append(attention.paged_attention(
                qr, kc, vc, table, torch.tensor([0, c], dtype=torch.int32, device="cuda"),
                torch.tensor([at], dtype=torch.int32, device="cuda"), max_q_len=c, max_kv_len=at))
        outs.append(torch.cat(rows).double())
    assert cuda.device_status() == 0
    for o in outs[1:]:
        assert ((o - outs[0]).abs() <= 2 * 2.0 ** -8 * (o.abs() + 4.0)).all()
    assert math.isfinite(float(outs[0].sum()))
