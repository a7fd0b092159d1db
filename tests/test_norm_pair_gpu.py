"""The norms around a block, with its gated addition to the residual stream, against a
plain implementation in 64 bits.

Tolerances, derived before the first run.  E = 2^-24; u: half a unit in the last place of
an output (2^-24 f32, 2^-8 bf16, 2^-11 f16).
A sum of d squares has a relative error below 44 E (up to 32 values a thread in turn, then
a tree), half of it in the root; the root itself and the division add 5 E; the scale, the
gate and the weight are products of their own, 5 roundings at most, in any order.  With
t = s g n this is |error of t| <= 35 E |t|, and with the one rounding of the sum
    dh = 35 E |t| + 2 E (|a r| + |t|)
bounds the error of h before it is stored (u |h| more, and 2^-25 for f16).
y has the factor w2 / rms(h); the root moves by at most sum |h| dh / sum h^2, so that
    |error of y| <= u |y| + 40 E |y| + |w2| dh / rms + |y| sum |h| dh / sum h^2.
A scale is within the largest such error of its group, and 4 E; a code is the e4m3 value
nearest to y / scale, or where rounding moved y / scale across a boundary its neighbour.
"""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from freemoe_b200._lib import FmError, NormAddNormArgs, check, load

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
ULP = {torch.float32: E, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FLOOR = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def tensor(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def exact(x, w1, res, w2, gate=None, scale=1.0, residual_scale=1.0, eps=1e-5):
    """h, y and the bounds of their errors before they are rounded to their types."""
    x, res, s, a = x.double(), res.double(), float(torch.tensor(scale)), float(torch.tensor(residual_scale))
    t = x if w1 is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w1.double()
    t = s * t * (1.0 if gate is None else gate.double())
    h = a * res + t
    dh = 35 * E * t.abs() + 2 * E * ((a * res).abs() + t.abs())
    if w2 is None:
        return h, dh, None, None
    root = torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    y = h / root * w2.double()
    moved = (h.abs() * dh).sum(-1, keepdim=True) / (h * h).sum(-1, keepdim=True).clamp(min=1e-300)
    return h, dh, y, 40 * E * y.abs() + w2.double().abs() * dh / root + y.abs() * moved


def within(got, want, slack):
    off = (got.double() - want).abs() - (ULP[got.dtype] * (want.abs() + slack) + slack + FLOOR[got.dtype])
    assert (off <= 0).all(), f"{off.max().item()} past the bound"


def hold(x, w1, res, w2, out=None, **how):
    from freemoe_b200 import attention

    y, h = attention.norm_add_norm(x, w1, res, w2, out_dtype=out, **how)
    how["eps"] = how.pop("epsilon", 1e-5)
    want_h, dh, want_y, dy = exact(x, w1, res, w2, **how)
    assert h.dtype == res.dtype and h.shape == x.shape
    within(h, want_h, dh)
    if w2 is None:
        assert y is None
    else:
        assert y.dtype == (out or x.dtype)
        within(y, want_y, dy)
    return y, h


@pytest.mark.parametrize("d", [1, 7, 8, 128, 130, 256, 264, 1000, 1024, 1032, 2048, 2050, 4096, 5000, 8192, 8200, 16384,
                               16392, 20001, 40000])
@pytest.mark.parametrize("tokens", [1, 3, 700])
def test_widths(cuda, d, tokens):
    x, w1, w2, res = tensor(tokens, d, seed=d), tensor(d, seed=1) + 1, tensor(d, seed=2) + 1, tensor(tokens, d, seed=3)
    hold(x, w1, res, w2, gate=tensor(d, seed=4), scale=0.3, residual_scale=0.9, epsilon=1e-6)
    hold(x.bfloat16(), w1, res.bfloat16(), w2)


@pytest.mark.parametrize("x_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("res_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("d", [514, 515, 768, 2048])
def test_types(cuda, x_dtype, res_dtype, out, d):
    x, res = tensor(5, d, dtype=x_dtype, seed=3), tensor(5, d, dtype=res_dtype, seed=5)
    for w_dtype in (F32, BF16):
        hold(x, tensor(d, dtype=w_dtype, seed=1), res, tensor(d, dtype=w_dtype, seed=2), out=out)


@pytest.mark.parametrize("gate_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", ["channel", "one row", "token", "one", "full"])
@pytest.mark.parametrize("tokens,d", [(1, 64), (37, 1000), (300, 4096), (5, 1537), (2, 30002)])
def test_gates(cuda, gate_dtype, shape, tokens, d):
    size = {"channel": (d,), "one row": (1, d), "token": (tokens, 1), "one": (1, 1), "full": (tokens, d)}[shape]
    gate = tensor(*size, dtype=gate_dtype, seed=9)
    x, res, w1, w2 = tensor(tokens, d, seed=1), tensor(tokens, d, dtype=BF16, seed=2), tensor(d, seed=3), tensor(d, seed=4)
    hold(x, w1, res, w2, out=BF16, gate=gate, scale=-1.7)
    hold(x, None, res, w2, gate=gate, residual_scale=0.0)


@pytest.mark.parametrize("d", [64, 700, 4096, 9999, 20000])
@pytest.mark.parametrize("tokens", [1, 400])
def test_without_one_of_the_norms(cuda, d, tokens):
    x, res, w = tensor(tokens, d, dtype=F16, seed=1), tensor(tokens, d, dtype=F16, seed=2), tensor(d, seed=3)
    hold(x, None, res, w)
    hold(x, w, res, None, scale=0.25)
    y, h = hold(x, None, res, None)
    assert torch.equal(h, x + res)


@pytest.mark.parametrize("d", [1, 100, 128, 130, 1000, 1024, 2050, 4096, 8192, 16384, 20000, 20001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_to_8_bits(cuda, d, dtype):
    from freemoe_b200 import attention

    x, res = tensor(9, d, dtype=dtype, seed=d, scale=3.0), tensor(9, d, dtype=BF16, seed=2)
    w1, w2, gate = tensor(d, seed=1), tensor(d, seed=4), tensor(9, 1, seed=5)
    codes, scales, h = attention.norm_add_norm_fp8(x, w1, res, w2, gate=gate, scale=0.5)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == (9, d)
    want_h, dh, want, dy = exact(x, w1, res, w2, gate=gate, scale=0.5)
    within(h, want_h, dh)
    groups = -(-d // 128)

    def by_group(v):
        return torch.nn.functional.pad(v, (0, groups * 128 - d)).view(9, groups, 128).abs().amax(-1)

    top = by_group(want).clamp(min=1e-10) / 448
    assert ((scales.double() - top).abs() <= by_group(dy) / 448 + 4 * E * top).all()
    scale = scales.double().repeat_interleave(128, 1)[:, :d]
    c = codes.float().double()

    def step(v):  # of e4m3 at |v|
        return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)

    off = (c * scale - want).abs() - 0.5 * (1 + 1e-4) * torch.maximum(step(c), step(want / scale)) * scale - dy
    assert (c.abs() <= 448).all() and (off <= 0).all()


def test_a_block_that_cancels_the_stream(cuda):
    """h is a millionth of its two parts: its norm is of what is left, not of rounding errors."""
    d = 4096
    x, w2 = tensor(6, d, seed=1), tensor(d, seed=2)
    res = -x + tensor(6, d, seed=3, scale=1e-6)
    y, _ = hold(x, None, res, w2, out=F32, epsilon=0.0)
    assert (y.double().square().mean(-1) > 0.1).all()


def test_rows_keep_to_themselves(cuda):
    """Zero rows, huge and tiny rows; NaN and infinity stay in their rows."""
    from freemoe_b200 import attention

    x, res, w = tensor(7, 512), tensor(7, 512, seed=1), tensor(512, seed=2)
    x[0] = 0
    x[1] *= 1e15
    x[2] *= 1e-18
    x[3, 7] = float("nan")
    res[4, 9] = float("inf")
    x[5] = 0
    res[5] = 0
    y, h = attention.norm_add_norm(x, w, res, w)
    assert torch.equal(h[0], res[0]) and torch.isnan(h[3]).all() and torch.isnan(y[3]).all()
    assert torch.isfinite(h[4, :9]).all() and h[4, 9] == float("inf") and torch.isnan(y[4, 9]) and (y[4, :9] == 0).all()
    assert (y[5] == 0).all() and (h[5] == 0).all()
    hold(x[1:3], w, res[1:3], w)
    hold(x[6:], w, res[6:], w)


def test_strides_streams_and_in_place(cuda):
    from freemoe_b200 import attention

    wide, other = tensor(33, 700, dtype=BF16), tensor(33, 900, dtype=F16, seed=1)
    w1, w2 = tensor(512, seed=1), tensor(512, seed=2)
    for at in (40, 41, 42):
        x, res, gate = wide[:, at:at + 512], other[:, at:at + 512], wide[:, at + 1:at + 513]
        want = attention.norm_add_norm(x.contiguous(), w1, res.contiguous(), w2, gate=gate.contiguous())
        got = attention.norm_add_norm(x, w1, res, w2, gate=gate)
        # another way through the row adds its squares in another order
        for a, b in zip(got, want):
            assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -6, atol=1e-6)
        hold(x, w1, res, w2, gate=gate)
        token = other[:, at:at + 1]
        hold(x, w1, res, w2, gate=token)
    x, res = wide[:, 40:552].contiguous(), tensor(33, 512, dtype=BF16, seed=3)
    want, h = attention.norm_add_norm(x, w1, res, w2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, _ = attention.norm_add_norm(x, w1, res, w2, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # y on x and residual_out on residual, as the C entry allows
    for rows, width in ((33, 512), (4, 20000)):
        x, res = tensor(rows, width, dtype=BF16), tensor(rows, width, dtype=BF16, seed=3)
        w = tensor(width, seed=4)
        want, h = attention.norm_add_norm(x, w, res, w)
        y, r = x.clone(), res.clone()
        a = NormAddNormArgs(x=y.data_ptr(), post_weight=w.data_ptr(), residual=r.data_ptr(), pre_weight=w.data_ptr(),
                            y=y.data_ptr(), residual_out=r.data_ptr(), x_stride=width, residual_stride=width,
                            y_stride=width, x_dtype=1, residual_dtype=1, weight_dtype=0, y_dtype=1, tokens=rows,
                            d_model=width, scale=1.0, residual_scale=1.0, epsilon=1e-5)
        check(load().fmcuda_norm_add_norm(C.byref(a), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(y, want) and torch.equal(r, h)


def test_rows_far_apart(cuda):
    """Rows whose distance passes 32 bits of values."""
    big = torch.empty((1 << 31) + 4096, dtype=BF16, device="cuda")
    x = big.as_strided((3, 1024), (1 << 30, 1))
    x.copy_(tensor(3, 1024, dtype=BF16))
    w = tensor(1024, seed=1)
    hold(x, w, tensor(3, 1024, seed=2), w)


@pytest.mark.parametrize("tokens,d", [(40, 2048), (3000, 7000), (3, 40000), (1, 4096)])
def test_captured_and_replayed(cuda, tokens, d):
    from freemoe_b200 import attention

    x, res, w = tensor(tokens, d, dtype=BF16), tensor(tokens, d, dtype=BF16, seed=1), tensor(d, seed=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = attention.norm_add_norm(x, w, res, w)
    for seed in (5, 6):
        x.copy_(tensor(tokens, d, dtype=BF16, seed=seed))
        graph.replay()
        want = attention.norm_add_norm(x, w, res, w)
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])


def test_a_very_wide_row(cuda):
    """2^22 values: a thread adds 4096 of them, chunk by chunk of eight and the chunks in turn, which the bound on a sum's error
    covers with (8 + 512 + 15) 2^-24 in place of 44 2^-24."""
    from freemoe_b200 import attention

    d = 1 << 22
    x, res, w1, w2 = (tensor(2, d, seed=1), tensor(2, d, dtype=BF16, seed=2), tensor(d, seed=3), tensor(d, seed=4))
    y, h = attention.norm_add_norm(x, w1, res, w2)
    want_h, dh, want_y, dy = exact(x, w1, res, w2)
    within(h, want_h, dh * (535 + 35) / 35)
    within(y, want_y, dy * (535 + 40) / 35)


def test_refusals(cuda):
    from freemoe_b200 import attention

    x, w, r = tensor(4, 64), tensor(64), tensor(4, 64, seed=1)

    def refused(code, *args, fn=attention.norm_add_norm, **how):
        with pytest.raises(FmError) as e:
            fn(*args, **how)
        assert e.value.code == code

    refused(26, x.double(), w, r, w)
    refused(26, x, w, r.int(), w)
    refused(26, x, w, r, w, out_dtype=torch.int8)
    refused(26, x, w, r, w.bfloat16())
    refused(8, x, w[:32], r, w)
    refused(8, x, w, r, w[:32])
    refused(8, x, w, r[:2], w)
    refused(8, x, w, r, w, gate=tensor(32))
    refused(8, x, w, r, w, gate=tensor(4))
    refused(8, x, w, r, w, gate=tensor(3, 64))
    refused(8, x, w, r, w, gate=tensor(1, 4, 64))
    refused(26, x, w, r, w, gate=w.double())
    refused(26, x, w, r, w, gate=w.cpu())
    refused(26, x, w, r, w, epsilon=-1.0)
    refused(26, x, w, r, w, epsilon=float("nan"))
    refused(26, x, w, r, w, scale=float("inf"))
    refused(26, x, w, r, w, residual_scale=float("nan"))
    refused(26, x.cpu(), w, r, w)
    refused(26, x, w, r.cpu(), w)
    refused(8, x.t(), tensor(4), r.t(), tensor(4))
    refused(8, x[0], w, r[0], w)
    refused(8, x[:1].expand(4, 64), w, r, w)
    refused(26, x.double(), w, r, w, fn=attention.norm_add_norm_fp8)
    y, h = attention.norm_add_norm(x[:0], w, r[:0], w)
    assert y.shape == h.shape == (0, 64)


@pytest.mark.parametrize("x_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("res_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [5, 700])
@pytest.mark.parametrize("d", [1026, 1537, 6001])
def test_types_of_long_odd_rows(cuda, x_dtype, res_dtype, tokens, d):
    x, res = tensor(tokens, d, dtype=x_dtype, seed=3), tensor(tokens, d, dtype=res_dtype, seed=5)
    for w_dtype in (F32, BF16, F16):
        w1, w2 = tensor(d, dtype=w_dtype, seed=1), tensor(d, dtype=w_dtype, seed=2)
        hold(x, w1, res, w2, out=F16, gate=tensor(d, dtype=x_dtype, seed=4), scale=0.7)
