"""The attention side where values, lengths and launches are at their edges.

Tolerances are those of tests/test_attention_gpu.py and tests/test_norm_rope_gpu.py; what has to be
the same row in another call is compared bit by bit."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from test_attention_gpu import Batch
from test_norm_rope_gpu import BF16, F16, F32, e4m3_step, hold_norm, norm_exact, rope_case, tensor

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


# widths of 16-byte accesses, of pairs and of single values, in a warp, in a CTA and read twice
@pytest.mark.parametrize("d", [512, 514, 513, 4096, 4098, 4097, 20000, 20002, 20001])
def test_infinite_results_to_8_bits(cuda, d):
    """The scale of a group with an infinity is infinite: finite values are 0 there, infinite
    ones infinity by infinity; the other groups are as they were."""
    from freemoe_b200 import attention

    x, w = tensor(5, d, seed=d), tensor(d, seed=1) + 2
    want, want_scales, _ = attention.add_rms_norm_fp8(x, w)
    at = 200
    w[at] = INF
    x[3, at] = 0  # 0 * infinity: NaN, which does not count for the largest
    want3, want3_scales, _ = attention.add_rms_norm_fp8(x, torch.where(w == INF, 0, w))
    codes, scales, _ = attention.add_rms_norm_fp8(x, w)
    codes, want, want3 = codes.float(), want.float(), want3.float()
    want[3], want_scales[3] = want3[3], want3_scales[3]
    rows = torch.tensor([0, 1, 2, 4], device="cuda")
    assert (scales[rows, 1] == INF).all()
    group = codes[rows, 128:256].clone()
    assert torch.isnan(group[:, at - 128]).all()
    group[:, at - 128] = 0
    assert (group == 0).all()
    assert torch.isnan(codes[3, at])
    codes[3, at] = 0
    codes[rows, 128:256], scales[rows, 1] = want[rows, 128:256], want_scales[rows, 1]
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)


# the sequences beside the chunk in even ranges, a CTA each, a warp each
@pytest.mark.parametrize("lens", [[(1, 7000), (150, 900), (1, 300), (1, 9000)], [(1, 700), (150, 900), (1, 300)],
                                  [(1, 100 + b) for b in range(150)] + [(70, 256)]])
def test_calls_see_what_was_written_just_before(cuda, lens):
    """Queries, keys, lengths and pages come from kernels right before the call, in both parts of its
    grid: other ones each time, and the results those of calls that nothing runs beside."""
    a, b = (Batch(lens, 8, 2, 128, 16, seed=61 + i) for i in range(2))
    names = ("q", "k_cache", "v_cache", "table")
    versions = [[getattr(x, n).clone() for n in names] + [x.kv_len - i] for i, x in enumerate((a, b))]
    want = []
    for version in versions:
        for n, t in zip((*names, "kv_len"), version):
            getattr(a, n).copy_(t)
        torch.cuda.synchronize()
        want.append(a.run())
        torch.cuda.synchronize()
    assert not torch.equal(want[0][0], want[1][0])
    got = []
    for i in range(20):
        for n, t in zip((*names, "kv_len"), versions[i % 2]):
            getattr(a, n).copy_(t)
        got.append(a.run())
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])
    assert cuda.device_status() == 0


# blocks dealt out in even ranges (the range that ends the first sequence goes on in one that was left
# out, and is longer than the CTAs behind it take) and in pieces, and items dealt whole
@pytest.mark.parametrize("rows,kvs", [(3000, [3000, 9, 60000, 9, 3000, 9, 3000, 9, 3000]), (300, [9000] * 9), (300, [600] * 9)])
def test_sequences_that_overlap_are_reported(cuda, rows, kvs):
    """q_start that goes back: more tiles than there are rows for.  Nothing is written but the rows and
    the workspace, and the next call is right."""
    from freemoe_b200._lib import PagedAttentionArgs, check, load

    good = Batch([(rows, kvs[0]), (1, 40)], 8, 2, 128, 64, seed=71)
    want, _ = good.run()
    b = Batch([(rows if i == 0 else 0, kv) for i, kv in enumerate(kvs)], 8, 2, 128, 64, seed=72)
    b.q_start.copy_(torch.tensor([0, rows] * 2 + [0, 64] * 3, dtype=torch.int32))
    args = PagedAttentionArgs(
        q=b.q.data_ptr(), k_cache=b.k_cache.data_ptr(), v_cache=b.v_cache.data_ptr(), out=b.q.data_ptr(),
        page_table=b.table.data_ptr(), q_start=b.q_start.data_ptr(), kv_len=b.kv_len.data_ptr(), q_token_stride=1024,
        q_head_stride=128, out_token_stride=1024, out_head_stride=128, cache_page_stride=b.k_cache.stride(0),
        cache_head_stride=b.k_cache.stride(1), cache_row_stride=128, page_table_stride=b.table.stride(0), dtype=1, seqs=9,
        tokens=rows, heads=8, kv_heads=2, head_dim=128, n_pages=b.k_cache.shape[0], page_size=64, max_q_len=rows,
        max_kv_len=max(kvs), causal=1, scale=b.scale)
    size = C.c_uint64()
    check(load().fmcuda_paged_attention_workspace_bytes(C.byref(args), C.byref(size)))
    guard = 1 << 20
    workspace = torch.full((size.value + guard,), 90, dtype=torch.uint8, device="cuda")
    out = torch.full((rows * 8 * 128 + guard,), 1.5, dtype=b.dtype, device="cuda")
    args.out = out.data_ptr()
    check(load().fmcuda_paged_attention(C.byref(args), workspace.data_ptr(), size.value,
                                        torch.cuda.current_stream().cuda_stream))
    assert cuda.device_status() == 26
    assert (workspace[size.value:] == 90).all() and (out[rows * 8 * 128:] == 1.5).all()
    assert torch.equal(good.run()[0], want)
    assert cuda.device_status() == 0


def test_a_rotation_of_no_tokens(cuda):
    from freemoe_b200 import attention

    q, k = tensor(3, 4, 64, dtype=torch.bfloat16), tensor(3, 2, 64, dtype=torch.bfloat16, seed=1)
    kc, vc = (torch.full((2, 2, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    inv_freq, _ = attention.rope_frequencies(64)
    at = torch.arange(3, device="cuda")
    for n in (slice(0, 0), slice(3, 3)):
        got = attention.rope_append(q[n], k[n], k[n], at.int()[n], inv_freq, kc, vc, at[n])
        assert got.shape == (0, 4, 64) and got.dtype == kc.dtype
        assert attention.rope_append(q[n], None, None, at.int()[n], inv_freq, None, None, None).shape == (0, 4, 64)
    assert (kc == 7).all() and (vc == 7).all() and cuda.device_status() == 0


def hold_codes(codes, scales, x, w, res):
    """As in tests/test_norm_rope_gpu.py: a code is the value nearest to y / scale or, at a boundary, its neighbour."""
    rows, d = x.shape
    _, want, root = norm_exact(x, w, res, 1e-5)
    groups = -(-d // 128)
    pad = torch.zeros(rows, groups * 128, dtype=torch.float64, device="cuda")
    pad[:, :d] = want
    top = pad.view(rows, groups, 128).abs().amax(-1).clamp(min=1e-10) / 448
    assert ((scales.double() - top).abs() <= 60 * 2.0 ** -24 * top).all()
    scale = scales.double().repeat_interleave(128, 1)[:, :d]
    c = codes.float().double()
    slack = 2.0 ** -22 * (x.double().abs() + res.double().abs()) * w.double().abs() / root
    step = torch.maximum(e4m3_step(c), e4m3_step(want / scale))
    assert ((c * scale - want).abs() <= 0.5 * (1 + 1e-4) * step * scale + slack).all()


# rows for teams of a warp (up to 1024 values) and of a CTA, in eights, pairs and single values,
# and more of them than the GPU holds at once: every team takes several
@pytest.mark.parametrize("tokens,d", [(20011, 200), (20011, 202), (20011, 201), (12007, 1024), (12007, 1022), (12007, 1021),
                                      (5003, 2048), (5003, 2050), (5003, 2049), (2999, 4096), (2999, 4094), (2999, 4095),
                                      (1201, 16384), (1201, 16382), (1201, 16381), (601, 20000), (601, 20001)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_of_more_rows_than_teams(cuda, tokens, d, dtype):
    from freemoe_b200 import attention
    from freemoe_b200._lib import RmsNormArgs, check, load

    x, w, res = tensor(tokens, d, dtype=dtype, seed=d), tensor(d, seed=1) + 1, tensor(tokens, d, dtype=dtype, seed=2)
    y, h = attention.add_rms_norm(x, w, residual=res)
    hold_norm(y, x, w, res, 1e-5, dtype)
    assert torch.equal(h, (x.float() + res.float()).to(dtype))
    y32, _ = attention.add_rms_norm(x, w, out_dtype=F32)
    hold_norm(y32, x, w, None, 1e-5, F32)
    del y32
    codes, scales, h8 = attention.add_rms_norm_fp8(x, w, residual=res)
    assert torch.equal(h8, h)
    hold_codes(codes, scales, x, w, res)
    kind = {F32: 0, BF16: 1, F16: 2}[dtype]  # y on x and residual_out on residual
    a = RmsNormArgs(x.data_ptr(), res.data_ptr(), w.data_ptr(), x.data_ptr(), res.data_ptr(), None, d, d, d, kind, kind, 0,
                    kind, tokens, d, 1e-5)
    check(load().fmcuda_add_rms_norm(C.byref(a), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(x, y) and torch.equal(res, h)


# more tokens than four an SM: several to a CTA, fewer to the last one
@pytest.mark.parametrize("tokens", [1001, 2371, 5000])
@pytest.mark.parametrize("dim,rot,interleaved", [(128, 128, True), (80, 42, True), (128, 128, False), (64, 32, False),
                                                 (96, 96, False), (80, 32, False), (80, 42, False), (128, 0, False)])
@pytest.mark.parametrize("in_dtype,out_dtype", [(F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_rotation_of_batches_of_tokens(cuda, tokens, dim, rot, interleaved, in_dtype, out_dtype, layout):
    if rot == 0:
        q, k = tensor(tokens, 3, dim, dtype=in_dtype), tensor(tokens, 1, dim, dtype=in_dtype, seed=1)
        kc, vc = (torch.zeros(tokens, 1, 8, dim, dtype=out_dtype, device="cuda") for _ in range(2))
        at = torch.arange(tokens, device="cuda")
        from freemoe_b200 import attention

        got = attention.rope_append(q, k, k, at.int(), torch.empty(0, device="cuda"), kc, vc, at * 8 + 3)
        assert torch.equal(got, q.to(out_dtype)) and torch.equal(kc[:, :, 3], k.to(out_dtype)) and torch.equal(kc, vc)
    else:
        rope_case(tokens, 5, 2, dim, rot, in_dtype, out_dtype, 48, interleaved, layout=layout, seed=tokens)
    assert cuda.device_status() == 0
