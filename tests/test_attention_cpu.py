"""The attention side without a GPU: refusals made before any CUDA call, rotary
frequencies against their formulas, the argument structs' layouts, and the
bounds of a call's workspace."""
from __future__ import annotations

import ctypes as C
import math
import subprocess

import pytest

from conftest import ROOT
from freemoe_b200 import load
from freemoe_b200 import _lib
from freemoe_b200._lib import FmError, PagedAttentionArgs, RmsNormArgs, RopeAppendArgs, RopeScaling

OK, SHAPE, ARG = 0, 8, 26
P = 1 << 20  # an address that is not null; nothing here is read


@pytest.mark.parametrize("name,struct", [("fmcuda_rms_norm_args", RmsNormArgs),
                                         ("fmcuda_rope_append_args", RopeAppendArgs),
                                         ("fmcuda_rope_scaling", RopeScaling),
                                         ("fmcuda_paged_attention_args", PagedAttentionArgs)])
def test_struct_layouts_match_the_header(tmp_path, name, struct):
    fields = [f for f, _ in struct._fields_]
    prints = "".join(f'printf("%zu ", offsetof({name}, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "freemoe_b200.h"\n'
                   f'int main(void) {{ {prints} printf("%zu", sizeof({name})); return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [getattr(struct, f).offset for f in fields] + [C.sizeof(struct)]


def norm_args(**change):
    a = RmsNormArgs(x=P, weight=P, y=P, x_stride=64, y_stride=64, tokens=4, d_model=64, epsilon=1e-5)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("code,change", [
    (ARG, {"x": None}), (ARG, {"weight": None}), (ARG, {"y": None}), (SHAPE, {"d_model": 0}),
    (SHAPE, {"d_model": (1 << 24) + 1}), (ARG, {"x_dtype": 3}), (ARG, {"x_dtype": -1}), (ARG, {"weight_dtype": 3}),
    (ARG, {"y_dtype": 4}), (ARG, {"y_dtype": 3}), (ARG, {"residual": P, "residual_dtype": 3, "residual_stride": 64}),
    (SHAPE, {"x_stride": 63}), (SHAPE, {"y_stride": 0}), (SHAPE, {"residual": P, "residual_stride": 10}),
    (ARG, {"epsilon": -1.0}), (ARG, {"epsilon": float("nan")}), (ARG, {"x": P + 1}), (ARG, {"y": P + 2}),
    (OK, {"tokens": 0}), (OK, {"tokens": 0, "x": None}),
])
def test_norm_refuses(code, change):
    lib = load()
    assert lib.fmcuda_add_rms_norm(C.byref(norm_args(**change)), None) == code
    if code:
        assert lib.fmcuda_last_error()


def test_null_arguments_are_refused():
    lib = load()
    assert lib.fmcuda_add_rms_norm(None, None) == ARG
    assert lib.fmcuda_rope_append(None, None) == ARG
    assert lib.fmcuda_paged_attention(None, None, 0, None) == ARG
    assert lib.fmcuda_paged_attention_workspace_bytes(None, C.byref(C.c_uint64())) == ARG
    assert lib.fmcuda_paged_attention_workspace_bytes(C.byref(attention_args()), None) == ARG


def rope_args(**change):
    a = RopeAppendArgs(q=P, k=P, v=P, q_out=P, k_cache=P, v_cache=P, positions=P, slots=P, inv_freq=P,
                       q_token_stride=128, q_head_stride=64, k_token_stride=64, k_head_stride=64, v_token_stride=64,
                       v_head_stride=64, q_out_token_stride=128, q_out_head_stride=64, cache_page_stride=1024,
                       cache_head_stride=1024, cache_row_stride=64, in_dtype=1, out_dtype=1, tokens=3, heads=2,
                       kv_heads=1, head_dim=64, rot_dim=64, attention_factor=1.0, n_pages=2, page_size=16)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("code,change", [
    (SHAPE, {"heads": 0}), (SHAPE, {"head_dim": 0}), (SHAPE, {"head_dim": 1025}), (SHAPE, {"rot_dim": 63}),
    (SHAPE, {"rot_dim": 66}), (ARG, {"in_dtype": 3}), (ARG, {"out_dtype": -1}), (ARG, {"k": None}), (ARG, {"slots": None}),
    (ARG, {"v_cache": None}), (SHAPE, {"kv_heads": 0}), (SHAPE, {"page_size": 0}), (ARG, {"q": None}), (ARG, {"q_out": None}),
    (ARG, {"positions": None}), (ARG, {"inv_freq": None}), (ARG, {"k": P + 1}), (SHAPE, {"tokens": 1 << 31}),
    (OK, {"tokens": 0}),
])
def test_rope_refuses(code, change):
    assert load().fmcuda_rope_append(C.byref(rope_args(**change)), None) == code


def attention_args(**change):
    a = PagedAttentionArgs(q=P, k_cache=P, v_cache=P, out=P, page_table=P, q_start=P, kv_len=P, q_token_stride=1024,
                           q_head_stride=128, out_token_stride=1024, out_head_stride=128, cache_page_stride=4096,
                           cache_head_stride=2048, cache_row_stride=128, page_table_stride=64, dtype=1, seqs=2, tokens=40,
                           heads=8, kv_heads=2, head_dim=128, n_pages=64, page_size=16, max_q_len=30, max_kv_len=1000,
                           causal=1, scale=0.1)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("code,change", [
    (ARG, {"dtype": 0}), (ARG, {"dtype": 3}), (SHAPE, {"head_dim": 0}), (SHAPE, {"head_dim": 100}), (SHAPE, {"head_dim": 136}),
    (SHAPE, {"heads": 7}), (SHAPE, {"kv_heads": 0}), (SHAPE, {"page_size": 0}), (SHAPE, {"page_size": 12}),
    (SHAPE, {"max_q_len": 41}), (SHAPE, {"max_kv_len": 1025}), (SHAPE, {"max_kv_len": 0xFFFFFFFF}),
    (ARG, {"window": 5, "causal": 0}), (ARG, {"scale": 0.0}), (ARG, {"scale": -1.0}), (ARG, {"scale": float("inf")}),
    (SHAPE, {"q_head_stride": 4}), (SHAPE, {"cache_row_stride": -8}), (SHAPE, {"tokens": 1 << 30, "max_q_len": 1}),
    (ARG, {"q": None}), (ARG, {"kv_len": None}), (ARG, {"out": P + 8}),
    (ARG, {"max_kv_len": 1 << 20, "page_table_stride": 1 << 16}),  # no workspace, and fragments to keep
    (OK, {"seqs": 0}), (OK, {"tokens": 0, "max_q_len": 0}), (OK, {"max_q_len": 0}),
])
def test_attention_refuses(code, change):
    assert load().fmcuda_paged_attention(C.byref(attention_args(**change)), None, 0, None) == code


def test_workspace_is_bounded_by_the_gpu_and_not_by_the_lengths():
    lib = load()

    def bytes_of(**change):
        v = C.c_uint64()
        assert lib.fmcuda_paged_attention_workspace_bytes(C.byref(attention_args(**change)), C.byref(v)) == OK
        return v.value

    long = dict(page_table_stride=1 << 20)
    assert bytes_of(tokens=1, seqs=1, max_q_len=1, max_kv_len=500) == 0  # one launch, no fragments
    a = bytes_of(tokens=1, seqs=1, max_q_len=1, max_kv_len=100000, **long)
    assert 0 < a == bytes_of(tokens=1, seqs=1, max_q_len=1, max_kv_len=10000000, **long) < 32 << 20
    b = bytes_of(tokens=2000, max_q_len=1500, max_kv_len=100000, **long)
    assert b <= 96 << 20
    assert bytes_of(seqs=0, tokens=0, max_q_len=0) == 0


# ---------------------------------------------------------------------------------- frequencies


def frequencies(rot, base, **scaling):
    lib = load()
    host, factor = (C.c_float * max(1, rot // 2))(), C.c_float()
    sc = RopeScaling(scaling.pop("kind", 0), scaling.pop("factor", 1.0), scaling.pop("trained_context", 0.0),
                     scaling.pop("fast", 0.0), scaling.pop("slow", 0.0))
    rc = lib.fmcuda_rope_frequencies(rot, base, C.byref(sc), host, C.byref(factor))
    return rc, list(host), factor.value


def close(got, want):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert abs(a - b) <= 2.0 ** -23 * abs(b)


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (80, 1e6)])
def test_plain_linear_and_base_frequencies(rot, base):
    plain = [base ** (-2 * i / rot) for i in range(rot // 2)]
    rc, got, factor = frequencies(rot, base)
    assert rc == 0 and factor == 1.0
    close(got, plain)
    rc, got, factor = frequencies(rot, base, kind=_lib.ROPE_LINEAR, factor=4.0)
    assert rc == 0 and factor == 1.0
    close(got, [f / 4 for f in plain])
    if rot > 2:
        rc, got, factor = frequencies(rot, base, kind=_lib.ROPE_BASE, factor=4.0)
        assert rc == 0 and factor == 1.0
        stretched = base * 4.0 ** (rot / (rot - 2))
        close(got, [stretched ** (-2 * i / rot) for i in range(rot // 2)])
        # the slowest pair turns a quarter as far, the fastest as before
        assert abs(got[-1] * 4 - plain[-1]) < 1e-6 * plain[-1] and got[0] == 1.0


def test_ramp_and_band_frequencies():
    rot, base, ctx = 128, 10000.0, 4096.0
    plain = [base ** (-2 * i / rot) for i in range(rot // 2)]
    rc, got, factor = frequencies(rot, base, kind=_lib.ROPE_RAMP, factor=8.0, trained_context=ctx, fast=32.0, slow=1.0)
    assert rc == 0 and abs(factor - (0.1 * math.log(8.0) + 1.0)) < 1e-6

    def pair_of(turns):
        return rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), rot - 1)
    want = []
    for i, f in enumerate(plain):
        part = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        want.append(f / 8 * part + f * (1 - part))
    close(got, want)
    assert got[0] == plain[0] and abs(got[-1] - plain[-1] / 8) < 1e-6 * plain[-1]
    rc, got, factor = frequencies(rot, base, kind=_lib.ROPE_BANDS, factor=8.0, trained_context=ctx, fast=4.0, slow=1.0)
    assert rc == 0 and factor == 1.0
    want = []
    for f in plain:
        turns = ctx * f / (2 * math.pi)
        keep = 1.0 if turns > 4 else 0.0 if turns < 1 else (turns - 1) / 3
        want.append(keep * f + (1 - keep) * f / 8)
    close(got, want)


@pytest.mark.parametrize("code,rot,base,scaling", [
    (SHAPE, 0, 1e4, {}), (SHAPE, 63, 1e4, {}), (SHAPE, 1026, 1e4, {}), (ARG, 64, 1.0, {}), (ARG, 64, float("nan"), {}),
    (ARG, 64, 1e4, {"kind": 9}), (ARG, 64, 1e4, {"kind": 1, "factor": 0.0}), (SHAPE, 2, 1e4, {"kind": 2, "factor": 2.0}),
    (ARG, 64, 1e4, {"kind": 3, "factor": 2.0}),
    (ARG, 64, 1e4, {"kind": 4, "factor": 2.0, "trained_context": 4096.0, "fast": 1.0, "slow": 4.0}),
])
def test_frequencies_refuse(code, rot, base, scaling):
    assert frequencies(rot, base, **scaling)[0] == code


def test_torch_calls_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from freemoe_b200 import attention

    for call in (lambda: attention.add_rms_norm(torch.zeros(2, 8), torch.ones(8)),
                 lambda: attention.add_rms_norm_fp8(torch.zeros(2, 8), torch.ones(8)),
                 lambda: attention.rope_append(torch.zeros(2, 1, 8), None, None, torch.zeros(2, dtype=torch.int32),
                                               torch.ones(4), None, None, None)):
        with pytest.raises(FmError) as e:
            call()
        assert e.value.code == ARG
    with pytest.raises(FmError) as e:
        attention.rope_frequencies(64, kind="unheard of")
    assert e.value.code == ARG
