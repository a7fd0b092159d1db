"""The operators around the attention side without a GPU: refusals made before any CUDA
call, the argument structs' layouts, and the axes of rotary pairs."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest
import torch

from conftest import ROOT
from freemoe_b200 import attention, hotpath, load
from freemoe_b200._lib import FmError, NormAddNormArgs, TokenLogprobsArgs
from test_attention_cpu import P, attention_args, rope_args

OK, SHAPE, ARG = 0, 8, 26


@pytest.mark.parametrize("name,struct", [("fmcuda_norm_add_norm_args", NormAddNormArgs),
                                         ("fmcuda_token_logprobs_args", TokenLogprobsArgs)])
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


# ------------------------------------------------------------------------- norms around a block


def pair_args(**change):
    a = NormAddNormArgs(x=P, post_weight=P, gate=P, residual=P, pre_weight=P, y=P, residual_out=P, scales=P, x_stride=64,
                        residual_stride=64, y_stride=64, gate_stride=64, x_dtype=1, tokens=4, d_model=64, scale=1.0,
                        residual_scale=1.0, epsilon=1e-5)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("code,change", [
    (ARG, {"x": None}), (ARG, {"residual": None}), (ARG, {"y": None}), (ARG, {"pre_weight": None, "residual_out": None}),
    (SHAPE, {"d_model": 0}), (SHAPE, {"d_model": (1 << 24) + 1}), (ARG, {"x_dtype": 3}), (ARG, {"x_dtype": -1}),
    (ARG, {"residual_dtype": 3}), (ARG, {"weight_dtype": 3}), (ARG, {"gate_dtype": 4}), (ARG, {"y_dtype": 4}),
    (ARG, {"y_dtype": 3, "scales": None}), (SHAPE, {"x_stride": 63}), (SHAPE, {"y_stride": 0}),
    (SHAPE, {"residual_stride": 10}), (SHAPE, {"gate_stride": 63}), (SHAPE, {"gate_stride": -64}),
    (SHAPE, {"gate_per_token": 1, "gate_stride": -1}), (ARG, {"epsilon": -1.0}), (ARG, {"epsilon": float("nan")}),
    (ARG, {"scale": float("nan")}), (ARG, {"residual_scale": float("inf")}), (ARG, {"x": P + 1}), (ARG, {"y": P + 2}),
    (ARG, {"gate": P + 2}), (ARG, {"post_weight": P + 2}), (ARG, {"residual": P + 1}), (ARG, {"residual_out": P + 2}),
    (ARG, {"y_dtype": 3, "scales": P + 2}), (OK, {"tokens": 0}), (OK, {"tokens": 0, "x": None, "y": None}),
])
def test_norms_refuse(code, change):
    lib = load()
    assert lib.fmcuda_norm_add_norm(C.byref(pair_args(**change)), None) == code
    if code:
        assert lib.fmcuda_last_error()


# ------------------------------------------------------------------------------- rotary axes


@pytest.mark.parametrize("code,change", [
    (SHAPE, {"axes": 0}), (SHAPE, {"axes": 9}), (ARG, {"axis": None}), (SHAPE, {"stride": 2}), (SHAPE, {"stride": -3}),
    (OK, {"tokens": 0, "axis": None}), (SHAPE, {"head_dim": 0}), (ARG, {"positions": None}), (ARG, {"positions": P + 2}),
])
def test_rotation_of_several_axes_refuses(code, change):
    entry = {"axes": 3, "axis": P, "stride": 3}
    for k in list(change):
        if k in entry:
            entry[k] = change.pop(k)
    assert load().fmcuda_rope_append_axes(C.byref(rope_args(**change)), entry["axis"], entry["axes"], entry["stride"],
                                          None) == code


def test_axes_in_blocks_and_in_turn():
    assert attention.rope_axes((2, 3, 1), device="cpu").tolist() == [0, 0, 1, 1, 1, 2]
    assert attention.rope_axes((2, 3, 1), "turn", device="cpu").tolist() == [0, 1, 2, 0, 1, 1]
    assert attention.rope_axes((0, 2), "turn", device="cpu").tolist() == [1, 1]
    turn = attention.rope_axes((24, 20, 20), "turn", device="cpu").tolist()
    assert turn[:60] == [0, 1, 2] * 20 and turn[60:] == [0] * 4
    assert attention.rope_axes((512,), device="cpu").dtype == torch.uint8


@pytest.mark.parametrize("code,sections,order", [
    (SHAPE, (), "blocks"), (SHAPE, (0, 0), "blocks"), (SHAPE, (1,) * 9, "turn"), (SHAPE, (513,), "blocks"),
    (SHAPE, (3, -1), "blocks"), (ARG, (3, 1), "rows"),
])
def test_axes_refuse(code, sections, order):
    with pytest.raises(FmError) as e:
        attention.rope_axes(sections, order, device="cpu")
    assert e.value.code == code


def test_axes_of_the_c_entry():
    lib, out, sections = load(), (C.c_uint8 * 4)(), (C.c_uint32 * 2)(1, 3)
    assert lib.fmcuda_rope_axes(sections, 2, 0, 8, out) == OK and list(out) == [0, 1, 1, 1]
    assert lib.fmcuda_rope_axes(sections, 2, 0, 10, out) == SHAPE  # not the pairs' number
    assert lib.fmcuda_rope_axes((C.c_uint32 * 2)(0xFFFFFFFF, 5), 2, 0, 8, out) == SHAPE
    assert lib.fmcuda_rope_axes(None, 2, 0, 8, out) == ARG and lib.fmcuda_rope_axes(sections, 2, 0, 8, None) == ARG


# -------------------------------------------------------------------- first keys behind a window


@pytest.mark.parametrize("code,sinks,change", [
    (ARG, 4, {}), (ARG, 4, {"causal": 0}), (ARG, 4, {"window": 9, "causal": 0}), (SHAPE, 4, {"window": 9, "head_dim": 100}),
    (SHAPE, 4, {"window": 9, "max_kv_len": 1025}), (ARG, 4, {"window": 9, "kv_len": None}), (ARG, 4, {"window": 9, "lse": P + 2}),
    (ARG, 1 << 20, {"window": 9, "max_kv_len": 1 << 20, "page_table_stride": 1 << 16}),  # no workspace, and fragments to keep
    (OK, 4, {"window": 9, "seqs": 0}), (OK, 0xFFFFFFFF, {"window": 9, "tokens": 0, "max_q_len": 0}),
])
def test_attention_with_first_keys_refuses(code, sinks, change):
    assert load().fmcuda_paged_attention_sinks(C.byref(attention_args(**change)), sinks, None, 0, None) == code


def test_workspace_with_first_keys():
    lib = load()

    def bytes_of(sinks, **change):
        v = C.c_uint64()
        assert lib.fmcuda_paged_attention_sinks_workspace_bytes(C.byref(attention_args(**change)), sinks, C.byref(v)) == OK
        return v.value

    plain = C.c_uint64()
    assert lib.fmcuda_paged_attention_workspace_bytes(C.byref(attention_args(window=50)), C.byref(plain)) == OK
    assert bytes_of(0, window=50) == plain.value
    long = dict(tokens=1, seqs=1, max_q_len=1, max_kv_len=10000000, page_table_stride=1 << 20)
    assert bytes_of(4, window=100, **long) == 0  # few keys are seen: one launch, no fragments
    assert 0 < bytes_of(0xFFFFFFFF, window=100, **long) < 32 << 20
    v = C.c_uint64()
    assert lib.fmcuda_paged_attention_sinks_workspace_bytes(C.byref(attention_args()), 1, C.byref(v)) == ARG
    assert lib.fmcuda_paged_attention_sinks_workspace_bytes(None, 1, C.byref(v)) == ARG
    assert lib.fmcuda_paged_attention_sinks_workspace_bytes(C.byref(attention_args()), 0, None) == ARG


# ---------------------------------------------------------------------- probabilities of tokens


@pytest.mark.parametrize("code,change", [
    (ARG, {"logits": None}), (ARG, {"token": None}), (ARG, {"logprobs": None}), (ARG, {"entropy": None}),
    (ARG, {"top_logprobs": None}), (ARG, {"top_ids": None}), (ARG, {"dtype": 3}), (ARG, {"dtype": -1}),
    (SHAPE, {"vocab": 0}), (SHAPE, {"vocab": (1 << 30) + 1}), (ARG, {"top": 33}), (ARG, {"vocab": 4, "top": 5}),
    (SHAPE, {"row_stride": 99}), (SHAPE, {"tokens": 1 << 31}), (ARG, {"scale": 0.0}), (ARG, {"scale": float("inf")}),
    (ARG, {"scale": float("nan")}), (ARG, {"logits": P + 1}), (ARG, {"token": P + 2}), (ARG, {"top_ids": P + 1}),
    (OK, {"tokens": 0}), (OK, {"tokens": 0, "logits": None}),
])
def test_logprobs_refuse(code, change):
    a = TokenLogprobsArgs(logits=P, token=P, logprobs=P, entropy=P, top_logprobs=P, top_ids=P, row_stride=100, scale=1.0,
                          dtype=1, tokens=3, vocab=100, top=5)
    for k, v in change.items():
        setattr(a, k, v)
    lib = load()
    assert lib.fmcuda_token_logprobs(C.byref(a), None) == code
    assert lib.fmcuda_token_logprobs(None, None) == ARG


def test_torch_calls_refuse_host_tensors():
    for call in (lambda: attention.norm_add_norm(torch.zeros(2, 8), torch.ones(8), torch.zeros(2, 8), torch.ones(8)),
                 lambda: hotpath.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)),
                 lambda: attention.norm_add_norm_fp8(torch.zeros(2, 8), None, torch.zeros(2, 8), torch.ones(8)),
                 lambda: attention.rope_append(torch.zeros(2, 1, 8), None, None, torch.zeros(1, 2, dtype=torch.int32),
                                               torch.ones(4), None, None, None,
                                               axes=torch.zeros(4, dtype=torch.uint8))):
        with pytest.raises(FmError) as e:
            call()
        assert e.value.code == ARG
