"""What the attention side hands on and takes at its edges, without a GPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from freemoe_b200 import TYPE_Q8_0, hotpath, load
from freemoe_b200._lib import X_BF16, X_F32, FmError
from test_attention_cpu import P, attention_args, rope_args

OK, SHAPE, ARG = 0, 8, 26
UNREAD = [torch.float16, torch.float8_e4m3fn, torch.float64]  # rows that no product, expert or exchange reads


def refused(code, call):
    with pytest.raises(FmError) as e:
        call()
    assert e.value.code == code


@pytest.mark.parametrize("dtype", UNREAD)
def test_experts_refuse_rows_that_they_do_not_read(dtype):
    x, logits = torch.zeros(3, 64).to(dtype), torch.zeros(3, 2)
    slots = [torch.zeros(3 * 64 * 68, dtype=torch.uint8) for _ in range(2)]
    table, y = hotpath.slot_table(slots, "cpu"), torch.zeros(3, 64)

    def args(rows):
        return hotpath.moe_args(rows, logits, table, experts=2, top_k=1, d_model=64, ffn=64, gate_type=TYPE_Q8_0,
                                up_type=TYPE_Q8_0, down_type=TYPE_Q8_0, up_offset=0, down_offset=0, y=y)

    assert args(x.float()).x_dtype == X_F32 and args(x.bfloat16()).x_dtype == X_BF16
    refused(ARG, lambda: args(x))
    for block in (hotpath.moe_block, hotpath.moe_prefill):
        refused(ARG, lambda: block(x, logits, slots, top_k=1, ffn=64, gate_type=TYPE_Q8_0))
    refused(ARG, lambda: hotpath.gemv_quant(TYPE_Q8_0, slots[0], x, 64, 64))


@pytest.mark.parametrize("dtype", UNREAD)
def test_exchanges_refuse_rows_that_they_do_not_read(dtype):
    from freemoe_b200.ep import DeviceOps

    ops = DeviceOps(experts_total=4, top_k=2, d_model=64, ffn=64, gate_type=TYPE_Q8_0, up_type=TYPE_Q8_0,
                    down_type=TYPE_Q8_0, local_slots=[], up_offset=0, down_offset=0)
    ops.world, ops.rank, ops.capacity, ops.timeout_ms = 2, 0, 16, 0
    x, ids, w = torch.zeros(3, 64).to(dtype), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    refused(ARG, lambda: ops.dispatch(ids, x, 2))
    refused(ARG, lambda: ops.dispatch_rows(ids, w, x, 2))
    refused(ARG, lambda: ops.p2p_dispatch(ids, w, x, 1))


def test_a_rotation_of_no_tokens_takes_null_rows():
    """The rows and slots of an empty batch have no address; its caches have."""
    lib = load()

    def code(**change):
        return lib.fmcuda_rope_append(C.byref(rope_args(tokens=0, q=None, k=None, v=None, q_out=None, positions=None,
                                                        slots=None, **change)), None)

    assert code() == OK and code(k_cache=None, v_cache=None) == OK
    assert code(in_dtype=3) == ARG and code(page_size=0) == SHAPE and code(rot_dim=63) == SHAPE


def test_the_library_needs_no_torch(tmp_path, monkeypatch, capsys):
    """Without torch the entry points for its tensors are left out, and the library is built."""
    import sys

    from freemoe_b200 import build

    monkeypatch.setattr(build, "PKG", tmp_path)  # no entry points there yet
    monkeypatch.setitem(sys.modules, "torch", None)  # importing it fails
    assert build.build() == build.LIB and build.LIB.exists()
    assert "torch is not installed" in capsys.readouterr().err
    assert not list(tmp_path.glob("*.so"))


def test_entry_points_are_those_of_this_torch(monkeypatch):
    from freemoe_b200 import attention, build

    mine = build.torch_calls_path()
    assert mine.exists() and mine.name.startswith("_torch_calls.")
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.torch_calls_path() != mine
    with pytest.raises(FmError) as e:
        attention._Calls().add_rms_norm
    assert e.value.code == 24 and "0.0.1" in str(e.value)


@pytest.mark.parametrize("name,off", [("positions", 2), ("slots", 4), ("inv_freq", 1)])
def test_rotation_refuses_arrays_that_are_not_aligned(name, off):
    lib, args = load(), rope_args()
    setattr(args, name, P + off)
    assert lib.fmcuda_rope_append(C.byref(args), None) == ARG
    assert b"aligned" in lib.fmcuda_last_error()


@pytest.mark.parametrize("name,off", [("lse", 2), ("page_table", 1), ("q_start", 2), ("kv_len", 3)])
def test_attention_refuses_arrays_that_are_not_aligned(name, off):
    lib, args = load(), attention_args()
    setattr(args, name, P + off)
    assert lib.fmcuda_paged_attention(C.byref(args), None, 0, None) == ARG
    assert b"aligned to their values" in lib.fmcuda_last_error()
