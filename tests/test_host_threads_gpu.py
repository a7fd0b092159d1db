"""The C entries from two host threads at once, each with a stream and buffers of its own: no call
is refused or changed by what the other thread asks for.

The threads call one kernel with different amounts of shared memory, whose limit is an attribute
of the kernel and not of the call.  (ctypes releases the interpreter's lock for a call.)
"""
from __future__ import annotations

import ctypes as C
import threading

import pytest
import torch

from freemoe_b200 import load
from freemoe_b200._lib import NormAddNormArgs, PagedAttentionArgs, RmsNormArgs

pytestmark = pytest.mark.gpu

CALLS = 3000


class Norms:
    """Many rows of the norms around a block."""

    def __init__(self, d, tokens=300):
        g = torch.Generator(device="cuda").manual_seed(d)
        self.x, self.r = (torch.randn(tokens, d, generator=g, device="cuda").bfloat16() for _ in range(2))
        self.w, self.y, self.h = torch.ones(d, device="cuda"), torch.empty_like(self.x), torch.empty_like(self.x)
        self.out = (self.y, self.h)
        self.args = NormAddNormArgs(
            x=self.x.data_ptr(), post_weight=self.w.data_ptr(), residual=self.r.data_ptr(), pre_weight=self.w.data_ptr(),
            y=self.y.data_ptr(), residual_out=self.h.data_ptr(), x_stride=d, residual_stride=d, y_stride=d, x_dtype=1,
            residual_dtype=1, weight_dtype=0, y_dtype=1, tokens=tokens, d_model=d, scale=1.0, residual_scale=1.0,
            epsilon=1e-5)

    def call(self, lib, stream):
        return lib.fmcuda_norm_add_norm(C.byref(self.args), stream)


class Norm:
    """Many rows of the norm."""

    def __init__(self, d, tokens=300):
        g = torch.Generator(device="cuda").manual_seed(d)
        self.x = torch.randn(tokens, d, generator=g, device="cuda").bfloat16()
        self.w, self.y = torch.ones(d, device="cuda"), torch.empty_like(self.x)
        self.out = (self.y,)
        self.args = RmsNormArgs(x=self.x.data_ptr(), weight=self.w.data_ptr(), y=self.y.data_ptr(), x_stride=d, y_stride=d,
                                x_dtype=1, weight_dtype=0, y_dtype=1, tokens=tokens, d_model=d, epsilon=1e-5)

    def call(self, lib, stream):
        return lib.fmcuda_add_rms_norm(C.byref(self.args), stream)


class Decoding:
    """Many short sequences: a warp each, and more warps to a CTA where there are more."""

    def __init__(self, seqs, kv=60, window=0, sinks=0):
        g = torch.Generator(device="cuda").manual_seed(seqs)
        self.q = torch.randn(seqs, 8, 128, generator=g, device="cuda").bfloat16()
        self.k, self.v = (torch.randn(seqs * 4, 8, 16, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
        self.table = torch.arange(seqs * 4, dtype=torch.int32, device="cuda").view(seqs, 4)
        self.starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
        self.lens = torch.full((seqs,), kv, dtype=torch.int32, device="cuda")
        self.o, self.sinks = torch.empty_like(self.q), sinks
        self.out = (self.o,)
        self.args = PagedAttentionArgs(
            q=self.q.data_ptr(), k_cache=self.k.data_ptr(), v_cache=self.v.data_ptr(), out=self.o.data_ptr(),
            page_table=self.table.data_ptr(), q_start=self.starts.data_ptr(), kv_len=self.lens.data_ptr(),
            q_token_stride=1024, q_head_stride=128, out_token_stride=1024, out_head_stride=128,
            cache_page_stride=16384, cache_head_stride=2048, cache_row_stride=128, page_table_stride=4, dtype=1, seqs=seqs,
            tokens=seqs, heads=8, kv_heads=8, head_dim=128, n_pages=seqs * 4, page_size=16, max_q_len=1, max_kv_len=kv,
            causal=1, window=window, scale=0.1)
        need = C.c_uint64()
        assert load().fmcuda_paged_attention_sinks_workspace_bytes(C.byref(self.args), sinks, C.byref(need)) == 0
        self.workspace = torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda")
        self.bytes = need.value

    def call(self, lib, stream):
        return lib.fmcuda_paged_attention_sinks(C.byref(self.args), self.sinks, self.workspace.data_ptr(), self.bytes, stream)


class Experts:
    """The grouped products of a batch of tokens, whose tables grow with the experts."""

    def __init__(self, experts, tokens=64, top_k=4, d=512, ffn=256):
        from freemoe_b200 import TYPE_Q8_0, hotpath

        g = torch.Generator(device="cuda").manual_seed(experts)
        self.x = torch.randn(tokens, d, generator=g, device="cuda").bfloat16()
        self.logits = torch.randn(tokens, experts, generator=g, device="cuda")
        self.slot = torch.cat([hotpath.synth_weights(TYPE_Q8_0, rows, cols, i, 0.05)
                               for i, (rows, cols) in enumerate(((ffn, d), (ffn, d), (d, ffn)))])
        self.table, self.y = hotpath.slot_table([self.slot] * experts, "cuda"), torch.empty(tokens, d, device="cuda")
        self.out = (self.y,)
        part = hotpath.row_bytes(TYPE_Q8_0, d) * ffn
        self.args = hotpath.moe_args(self.x, self.logits, self.table, experts=experts, top_k=top_k, d_model=d, ffn=ffn,
                                     gate_type=TYPE_Q8_0, up_type=TYPE_Q8_0, down_type=TYPE_Q8_0, up_offset=part,
                                     down_offset=2 * part, y=self.y)
        self.workspace = torch.empty(hotpath.moe_prefill_workspace_bytes(tokens, experts, top_k, d, ffn),
                                     dtype=torch.uint8, device="cuda")

    def call(self, lib, stream):
        return lib.fmcuda_moe_prefill(C.byref(self.args), None, self.workspace.data_ptr(), self.workspace.numel(), stream)


@pytest.mark.parametrize("make", [
    lambda: (Norms(6144), Norms(8192)), lambda: (Norms(5120), Norms(7168)), lambda: (Norms(9216), Norms(16384)),
    lambda: (Norm(12288), Norm(16384)), lambda: (Norm(9216), Norm(12288)), lambda: (Decoding(40), Decoding(160)),
    lambda: (Decoding(40, window=20, sinks=3), Decoding(160, window=20, sinks=3)), lambda: (Experts(8), Experts(700)),
], ids=["norms 6144 8192", "norms 5120 7168", "norms 9216 16384", "norm 12288 16384", "norm 9216 12288", "decoding",
        "decoding with first keys", "experts"])
def test_two_threads(cuda, make):
    lib, jobs = load(), make()
    streams = [torch.cuda.Stream() for _ in jobs]
    want = []
    for job in jobs:
        assert job.call(lib, torch.cuda.current_stream().cuda_stream) == 0
        want.append([t.clone() for t in job.out])
    torch.cuda.synchronize()
    codes = [set(), set()]
    go = threading.Barrier(2)

    def many(i):
        torch.cuda.set_device(0)
        go.wait()
        for _ in range(CALLS):
            codes[i].add(jobs[i].call(lib, streams[i].cuda_stream))

    threads = [threading.Thread(target=many, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [{0}, {0}], lib.fmcuda_last_error()
    for job, values in zip(jobs, want):
        assert all(torch.equal(a, b) for a, b in zip(job.out, values))
    assert cuda.device_status() == 0
