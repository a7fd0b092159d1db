"""What the kernel before wrote is what the next one reads, though it begins before that one's end
(launch.cuh): chains over the same buffers without a wait between their calls, against the same
calls with one after each."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from freemoe_b200 import load
from freemoe_b200._lib import PagedAttentionArgs, RmsNormArgs, TokenLogprobsArgs

pytestmark = pytest.mark.gpu

ROUNDS = 60


def both_ways(step):
    """`step(i)` enqueues round i and returns its result: with a wait after each call, then without."""
    results = []
    for wait in (True, False):
        outs = [step(i, torch.cuda.synchronize if wait else lambda: None) for i in range(ROUNDS)]
        torch.cuda.synchronize()
        results.append([t.clone() for out in outs for t in out])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert len({float(t.double().sum()) for t in results[0]}) > ROUNDS // 2  # the rounds differ


@pytest.mark.parametrize("rows,vocab", [(1, 8192), (3, 16000), (700, 4096), (2000, 1023)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_of_a_norm(cuda, rows, vocab, dtype):
    lib, stream, kind = load(), torch.cuda.current_stream().cuda_stream, 0 if dtype == torch.float32 else 1
    g = torch.Generator(device="cuda").manual_seed(rows)
    inputs = [torch.randn(rows, vocab, generator=g, device="cuda").to(dtype) for _ in range(4)]
    weights = [torch.rand(vocab, generator=g, device="cuda") + i for i in range(3)]
    logits, tokens = torch.empty(rows, vocab, dtype=dtype, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    stores = [[torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, 4, device="cuda"),
               torch.empty(rows, 4, dtype=torch.int32, device="cuda")] for _ in range(ROUNDS)]

    def step(i, done):
        x, w, out = inputs[i % 4], weights[i % 3], stores[i]
        norm = RmsNormArgs(x=x.data_ptr(), weight=w.data_ptr(), y=logits.data_ptr(), x_stride=vocab, y_stride=vocab,
                           x_dtype=kind, weight_dtype=0, y_dtype=kind, tokens=rows, d_model=vocab, epsilon=1e-5)
        score = TokenLogprobsArgs(
            logits=logits.data_ptr(), token=tokens.data_ptr(), logprobs=out[0].data_ptr(), entropy=out[1].data_ptr(),
            top_logprobs=out[2].data_ptr(), top_ids=out[3].data_ptr(), row_stride=vocab, scale=1.0 + i / 100, dtype=kind,
            tokens=rows, vocab=vocab, top=4)
        assert lib.fmcuda_add_rms_norm(C.byref(norm), stream) == 0
        done()
        assert lib.fmcuda_token_logprobs(C.byref(score), stream) == 0
        done()
        return out

    both_ways(step)


@pytest.mark.parametrize("lens", [[(1, 700)], [(1, 40)] * 30, [(300, 900), (1, 500)], [(1, 2000)] * 60])
@pytest.mark.parametrize("sinks", [0, 9])
def test_attention_of_a_norm(cuda, lens, sinks):
    """The queries and then the keys come from the kernel before."""
    lib, stream, dim, heads = load(), torch.cuda.current_stream().cuda_stream, 64, 4
    g = torch.Generator(device="cuda").manual_seed(len(lens))
    rows, pages = sum(n for n, _ in lens), [-(-kv // 16) for _, kv in lens]
    table = torch.zeros(len(lens), max(pages), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    q, k, v = (torch.empty(n, dim, dtype=torch.bfloat16, device="cuda") for n in (rows * heads, at * 16, at * 16))
    inputs = [torch.randn(max(len(q), len(k)), dim, generator=g, device="cuda").bfloat16() for _ in range(3)]
    weights = [torch.rand(dim, generator=g, device="cuda") + i for i in range(2)]
    starts = torch.tensor([sum(n for n, _ in lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
    outs = torch.empty(ROUNDS, rows, heads, dim, dtype=torch.bfloat16, device="cuda")
    most_q, most_kv = max(n for n, _ in lens), max(kv for _, kv in lens)

    def attention(out, scale=0.1):
        return PagedAttentionArgs(
            q=q.data_ptr(), k_cache=k.data_ptr(), v_cache=v.data_ptr(), out=out.data_ptr(), page_table=table.data_ptr(),
            q_start=starts.data_ptr(), kv_len=kv_len.data_ptr(), q_token_stride=heads * dim, q_head_stride=dim,
            out_token_stride=heads * dim, out_head_stride=dim, cache_page_stride=16 * dim, cache_head_stride=16 * dim,
            cache_row_stride=dim, page_table_stride=table.stride(0), dtype=1, seqs=len(lens), tokens=rows, heads=heads,
            kv_heads=1, head_dim=dim, n_pages=at, page_size=16, max_q_len=most_q, max_kv_len=most_kv, causal=1,
            window=300 if sinks else 0, scale=scale)

    need = C.c_uint64()
    assert lib.fmcuda_paged_attention_sinks_workspace_bytes(C.byref(attention(outs[0])), sinks, C.byref(need)) == 0
    workspace = torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda")

    def norm(x, w, y):
        a = RmsNormArgs(x=x.data_ptr(), weight=w.data_ptr(), y=y.data_ptr(), x_stride=dim, y_stride=dim, x_dtype=1,
                        weight_dtype=0, y_dtype=1, tokens=len(y), d_model=dim, epsilon=1e-5)
        assert lib.fmcuda_add_rms_norm(C.byref(a), stream) == 0

    def step(i, done):
        for j, y in enumerate((v, k, q) if i % 2 else (v, q, k)):
            norm(inputs[(i + j) % 3], weights[(i + j) % 2], y)
            done()
        a = attention(outs[i], 0.1 + i / 100)
        assert lib.fmcuda_paged_attention_sinks(C.byref(a), sinks, workspace.data_ptr(), need.value, stream) == 0
        done()
        return [outs[i]]

    both_ways(step)
    assert cuda.device_status() == 0
