"""Attention over a window behind which the first keys stay visible, against a plain
implementation in 64 bits; the tolerances are those of attention without them, derived in
test_attention_gpu.py (the same sums over other keys).

In the caches everything that no row of a call sees holds NaN, and the pages between the
first keys and the windows are freed: their table entries are -1.
"""
from __future__ import annotations

import math

import pytest
import torch

from freemoe_b200._lib import FmError
from test_attention_gpu import hold

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


class Batch:
    def __init__(self, lens, heads, kv_heads, dim, page, window, sinks, dtype=BF16, layout="hnd", seed=0, first_page=0,
                 q_scale=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.dim, self.dtype = lens, heads, kv_heads, dim, dtype
        self.window, self.sinks, self.scale = window, sinks, 1.0 / math.sqrt(dim)
        need = [-(-kv // page) for _, kv in lens]
        low = [max(0, kv - n - window + 1) for n, kv in lens]
        held = [[i for i in range(need[b]) if (i + 1) * page > low[b] or i * page < sinks] for b in range(len(lens))]
        pages = sum(map(len, held)) + 3 + first_page
        shape = (pages, kv_heads, page, dim) if layout == "hnd" else (pages, page, kv_heads, dim)
        caches = []
        for _ in range(2):
            c = torch.empty(shape, dtype=dtype, device="cuda")
            c[first_page:] = float("nan")
            caches.append(c if layout == "hnd" else c.permute(0, 2, 1, 3))
        self.k_cache, self.v_cache = caches
        order = iter((torch.randperm(pages - first_page, generator=g, device="cuda") + first_page).tolist())
        self.table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32, device="cuda")
        self.k, self.v = [], []
        for b, (n, kv) in enumerate(lens):
            k, v = (torch.randn(kv, kv_heads, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            for i in held[b]:
                pg = next(order)
                self.table[b, i] = pg
                at = torch.arange(i * page, min(kv, (i + 1) * page), device="cuda")
                at = at[(at >= low[b]) | (at < sinks)]
                self.k_cache[pg, :, at - i * page] = k[at].transpose(0, 1)
                self.v_cache[pg, :, at - i * page] = v[at].transpose(0, 1)
        self.q = (torch.randn(sum(n for n, _ in lens), heads, dim, generator=g, device="cuda") * q_scale).to(dtype)
        self.starts = [0]
        for n, _ in lens:
            self.starts.append(self.starts[-1] + n)
        self.q_start = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")

    def run(self, **change):
        from freemoe_b200 import attention

        args = dict(max_q_len=max(n for n, _ in self.lens), max_kv_len=max(kv for _, kv in self.lens), window=self.window,
                    sinks=self.sinks, scale=self.scale, return_lse=True)
        args.update(change)
        return attention.paged_attention(self.q, self.k_cache, self.v_cache, self.table, self.q_start, self.kv_len, **args)

    def exact(self):
        """o, sum p |v| and lse, in 64 bits."""
        group, parts = self.heads // self.kv_heads, ([], [], [])
        for b, (n, kv) in enumerate(self.lens):
            q = self.q[self.starts[b]:self.starts[b + 1]].double().view(n, self.kv_heads, group, self.dim)
            pos = torch.arange(kv - n, kv, device="cuda")[:, None]
            low = max(0, kv - n - self.window + 1)
            key = torch.arange(kv, device="cuda")
            key = key[(key >= low) | (key < self.sinks)]
            k, v = self.k[b][key].double(), self.v[b][key].double()
            seen = (key <= pos) & ((key > pos - self.window) | (key < self.sinks))
            s = torch.einsum("nhgd,khd->hgnk", q, k) * self.scale
            s.masked_fill_(~seen, -math.inf)
            lse = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
            parts[0].append(torch.einsum("hgnk,khd->nhgd", p, v).reshape(n, self.heads, self.dim))
            parts[1].append(torch.einsum("hgnk,khd->nhgd", p, v.abs()).reshape(n, self.heads, self.dim))
            parts[2].append(lse.permute(2, 0, 1).reshape(n, self.heads))
        return tuple(torch.cat(x) for x in parts)


def check(cuda, *args, **how):
    b = Batch(*args, **how)
    out, lse = b.run()
    assert cuda.device_status() == 0
    hold(b, out, lse)
    return b


@pytest.mark.parametrize("window", [1, 16, 100, 1000])
@pytest.mark.parametrize("sinks", [1, 4, 16, 17, 33, 130, 500, 5000])
@pytest.mark.parametrize("kv", [1, 5, 40, 133, 1100, 4000])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decoding(cuda, window, sinks, kv, dtype):
    check(cuda, [(1, kv)], 8, 2, 128, 16, window, sinks, dtype, seed=kv)
    check(cuda, [(1, kv)], 4, 2, 64, 8, window, sinks, dtype, seed=kv)


@pytest.mark.parametrize("seqs,window", [(3, 40), (20, 300), (64, 2000), (200, 150), (200, 700)])
@pytest.mark.parametrize("sinks", [3, 64, 257])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 32, 8), (64, 28, 4), (80, 16, 1)])
def test_decoding_together(cuda, seqs, window, sinks, dim, heads, kv_heads):
    """A cluster or a warp a unit, and even ranges, by the number of sequences and keys."""
    lens = [(1, 1 + (b * 977) % 3000) for b in range(seqs)]
    check(cuda, lens, heads, kv_heads, dim, 32, window, sinks, layout="nhd", seed=seqs)


def test_one_long_sequence(cuda):
    """Many fragments of one unit, some of them first keys alone."""
    check(cuda, [(1, 70000)], 16, 1, 128, 64, 20000, 9000, F16)
    check(cuda, [(2, 70001)], 8, 1, 64, 64, 300, 40000)


@pytest.mark.parametrize("window", [1, 17, 128, 200, 1000])
@pytest.mark.parametrize("sinks", [1, 16, 128, 129, 300, 1500])
@pytest.mark.parametrize("dim,heads,kv_heads,n,kv", [(128, 8, 2, 300, 300), (128, 4, 4, 700, 2900), (64, 28, 4, 129, 1500),
                                                     (96, 4, 1, 513, 4001), (64, 2, 2, 1200, 1200)])
def test_chunks(cuda, window, sinks, dim, heads, kv_heads, n, kv):
    check(cuda, [(n, kv)], heads, kv_heads, dim, 16, window, sinks, BF16 if n % 2 else F16, seed=n)


@pytest.mark.parametrize("page", [8, 24, 48, 128, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("window,sinks", [(100, 4), (700, 200)])
def test_pages(cuda, page, layout, window, sinks):
    check(cuda, [(300, 2000), (1, 1777), (40, 40), (129, 900)], 16, 4, 64, page, window, sinks, layout=layout, seed=page)
    check(cuda, [(1, 1), (1, 3001), (1, 777)], 16, 4, 128, page, window, sinks, layout=layout, seed=page)


@pytest.mark.parametrize("sinks", [5, 140, 600])
@pytest.mark.parametrize("window", [60, 1000])
def test_chunks_beside_decoding(cuda, sinks, window):
    for lens in ([(500, 3000), (1, 2500), (1, 17)], [(1, 4000)] * 30 + [(200, 5000)], [(90, 90), (2, 3000), (1, 130), (300, 301)],
                 [(64, 2000)] * 9 + [(1, 1900)] * 7, [(260, 1000)] * 40):
        check(cuda, lens, 8, 4, 128, 32, window, sinks, seed=sinks)
        check(cuda, lens, 28, 4, 64, 32, window, sinks, F16, seed=sinks)


def test_more_rows_than_keys(cuda):
    """Rows before the first key see nothing: zeros and -inf."""
    for n, kv in ((5, 3), (300, 200), (40, 0)):
        b = Batch([(n, max(kv, 1))], 4, 2, 64, 8, 50, 20)
        b.lens = [(n, kv)]
        b.k, b.v = [b.k[0][:kv]], [b.v[0][:kv]]
        b.kv_len[:] = kv
        out, lse = b.run(max_kv_len=max(kv, 1))
        assert cuda.device_status() == 0
        hold(b, out, lse)
        assert (out[:n - kv] == 0).all() and (lse[:n - kv] == -math.inf).all()


def test_sequences_without_rows(cuda):
    for lens in ([(0, 50), (1, 300), (0, 900), (130, 900), (0, 7)], [(0, 500), (1, 700), (0, 3)], [(0, 5)] * 200 + [(1, 400)]):
        check(cuda, lens, 8, 2, 64, 16, 70, 20)


def test_rows_behind_the_last_sequence_stay(cuda):
    """Rows past q_start's end, a batch's padding, are neither read nor written."""
    import ctypes as C

    from freemoe_b200._lib import PagedAttentionArgs, check as ok, load

    for lens in ([(1, 500), (1, 90)], [(150, 700), (1, 90)]):
        b = Batch(lens, 8, 2, 64, 16, 100, 9)
        used, tokens = b.starts[-1], b.starts[-1] + 300
        want, _ = b.run()
        q = torch.full((tokens, 8, 64), float("nan"), dtype=BF16, device="cuda")
        q[:used] = b.q
        out = torch.full((tokens, 8, 64), 7.0, dtype=BF16, device="cuda")
        a = PagedAttentionArgs(
            q=q.data_ptr(), k_cache=b.k_cache.data_ptr(), v_cache=b.v_cache.data_ptr(), out=out.data_ptr(),
            page_table=b.table.data_ptr(), q_start=b.q_start.data_ptr(), kv_len=b.kv_len.data_ptr(), q_token_stride=512,
            q_head_stride=64, out_token_stride=512, out_head_stride=64, cache_page_stride=b.k_cache.stride(0),
            cache_head_stride=b.k_cache.stride(1), cache_row_stride=b.k_cache.stride(2), page_table_stride=b.table.stride(0),
            dtype=1, seqs=len(lens), tokens=tokens, heads=8, kv_heads=2, head_dim=64, n_pages=b.k_cache.shape[0],
            page_size=16, max_q_len=max(n for n, _ in lens), max_kv_len=max(kv for _, kv in lens), causal=1, window=100,
            scale=b.scale)
        need = C.c_uint64()
        ok(load().fmcuda_paged_attention_sinks_workspace_bytes(C.byref(a), 9, C.byref(need)))
        ws = torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda")
        ok(load().fmcuda_paged_attention_sinks(C.byref(a), 9, ws.data_ptr(), need.value,
                                               torch.cuda.current_stream().cuda_stream))
        assert cuda.device_status() == 0 and (out[used:] == 7).all()
        off = (out[:used].float() - want.float()).abs()
        assert (off <= 2 * 2.0 ** -8 * (want.float().abs() + 4)).all()  # cut otherwise, perhaps: the weights' rounding


def test_sinks_that_add_nothing(cuda):
    """Where the window reaches the first keys, or covers all, the result is the window's; 0 is the call without them."""
    b = Batch([(130, 900), (1, 600)], 8, 2, 128, 16, 10000, 40)
    assert torch.equal(b.run()[0], b.run(sinks=0)[0])
    whole = Batch([(130, 900), (1, 600)], 8, 2, 128, 16, 10000, 40, seed=1)
    a, c = whole.run(window=7, sinks=(1 << 32) - 1)[0], whole.run()[0]
    u = 2.0 ** -8
    assert ((a.float() - c.float()).abs() <= 2 * u * (c.float().abs() + 4)).all()
    assert not torch.equal(whole.run(window=64, sinks=20)[0], whole.run(window=64, sinks=0)[0])
    assert cuda.device_status() == 0


def test_offsets_past_32_bits(cuda):
    check(cuda, [(1, 3000), (200, 1500)], 8, 8, 128, 64, 500, 70, first_page=33000)


def test_bad_pages_of_first_keys_are_reported(cuda):
    for lens in ([(1, 3000)], [(200, 3000)]):
        b = Batch(lens, 8, 2, 128, 16, 100, 40)
        b.table[0, 1] = -1
        b.run()
        assert cuda.device_status() == 26
        b.table[0, 1] = 10 ** 9
        b.run()
        assert cuda.device_status() == 26
        b = Batch(lens, 8, 2, 128, 16, 100, 16)
        b.table[0, 1] = 10 ** 9  # a freed page: not followed
        out, lse = b.run()
        assert cuda.device_status() == 0
        hold(b, out, lse)


def test_captured_replayed_and_on_another_stream(cuda):
    for lens in ([(1, 3000), (1, 100)], [(200, 1000), (1, 3000)]):
        b = Batch(lens, 8, 2, 128, 16, 300, 20)
        want, lse = b.run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got, _ = b.run(stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, _ = b.run()
        graph.replay()
        assert torch.equal(got, want)
        b.q.mul_(0.5)
        graph.replay()
        assert torch.equal(got, b.run()[0])
    assert cuda.device_status() == 0


def test_refusals(cuda):
    b = Batch([(1, 300)], 8, 2, 128, 16, 100, 4)

    def refused(code, **change):
        with pytest.raises(FmError) as e:
            b.run(**change)
        assert e.value.code == code

    refused(26, window=0)
    refused(26, sinks=-1)
    refused(8, sinks=1 << 32)
    refused(26, causal=False)
    refused(26, workspace=torch.empty(0, dtype=torch.uint8), window=100)


@pytest.mark.parametrize("sinks", [900, 901, (1 << 31) - 1, 1 << 31, (1 << 32) - 1])
@pytest.mark.parametrize("window", [1, 7, 128])
def test_more_first_keys_than_keys(cuda, sinks, window):
    """All of a sequence's keys, however many more are asked for: against 64 bits, no key lost or counted twice
    (one of 900 moves the log-sum-exp by 1e-3, 20 times what is allowed)."""
    b = Batch([(130, 900), (1, 600), (900, 900)], 8, 2, 128, 16, 10000, 40, seed=1)
    out, lse = b.run(window=window, sinks=sinks)
    assert cuda.device_status() == 0
    b.window, b.sinks = window, sinks
    hold(b, out, lse)
    d = Batch([(1, 900), (1, 600)], 8, 2, 64, 16, 10000, 40, F16, seed=2)
    out, lse = d.run(window=window, sinks=sinks)
    d.window, d.sinks = window, sinks
    hold(d, out, lse)


@pytest.mark.parametrize("lens", [[(1, 500), (1, 90)], [(150, 700), (1, 90)], [(0, 30), (40, 40)]])
def test_padded_batches(cuda, lens):
    """Rows behind the last sequence change nothing: the others against 64 bits."""
    b = Batch(lens, 8, 2, 64, 16, 100, 9)
    used = b.starts[-1]
    b.q = torch.cat([b.q, torch.full((300, 8, 64), float("nan"), dtype=BF16, device="cuda")])
    out, lse = b.run()
    assert cuda.device_status() == 0
    b.q = b.q[:used]
    hold(b, out[:used], lse[:used])
