"""Attention over a paged cache against a plain implementation in 64 bits.

Tolerances, derived before the first run.  u is half a unit in the last place of
the 16-bit type (2^-8 bf16, 2^-11 f16).  The kernels round each softmax weight
once (error <= u of it) and the result once; scores and sums are f32.  With
A = sum_i p_i |v_i| (p the exact weights) an element is within
    u |o| + u (1 + 2u) A + 4e-5 A
of the exact o: 4e-5 covers a 128-term f32 dot product of scores below 32 (its
error, as an exponent, is a relative error of the weight) and the hardware
exponential.  f16 weights below 2^-14 lose bits: n keys add n 2^-25 max|v|.
The f32 log-sum-exp is within 4e-5 + 1e-6 |lse|.
"""
from __future__ import annotations

import math

import pytest
import torch

from freemoe_b200._lib import FmError

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Batch:
    """A batch of sequences in a paged cache whose unseen rows hold NaN."""

    def __init__(self, lens, heads, kv_heads, dim, page, dtype=torch.bfloat16, layout="hnd", seed=0, spare=3,
                 q_scale=1.0, first_page=0, window=0, causal=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.dim, self.page, self.dtype = lens, heads, kv_heads, dim, page, dtype
        self.window, self.causal = window, causal
        tokens = sum(n for n, _ in lens)
        need = [-(-kv // page) for _, kv in lens]
        pages = sum(need) + spare + first_page
        shape = (pages, kv_heads, page, dim) if layout == "hnd" else (pages, page, kv_heads, dim)
        caches = []
        for _ in range(2):
            c = torch.empty(shape, dtype=dtype, device="cuda")
            c[first_page:] = float("nan")
            caches.append(c if layout == "hnd" else c.permute(0, 2, 1, 3))
        self.k_cache, self.v_cache = caches
        order = (torch.randperm(sum(need) + spare, generator=g, device="cuda") + first_page).tolist()
        width = max(need + [1])
        # unused entries must not be followed
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        self.k, self.v = [], []
        at = 0
        for b, (n, kv) in enumerate(lens):
            k = torch.randn(kv, kv_heads, dim, generator=g, device="cuda").to(dtype)
            v = torch.randn(kv, kv_heads, dim, generator=g, device="cuda").to(dtype)
            self.k.append(k)
            self.v.append(v)
            pages_b = order[at:at + need[b]]
            at += need[b]
            first_seen = max(0, kv - n - window + 1) if window else 0
            for i, pg in enumerate(pages_b):
                lo, hi = i * page, min(kv, (i + 1) * page)
                if hi <= first_seen:
                    continue  # a page before the window: freed, its entry is not followed
                self.table[b, i] = pg
                lo2 = max(lo, first_seen)
                self.k_cache[pg, :, lo2 - lo:hi - lo] = k[lo2:hi].transpose(0, 1)
                self.v_cache[pg, :, lo2 - lo:hi - lo] = v[lo2:hi].transpose(0, 1)
        self.q = (torch.randn(tokens, heads, dim, generator=g, device="cuda") * q_scale).to(dtype)
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        self.scale = 1.0 / math.sqrt(dim)

    def run(self, **kw):
        from freemoe_b200 import attention

        args = dict(max_q_len=max([n for n, _ in self.lens] + [0]), max_kv_len=max(kv for _, kv in self.lens),
                    causal=self.causal, window=self.window, scale=self.scale, return_lse=True)
        args.update(kw)
        return attention.paged_attention(self.q, self.k_cache, self.v_cache, self.table, self.q_start, self.kv_len,
                                         **args)

    def exact(self):
        """o, A = sum p |v|, lse and the number of keys, in 64 bits."""
        group = self.heads // self.kv_heads
        outs, sizes, lses = [], [], []
        at = 0
        for b, (n, kv) in enumerate(self.lens):
            q = self.q[at:at + n].double().view(n, self.kv_heads, group, self.dim)
            at += n
            s = torch.einsum("nhgd,khd->hgnk", q, self.k[b].double()) * self.scale
            pos = torch.arange(kv - n, kv, device="cuda")[:, None]
            key = torch.arange(kv, device="cuda")[None]
            hidden = torch.zeros(n, kv, dtype=torch.bool, device="cuda")
            if self.causal:
                hidden |= key > pos
            if self.window:
                hidden |= key <= pos - self.window
            s.masked_fill_(hidden, -math.inf)
            lse = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
            v = self.v[b].double()
            outs.append(torch.einsum("hgnk,khd->nhgd", p, v).reshape(n, self.heads, self.dim))
            sizes.append(torch.einsum("hgnk,khd->nhgd", p, v.abs()).reshape(n, self.heads, self.dim))
            lses.append(lse.permute(2, 0, 1).reshape(n, self.heads))
        return torch.cat(outs), torch.cat(sizes), torch.cat(lses)


def hold(batch, got, lse, o=None):
    o, size, exact_lse = batch.exact() if o is None else o
    u = HALF_ULP[batch.dtype]
    keys = max(kv for _, kv in batch.lens)
    tol = u * o.abs() + (u * (1 + 2 * u) + 4e-5) * size
    if batch.dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * 6.0 + 2.0 ** -24
    assert torch.isfinite(got).all()
    off = (got.double() - o).abs() - tol
    assert off.max().item() <= 0, f"{off.max().item()} past the bound"
    empty = exact_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (got[empty] == 0).all()
    d = (lse.double() - exact_lse)[~empty].abs()
    assert (d <= 4e-5 + 1e-6 * exact_lse[~empty].abs()).all()


def check(batch, cuda, **kw):
    out, lse = batch.run(**kw)
    hold(batch, out, lse)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 127, 128, 129, 1000])
def test_decode_lengths(cuda, dtype, kv):
    check(Batch([(1, kv)], 8, 2, 128, 16, dtype, seed=kv), cuda)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 8), (28, 4), (16, 1), (64, 4), (40, 2), (33, 1)])
@pytest.mark.parametrize("dim", [8, 16, 64, 72, 80, 96, 128])
def test_head_layouts(cuda, heads, kv_heads, dim):
    check(Batch([(1, 200), (3, 77), (1, 1)], heads, kv_heads, dim, 16, seed=dim), cuda)


@pytest.mark.parametrize("page", [8, 16, 24, 48, 64, 128, 136, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages(cuda, page, layout):
    check(Batch([(1, 333), (40, 333), (1, page), (2, page + 1), (130, 290)], 8, 2, 64, page, torch.float16, layout,
                seed=page), cuda)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 5, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700])
def test_whole_prompts(cuda, n, dim, dtype):
    check(Batch([(n, n)], 8, 2, dim, 64, dtype, seed=n), cuda)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 16])
@pytest.mark.parametrize("kv", [129, 1001])
def test_chunks_on_contexts(cuda, group, kv):
    check(Batch([(100, kv), (1, 1), (129, kv + 300), (0, 50), (17, 17)], 2 * group, 2, 128, 16, seed=group), cuda)


@pytest.mark.parametrize("window", [1, 2, 7, 16, 100, 128, 1000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_windows(cuda, window, dtype):
    check(Batch([(1, 500), (150, 500), (300, 300), (1, 3)], 4, 2, 64, 16, dtype, seed=window, window=window), cuda)


def test_window_long_context(cuda):
    check(Batch([(1, 9000), (200, 9001)], 8, 2, 128, 32, seed=4, window=257), cuda)


@pytest.mark.parametrize("n,kv", [(1, 300), (40, 40), (200, 77), (130, 1000)])
def test_every_row_sees_every_key(cuda, n, kv):
    check(Batch([(n, kv), (3, 5)], 8, 4, 128, 16, seed=n, causal=False), cuda)


@pytest.mark.parametrize("lens", [[(1, 0)], [(5, 0), (3, 9)], [(200, 150)], [(40, 3), (1, 0), (1, 40)]])
def test_rows_without_keys(cuda, lens):
    """Causal rows before the first key, and sequences without any key."""
    check(Batch(lens, 8, 2, 128, 16, seed=1), cuda)


def test_nothing_to_do(cuda):
    b = Batch([(0, 40), (0, 0)], 4, 2, 64, 16)
    out, lse = b.run()
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


@pytest.mark.parametrize("lens", [[(1, 20000)], [(1, 3000), (1, 17), (1, 9000), (1, 1)], [(4, 30000)],
                                  [(64, 20000)], [(300, 8200), (1, 8000)]])
def test_long_axis_is_split(cuda, lens):
    check(Batch(lens, 8, 1, 128, 64, seed=3), cuda)


@pytest.mark.parametrize("lens,heads,kv_heads,dim", [
    ([(2500, 2500)], 8, 2, 128),                                   # items dealt whole, one prompt
    ([(64, 64 + b % 50) for b in range(100)], 16, 16, 64),         # items dealt whole, many sequences
    ([(100 + 7 * b, 2000 + 31 * b) for b in range(20)], 8, 8, 64), # blocks dealt out, several items a CTA
    ([(40, 100), (300, 300), (1, 5000), (33, 9000)], 8, 4, 128),   # small and large items, rows beside them
])
def test_ways_of_dealing_out_the_work(cuda, lens, heads, kv_heads, dim):
    check(Batch(lens, heads, kv_heads, dim, 64, seed=21), cuda)


@pytest.mark.parametrize("lens,heads,kv_heads,dim,window", [
    ([(100, 2000)], 32, 8, 128, 0),                                 # sixteen items, pieces of a few blocks
    ([(64, 9000), (0, 50), (700, 1500), (33, 33)], 16, 2, 64, 0),   # long and short items, some not cut, one empty
    ([(300, 9000), (64, 64)], 8, 2, 128, 3000),                     # the pieces begin at the window
    ([(40, 1700 + 300 * b) for b in range(30)], 16, 4, 96, 0),      # pieces close to whole items: even ranges
    ([(260, 20), (300, 5000)], 8, 1, 80, 0),                        # rows without keys in an item that is not cut
])
def test_pieces_of_items(cuda, lens, heads, kv_heads, dim, window):
    check(Batch(lens, heads, kv_heads, dim, 32, window=window, seed=41), cuda)


def test_not_a_number_stays_in_its_row(cuda):
    """A NaN in a query row gives NaN there and nowhere else; an infinite score gives NaN."""
    for value in (float("nan"), float("inf")):
        for lens in ([(1, 100), (1, 90)], [(200, 300), (1, 90)]):
            b = Batch(lens, 4, 2, 64, 16, seed=22)
            want, _ = b.run()
            b.q[0, 1, 5] = value
            got, lse = b.run()
            assert torch.isnan(got[0, 1]).all() and torch.isnan(lse[0, 1])
            got[0, 1] = want[0, 1]
            assert torch.equal(got, want)
            assert cuda.device_status() == 0


def test_not_a_number_among_the_keys(cuda):
    """A key that every row of its sequence sees: NaN there, the other sequence as before."""
    for n in (1, 150):
        b = Batch([(n, 300), (n, 200)], 4, 2, 64, 16, seed=23, causal=False)
        want, _ = b.run()
        page, row = divmod(77, 16)
        b.k_cache[b.table[0, page], 1, row, 3] = float("nan")
        got, _ = b.run()
        assert torch.isnan(got[:n, 2:]).all()
        assert torch.equal(got[:n, :2], want[:n, :2]) and torch.equal(got[n:], want[n:])


def test_calls_that_overlap(cuda):
    """Two streams, a workspace each (the calls allocate their own)."""
    a, b = Batch([(1, 7000), (150, 900)], 8, 2, 128, 16, seed=24), Batch([(1, 9000), (40, 4000)], 8, 2, 128, 16, seed=25)
    want = a.run()[0], b.run()[0]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        got = [x.run(stream=s)[0] for x, s in zip((a, b), streams)]
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_example_layer(cuda):
    """A whole layer in one chunk, in chunks and token by token: within what two roundings
    of the stream to bf16 (2^-8 each, relative) and their way through the experts may differ,
    over the rows that took the same experts (a row whose second and third expert are within
    rounding of each other may take either, and is then another row); those are nearly all."""
    import sys

    from conftest import ROOT

    sys.path.insert(0, str(ROOT / "examples"))
    import decoder_layer as example

    config, lens = example.Config(window=100), [130, 1, 77]
    whole, took = example.run(config, lens, steps=2)
    for chunk in (1, 40):
        parts, took2 = example.run(config, lens, steps=2, chunk=chunk)
        for a, b, i, j in zip(whole, parts, took, took2):
            assert torch.isfinite(a.float()).all()
            same = (i == j).all(1)
            assert int((~same).sum()) <= 0.05 * same.numel()
            a, b = a.float()[same], b.float()[same]
            assert float((a - b).norm() / a.norm()) < 4 * 2.0 ** -8


def test_many_sequences(cuda):
    """More sequences than a CTA has threads."""
    lens = [(1, 1 + (37 * b) % 90) for b in range(700)]
    check(Batch(lens, 4, 2, 64, 16, seed=9), cuda)


@pytest.mark.parametrize("lens,heads,kv_heads,dim,window", [
    ([(1, 1 + (37 * b) % 600) for b in range(700)], 4, 2, 128, 0),                  # more units than warps, cut, past 256 sequences
    ([(b % 4, 2 + b % 9 if b % 50 else 1500) for b in range(300)], 16, 4, 64, 0),   # many tiny units around long ones
    ([(1 + b % 8, 8 + b * 13 % 600) for b in range(90)], 64, 16, 96, 0),            # two row tiles, more units than warps
    ([(1, 1 + (37 * b) % 256) for b in range(200)], 8, 2, 128, 0),                  # a warp a unit
    ([(b % 5, 4 + b * 7 % 250) for b in range(60)], 16, 4, 80, 0),                  # the same, two row tiles, some without rows
    ([(1, b % 3) for b in range(170)], 8, 1, 64, 0),                                # units without keys
    ([(2, 9000 - 40 * b) for b in range(100)], 8, 4, 64, 100),                      # short by their window
    ([(1, 1 + b % 200) for b in range(150)] + [(70, 256)], 8, 2, 128, 0),           # beside a chunk
])
def test_many_units(cuda, lens, heads, kv_heads, dim, window):
    check(Batch(lens, heads, kv_heads, dim, 32, window=window, seed=33), cuda)


def test_sharp_and_growing_scores(cuda):
    """Scores of some hundred, the largest one last: the running maximum moves at every step."""
    b = Batch([(1, 600), (140, 600)], 4, 2, 64, 16, torch.float16, seed=5, q_scale=4.0)
    ramp = torch.linspace(0.05, 3.0, 600, device="cuda")[:, None, None]
    for i in range(2):
        b.k[i] = (b.k[i].abs() * ramp).to(b.dtype)
        for page in range(b.table.shape[1]):
            rows = b.k[i][page * 16:(page + 1) * 16]
            b.k_cache[b.table[i, page], :, :rows.shape[0]] = rows.transpose(0, 1)
    b.q = b.q.abs()
    # scores of some hundreds: the f32 dot product's error grows with them
    b.scale = 0.25
    o, size, lse = b.exact()
    got, got_lse = b.run()
    big = float(lse.max())
    u = HALF_ULP[b.dtype]
    noise = 64 * 2.0 ** -24 * big + 4e-5  # of an exponent, so relative in a weight
    assert ((got.double() - o).abs() <= u * o.abs() + (u + 2 * noise) * size + 600 * 2.0 ** -25 * 6 + 2.0 ** -24).all()
    assert ((got_lse.double() - lse).abs() <= noise + 1e-6 * lse.abs()).all()
    assert cuda.device_status() == 0


def test_equal_scores_give_the_mean(cuda):
    b = Batch([(1, 512), (130, 512)], 4, 2, 128, 64, seed=6)
    b.q.zero_()
    out, lse = b.run()
    hold(b, out, lse)
    assert torch.allclose(lse[0], torch.full_like(lse[0], math.log(512.0)), atol=4e-5)


def test_strided_queries_and_streams(cuda):
    """q is a slice of a wider projection; the call runs on its own stream."""
    b = Batch([(1, 100), (90, 250)], 8, 2, 64, 16, seed=8)
    wide = torch.zeros(91, 12, 64, dtype=b.dtype, device="cuda")
    wide[:, 2:10] = b.q
    want, want_lse = b.run()
    b.q = wide[:, 2:10]
    assert not b.q.is_contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, lse = b.run(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


def test_same_bits_every_time(cuda):
    b = Batch([(1, 5000), (33, 4000), (1, 700), (200, 3000)], 16, 2, 128, 16, seed=2)
    first, lse = b.run()
    for _ in range(4):
        again, lse2 = b.run()
        assert torch.equal(first, again) and torch.equal(lse, lse2)


def test_graph_replay(cuda):
    b = Batch([(1, 900), (70, 400)], 8, 2, 128, 16, seed=12)
    want, _ = b.run()
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.run(workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = b.run(workspace=ws)
    # the lengths are the device's: a replay sees new ones
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    b.kv_len[0] = 450
    b.lens[0] = (1, 450)
    b.k[0], b.v[0] = b.k[0][:450], b.v[0][:450]
    graph.replay()
    torch.cuda.synchronize()
    hold(b, got, b.exact()[2].float())


def test_offsets_past_32_bits(cuda):
    """Pages behind 2^31 elements (and 2^32 bytes) of the cache."""
    page, heads, dim = 64, 8, 128
    first = (1 << 31) // (page * heads * dim) + 5
    b = Batch([(1, 400), (70, 200)], 16, heads, dim, page, seed=13, first_page=first)
    assert int(b.table.max()) * page * heads * dim > 1 << 31
    check(b, cuda)


def test_bad_device_lengths_and_pages_are_reported(cuda):
    b = Batch([(1, 100), (20, 60)], 8, 2, 64, 16, seed=14)
    want, _ = b.run()
    kept = b.table.clone()
    for bad in (-1, 1 << 20):
        b.table[0, 2] = bad
        got, _ = b.run()
        assert cuda.device_status() == 26
        assert torch.equal(got[1:], want[1:])
    b.table.copy_(kept)
    got, _ = b.run(max_kv_len=80)  # sequence 0 has 100 keys
    assert cuda.device_status() == 26
    assert torch.equal(got[1:], want[1:])
    got, _ = b.run(max_q_len=10)  # sequence 1 has 20 rows
    assert cuda.device_status() == 26
    assert torch.equal(got[0], want[0])
    b.q_start[2] = 1000
    b.run()
    assert cuda.device_status() == 26


def test_refusals(cuda):
    from freemoe_b200 import attention

    b = Batch([(1, 40)], 8, 2, 64, 16)

    def refused(code, change=None, **kw):
        c = Batch([(1, 40)], 8, 2, 64, 16)
        if change:
            change(c)
        with pytest.raises(FmError) as e:
            c.run(**kw)
        assert e.value.code == code

    def set_(name, value):
        return lambda c: setattr(c, name, value(c))

    refused(26, set_("q", lambda c: c.q.float()))
    refused(26, set_("q", lambda c: c.q.cpu()))
    refused(26, set_("kv_len", lambda c: c.kv_len.long()))
    refused(8, set_("q", lambda c: c.q[:, :7]))
    refused(8, set_("q", lambda c: c.q[:, :, :60]))
    refused(8, max_kv_len=1000)
    refused(26, window=3, causal=False)
    refused(26, scale=float("nan"))
    with pytest.raises(FmError) as e:  # a long sequence: its work is cut, and the fragments need room
        Batch([(1, 40000)], 8, 2, 64, 16).run(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    assert e.value.code == 26
    refused(8, set_("q", lambda c: torch.zeros(1, 8, 65, dtype=c.dtype, device="cuda")[:, :, :64]))
    refused(26, set_("q", lambda c: torch.zeros(8 * 64 + 1, dtype=c.dtype, device="cuda")[1:].view(1, 8, 64)))
    odd = torch.zeros(4, 2, 12, 64, dtype=b.dtype, device="cuda")
    with pytest.raises(FmError) as e:
        attention.paged_attention(b.q, odd, odd, b.table, b.q_start, b.kv_len, max_q_len=1, max_kv_len=36)
    assert e.value.code == 8
    wide = torch.zeros(4, 2, 16, 136, dtype=b.dtype, device="cuda")
    with pytest.raises(FmError) as e:
        attention.paged_attention(torch.zeros(1, 8, 136, dtype=b.dtype, device="cuda"), wide, wide, b.table, b.q_start,
                                  b.kv_len, max_q_len=1, max_kv_len=40)
    assert e.value.code == 8
