"""Log probabilities of tokens, entropy and the most probable tokens against a plain
implementation in 64 bits.

Tolerances, derived before the first run.  E = 2^-24.  A term 2^t, t = (x - ref) scale log2 e
in f32, has a relative error of 2^-22 (the hardware exponential) + ln 2 * 3 E |t|; with
W = mean of |t| under the distribution (ref is at most 8 below the largest value: 8 more) and
n terms a thread in turn, then a tree, the sum has a relative error of
    r = 2^-22 + 2.1 E W + (n + 15) E,   n <= V / 512 + 80,
which is the error of L.  A log probability is then off by r + 2 E |log p|.  The terms t 2^t
carry the same errors, 4 E more and, in t itself, 3 E |t|, so that the entropy is off by
    r + ln 2 (2 r W + 6 E W2) + 2 E H,   W2 = mean of t^2 (64 + 16 W more).
Ids are whole numbers: they are equal.
"""
from __future__ import annotations

import math

import pytest
import torch

from freemoe_b200._lib import FmError

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def logits_of(rows, vocab, dtype=F32, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * spread
    x += 10 * torch.rand(rows, 1, generator=g, device="cuda") * (torch.rand(rows, vocab, generator=g, device="cuda") > 0.999)
    return x.to(dtype)


def hold(logits, tokens, top, scale=1.0, got=None):
    from freemoe_b200 import hotpath

    chosen, entropy, best, ids = hotpath.token_logprobs(logits, tokens, top=top, scale=scale) if got is None else got
    rows, vocab = logits.shape
    assert chosen.shape == entropy.shape == (rows,) and best.shape == ids.shape == (rows, top)
    assert chosen.dtype == entropy.dtype == best.dtype == F32 and ids.dtype == torch.int32
    for at in range(0, rows, 512):
        x = logits[at:at + 512]
        z = x.double() * scale
        log_p = torch.log_softmax(z, -1)
        p = log_p.exp()
        t = torch.where(p > 0, (z - z.amax(-1, keepdim=True)) / math.log(2), 0.0)
        w, w2 = (p * t.abs()).sum(-1) + 8, (p * t * t).sum(-1)
        w2 = w2 + 64 + 16 * w
        r = 2.0 ** -22 + 2.1 * E * w + (vocab / 512 + 95) * E
        h = torch.special.entr(p).sum(-1)
        off = (entropy[at:at + 512].double() - h).abs()
        assert (off <= r + math.log(2) * (2 * r * w + 6 * E * w2) + 2 * E * h).all()
        assert (entropy[at:at + 512] >= 0).all()
        order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(ids[at:at + 512].long(), order)
        tok = tokens[at:at + 512].long()
        want = torch.where(tok < 0, 0.0, log_p.gather(1, tok.clamp(min=0)[:, None])[:, 0])
        for have, exact in ((chosen[at:at + 512, None], want[:, None]), (best[at:at + 512], log_p.gather(1, order))):
            gone = exact == -math.inf
            assert torch.equal(have == -math.inf, gone)
            off = torch.where(gone, 0.0, have.double() - exact).abs()
            assert (off <= r[:, None] + 2 * E * torch.where(gone, 0.0, exact).abs()).all()


def tokens_of(rows, vocab, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 31, 32, 33, 100, 255, 257, 1000, 4096, 16384, 32003, 50001, 151936,
                                   (1 << 20) + 5])
@pytest.mark.parametrize("rows", [1, 2, 17, 40, 75, 150, 600])
def test_sizes(cuda, vocab, rows):
    if rows * vocab > 1 << 26:
        rows = (1 << 26) // vocab
    for dtype, top in ((F32, 20), (BF16, 5), (F16, 32)):
        hold(logits_of(rows, vocab, dtype, seed=vocab), tokens_of(rows, vocab), min(top, vocab))
    assert cuda.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("top", [0, 1, 2, 31, 32])
@pytest.mark.parametrize("scale", [1.0, 0.37, 8.0, 1e-4])
def test_tops_and_scales(cuda, dtype, top, scale):
    for rows, vocab in ((1, 40000), (200, 3001)):
        hold(logits_of(rows, vocab, dtype, seed=top), tokens_of(rows, vocab), top, scale)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("off", [0, 1, 2, 3, 5, 8])
def test_rows_of_a_wider_tensor(cuda, dtype, off):
    """Rows that begin and end anywhere; what lies around them is not read into the sums."""
    for rows, vocab in ((3, 20001), (160, 997), (2, 5), (2, 1)):
        wide = torch.full((rows, vocab + 21), float("nan"), dtype=dtype, device="cuda")
        x = wide[:, off:off + vocab]
        x.copy_(logits_of(rows, vocab, dtype, seed=off))
        hold(x, tokens_of(rows, vocab), min(9, vocab))


@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_orders(cuda, rows, dtype):
    """Ties go to the lower id; values that grow, fall, or lie one thread's after another's."""
    vocab = 30000
    i = torch.arange(vocab, device="cuda")
    for row in (torch.zeros(vocab, device="cuda"), i % 2, -(i % 3), i * (8.0 / vocab), -i * (8.0 / vocab), (i // 8 % 512) * -0.1,
                (i // 8 % 512) * -1.0 + (i // 4096) * 0.125, (i // 4 % 512) * -1.0 + (i // 2048) * 0.0625,
                (i // 4 % 4096) * -1.0, (i // 8 % 2048) * 0.5):
        x = row.to(dtype).float().to(dtype).expand(rows, vocab).contiguous()
        hold(x, tokens_of(rows, vocab), 32)
    zeros = torch.zeros(rows, 1000, dtype=dtype, device="cuda")
    zeros[:, ::2] = -0.0  # equal to 0
    hold(zeros, tokens_of(rows, 1000), 20)


@pytest.mark.parametrize("rows", [1, 33, 400])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_ruled_out_tokens(cuda, rows, dtype):
    vocab = 9000
    x = logits_of(rows, vocab, dtype)
    x[:, 3000:] = -math.inf
    hold(x, tokens_of(rows, vocab), 32)
    x[:, 7:] = -math.inf  # fewer left than are asked for
    hold(x, tokens_of(rows, vocab), 32)
    x = logits_of(rows, vocab, dtype)
    x[:, 100:8000] = torch.finfo(dtype).min  # the type's lowest value in place of -inf
    hold(x, tokens_of(rows, vocab), 20)
    x[:] = torch.finfo(dtype).min
    hold(x, tokens_of(rows, vocab), 20)


@pytest.mark.parametrize("rows,vocab", [(5, 40), (5, 70000), (400, 5000)])
def test_rows_without_probabilities(cuda, rows, vocab):
    from freemoe_b200 import hotpath

    x, tok = logits_of(rows, vocab), tokens_of(rows, vocab)
    x[0] = -math.inf
    x[1, 3] = float("nan")
    x[2, 5] = math.inf
    x[3] = float("nan")
    chosen, entropy, best, ids = hotpath.token_logprobs(x, tok, top=4)
    assert chosen[0] == -math.inf and entropy[0] == 0 and (best[0] == -math.inf).all()
    assert ids[0].tolist() == [0, 1, 2, 3] and ids[3].tolist() == [0, 1, 2, 3]
    assert torch.isnan(chosen[1:4]).all() and torch.isnan(entropy[1:4]).all() and torch.isnan(best[1:4]).all()
    assert ids[2, 0] == 5 and 3 not in ids[1].tolist()
    hold(x[4:], tok[4:], 4, got=[v[4:] for v in (chosen, entropy, best, ids)])
    assert cuda.device_status() == 0


def test_no_token_and_a_token_past_the_vocabulary(cuda):
    from freemoe_b200 import hotpath

    x = logits_of(3, 100)
    tok = torch.tensor([-1, 99, -2147483648], dtype=torch.int32, device="cuda")
    hold(x, tok, 3)
    assert cuda.device_status() == 0
    tok[1] = 100
    chosen, entropy, _, _ = hotpath.token_logprobs(x, tok)
    assert cuda.device_status() == 26
    assert torch.isnan(chosen[1]) and chosen[0] == 0 and torch.isfinite(entropy).all()


def test_one_sure_token(cuda):
    """One token has all of the probability: entropy 0, not below."""
    from freemoe_b200 import hotpath

    x = torch.full((2, 5000), -1000.0, device="cuda")
    x[:, 77] = 1000.0
    chosen, entropy, best, ids = hotpath.token_logprobs(x, torch.tensor([77, 5], dtype=torch.int32, device="cuda"), top=2)
    assert chosen.tolist() == [0.0, -2000.0] and entropy.tolist() == [0.0, 0.0]
    assert ids.tolist() == [[77, 0]] * 2 and best.tolist() == [[0.0, -2000.0]] * 2


def test_offsets_past_32_bits(cuda):
    from freemoe_b200 import hotpath

    rows, vocab = 17000, 131072
    x = torch.empty(rows, vocab, dtype=BF16, device="cuda")
    x[:] = logits_of(1, vocab, BF16)
    x[-40:] = logits_of(40, vocab, BF16, seed=1)
    tok = tokens_of(rows, vocab)
    got = hotpath.token_logprobs(x, tok, top=3)
    hold(x[-40:], tok[-40:], 3, got=[v[-40:] for v in got])
    assert (got[3][:-40] == got[3][0]).all()


def test_a_very_large_vocabulary(cuda):
    for dtype in (BF16, F32):
        x = logits_of(2, (1 << 24) + 37, dtype)
        hold(x, tokens_of(2, x.shape[1]), 32)


def test_the_same_bits_each_time_on_any_stream_and_replayed(cuda):
    from freemoe_b200 import hotpath

    for rows, vocab in ((1, 100000), (12, 30001), (500, 8000)):
        x, tok = logits_of(rows, vocab, BF16), tokens_of(rows, vocab)
        want = hotpath.token_logprobs(x, tok, top=10, scale=0.9)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = hotpath.token_logprobs(x, tok, top=10, scale=0.9, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = hotpath.token_logprobs(x, tok, top=10, scale=0.9)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        x.copy_(logits_of(rows, vocab, BF16, seed=3))
        graph.replay()
        want = hotpath.token_logprobs(x, tok, top=10, scale=0.9)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_after_the_output_head(cuda):
    """The head's product and the probabilities of what it gives, one after the other."""
    from freemoe_b200 import TYPE_Q8_0, hotpath

    w = hotpath.synth_weights(TYPE_Q8_0, 5000, 256, seed=3, std=0.2)
    for tokens in (1, 9):
        g = torch.Generator(device="cuda").manual_seed(tokens)
        x = torch.randn(tokens, 256, generator=g, device="cuda").bfloat16()
        logits = hotpath.gemv_quant(TYPE_Q8_0, w, x, 5000, 256)
        hold(logits, tokens_of(tokens, 5000), 5)


def test_refusals(cuda):
    from freemoe_b200 import hotpath

    x, tok = logits_of(3, 50), tokens_of(3, 50)

    def refused(code, *args, **how):
        with pytest.raises(FmError) as e:
            hotpath.token_logprobs(*args, **how)
        assert e.value.code == code

    refused(26, x.double(), tok)
    refused(26, x, tok, top=33)
    refused(26, x, tok, top=-1)
    refused(26, x[:, :10].contiguous(), tok, top=11)
    refused(26, x, tok, scale=0.0)
    refused(26, x, tok, scale=-1.0)
    refused(26, x, tok, scale=float("nan"))
    refused(26, x, tok, scale=1e31)
    refused(8, x, tok.long())
    refused(8, x, tok[:2])
    refused(8, x[0], tok)
    refused(8, x.t(), tokens_of(50, 3))
    refused(8, x[:, :0], tok)
    refused(8, x[:1].expand(3, 50), tok)
    refused(26, x.cpu(), tok)
    refused(26, x, tok.cpu())
    out = hotpath.token_logprobs(x[:0], tok[:0], top=2)
    assert [v.shape for v in out] == [(0,), (0,), (0, 2), (0, 2)]
