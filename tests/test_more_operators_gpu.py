"""The operators around the attention side as they are used together: a layer with norms
behind its blocks, positions of several axes, a window with first keys that stay visible over a
cache whose pages between are freed, and an output head whose rows are scored.

Tolerances, derived before the first run.  A layer in one chunk, in chunks and token by token
differs by the roundings of the softmax weights (2^-8 of bf16, relative, in another order of
sums), of the stream after the attention and after the experts, and of the normed rows between:
four of at most 2^-8 each.  As for the layer without these operators that is held over the rows
that took the same experts.
"""
from __future__ import annotations

import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(ROOT / "examples"))
BF16, F32 = torch.bfloat16, torch.float32


def layer_config(**change):
    import decoder_layer as example

    return example.Config(**{**dict(window=60, sinks=5, sections=(8, 12, 12), block_norms=True, block_scale=0.5), **change})


@pytest.mark.parametrize("change", [{}, {"sinks": 40, "window": 33, "page_size": 8}, {"block_scale": -0.3, "sections": (20, 12)}])
def test_a_layer_in_chunks(cuda, change):
    import decoder_layer as example

    config, lens = layer_config(**change), [230, 1, 77]
    whole, took = example.run(config, lens, steps=3)
    for chunk in (1, 40):
        parts, took2 = example.run(config, lens, steps=3, chunk=chunk)
        for a, b, i, j in zip(whole, parts, took, took2):
            assert torch.isfinite(a.float()).all()
            same = (i == j).all(1)
            assert int((~same).sum()) <= 0.05 * same.numel()
            a, b = a.float()[same], b.float()[same]
            assert float((a - b).norm() / a.norm()) < 4 * 2.0 ** -8


def test_the_parts_matter(cuda):
    """Each of the layer's options changes its result."""
    import decoder_layer as example

    base = example.run(layer_config(), [150], steps=1)[0][0].float()
    for change in ({"sinks": 0}, {"sections": ()}, {"block_norms": False}, {"block_scale": 0.6}, {"window": 50}):
        other = example.run(layer_config(**change), [150], steps=1)[0][0].float()
        assert float((base - other).norm() / base.norm()) > 1e-3, change


def test_freed_pages_are_used_again(cuda):
    """A stream far longer than its cache: its pages are those of the first keys and of the window."""
    import decoder_layer as example

    config = layer_config(window=32, sinks=6, page_size=8)
    layer = example.Layer.synthetic(config)
    inv_freq, _ = example.attention.rope_frequencies(config.head_dim)
    x = torch.randn(400, config.d_model, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(BF16)
    outs = []
    for pages, chunk in ((60, 400), (9, 16), (7, 1)):
        cache = example.Cache(config, pages, 1, 400)
        rows, took = [], []
        for at in range(0, 400, chunk):
            y, ids = example.decoder_layer(layer, cache, x[at:at + chunk], cache.extend([min(chunk, 400 - at)]), inv_freq)
            rows.append(y)
            took.append(ids)
        outs.append((torch.cat(rows).float(), torch.cat(took)))
    assert cuda.device_status() == 0
    (a, i), rest = outs[0], outs[1:]
    for b, j in rest:
        same = (i == j).all(1)
        assert int((~same).sum()) <= 0.05 * same.numel()
        assert float((a - b)[same].norm() / a[same].norm()) < 4 * 2.0 ** -8


def test_scores_of_the_stream(cuda):
    """Log probabilities behind norm and head: those of the head's logits in 64 bits, to 1e-5 (the sums' f32 errors
    of logits below 16, see test_logprobs_gpu.py)."""
    import decoder_layer as example

    config = layer_config(vocab=5003)
    layer = example.Layer.synthetic(config)
    (x,), _ = example.run(config, [50], steps=0)
    following = torch.arange(50, dtype=torch.int32, device="cuda") * 100
    following[-1] = -1
    logprobs, entropy, best, ids = example.score(layer, x, following, top=7)
    normed, _ = example.attention.add_rms_norm(x, layer.weights["norm_head"])
    logits = layer.product("head", normed)
    want = torch.log_softmax(logits.double(), -1)
    assert logits.abs().max() < 16
    assert (logprobs[:-1] - want[:-1].gather(1, following[:-1, None].long())[:, 0]).abs().max() < 1e-5 and logprobs[-1] == 0
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :7]
    assert torch.equal(ids.long(), order) and (best - want.gather(1, order)).abs().max() < 1e-5
    assert (entropy - torch.special.entr(want.exp()).sum(-1)).abs().max() < 1e-4


def test_two_streams_at_once(cuda):
    """All four on two streams, with buffers of their own: the results of one after the other, bit for bit."""
    from freemoe_b200 import attention, hotpath

    inv_freq, _ = attention.rope_frequencies(64)
    axes = attention.rope_axes((8, 12, 12), "turn")

    def chain(seed, n):
        g = torch.Generator("cuda").manual_seed(seed)
        q, k, v = (torch.randn(n, h, 64, generator=g, device="cuda").to(BF16) for h in (8, 2, 2))
        x, r, w = (torch.randn(n, 512, generator=g, device="cuda"), torch.randn(n, 512, generator=g, device="cuda").to(BF16),
                   torch.randn(512, generator=g, device="cuda"))
        positions = torch.randint(0, 5000, (3, n), generator=g, device="cuda", dtype=torch.int32)
        pages = -(-n // 16)
        caches = [torch.zeros(pages, 2, 16, 64, dtype=BF16, device="cuda") for _ in range(2)]
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        q_start, kv_len = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, n], [n]))
        logits = torch.randn(n, 20000, generator=g, device="cuda")
        tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
        slots = torch.arange(n, device="cuda")

        def run(stream):
            rotated = attention.rope_append(q, k, v, positions, inv_freq, *caches, slots, axes=axes, stream=stream)
            o = attention.paged_attention(rotated, *caches, table, q_start, kv_len, max_q_len=n, max_kv_len=n, window=50,
                                          sinks=9, stream=stream)
            y, h = attention.norm_add_norm(x, w, r, w, gate=r, out_dtype=BF16, stream=stream)
            return (o, y, h, *hotpath.token_logprobs(logits, tokens, top=9, stream=stream))

        return run

    chains = [chain(1, 300), chain(2, 17)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    want = [c(torch.cuda.current_stream()) for c in chains]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [None, None]
        for i in (0, 1):
            got[i] = chains[i](streams[i])
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert cuda.device_status() == 0


def test_the_axes_are_worked_out_once(cuda, monkeypatch):
    """A layer has the axes of its pairs at hand: its calls make no copy from the host for them."""
    import decoder_layer as example

    config = layer_config()
    layer, cache = example.Layer.synthetic(config), example.Cache(config, 8, 1, 100)
    inv_freq, _ = example.attention.rope_frequencies(config.head_dim)
    x = torch.randn(3, config.d_model, device="cuda").to(BF16)
    monkeypatch.setattr(example.attention, "rope_axes", lambda *a, **k: pytest.fail("worked out in a call"))
    example.decoder_layer(layer, cache, x, cache.extend([3]), inv_freq)
