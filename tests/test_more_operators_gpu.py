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


def rms(x, w, epsilon):
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + epsilon) * w.double()


def plain_layer(layer, x, inv_freq, swap={}):
    """One sequence from its begin through the layer in plain torch, in 64 bits but for the products and the
    experts, which are the layer's own, and with the roundings that it makes."""
    import decoder_layer as example

    from freemoe_b200 import TYPE_Q4_K, hotpath

    c, n = layer.config, x.shape[0]
    w = {name: layer.weights[swap.get(name, name)] for name in layer.weights}
    qkv = layer.product("qkv", rms(x, w["norm_attention"], c.epsilon).to(BF16)).view(n, c.heads + 2 * c.kv_heads, c.head_dim)
    q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), dim=1)
    positions = example.Cache(c, 1, 1, n).axes(torch.arange(n, dtype=torch.int32, device="cuda"))
    positions = positions if c.sections else positions[None]
    axis = sum(([a] * pairs for a, pairs in enumerate(c.sections)), []) or [0] * (c.head_dim // 2)
    angle = torch.stack([positions[a].double() * f for a, f in zip(axis, inv_freq.double())], -1)[:, None]

    def turn(t):
        a, b = t.double().split(c.head_dim // 2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1).to(BF16).double()

    group = c.heads // c.kv_heads
    q, k, v = turn(q), turn(k).repeat_interleave(group, 1), v.to(BF16).double().repeat_interleave(group, 1)
    at = torch.arange(n, device="cuda")
    seen = at <= at[:, None]
    if c.window:
        seen &= (at > at[:, None] - c.window) | (at < c.sinks)
    s = (torch.einsum("qhd,khd->hqk", q, k) / c.head_dim ** 0.5).masked_fill(~seen, float("-inf"))
    o = layer.product("out", torch.einsum("hqk,khd->qhd", s.softmax(-1), v).reshape(n, -1).to(BF16)).double()
    if c.block_norms:
        h = x.double() + c.block_scale * w["gate_attention"].double() * rms(o, w["behind_attention"], c.epsilon)
    else:
        h = x.double() + o
    normed, h = rms(h, w["norm_experts"], c.epsilon).to(BF16), h.to(BF16).double()
    experts = hotpath.moe_block if n <= 64 else hotpath.moe_prefill
    y, ids, _ = experts(normed, layer.product("router", normed), layer.experts, top_k=c.top_k, ffn=c.ffn,
                        gate_type=TYPE_Q4_K, return_routing=True)
    if c.block_norms:
        return h + c.block_scale * w["gate_experts"].double() * rms(y, w["behind_experts"], c.epsilon), ids
    return h + y.double(), ids


@pytest.mark.parametrize("change", [{}, {"block_norms": False}, {"sections": (), "window": 0, "sinks": 0},
                                    {"block_scale": -0.3, "sections": (20, 12), "page_size": 8}])
@pytest.mark.parametrize("n", [5, 200])
def test_a_layer_against_plain_torch(cuda, change, n):
    """Each weight and gate where it belongs: the layer's roundings are those of the header, and each of them is
    made in the plain form too, so that the two differ by the softmax weights' and by ties that fall otherwise."""
    import decoder_layer as example

    config = layer_config(**change)
    layer, cache = example.Layer.synthetic(config, 7), example.Cache(config, 40, 1, 300)
    inv_freq, _ = example.attention.rope_frequencies(config.head_dim)
    x = torch.randn(n, config.d_model, generator=torch.Generator("cuda").manual_seed(9), device="cuda").to(BF16)
    got, took = example.decoder_layer(layer, cache, x, cache.extend([n]), inv_freq)
    assert cuda.device_status() == 0

    def off(**swap):
        want, ids = plain_layer(layer, x, inv_freq, swap)
        same = (took == ids).all(1)
        return float((got.double() - want)[same].norm() / want[same].norm()), float(same.float().mean())

    distance, same = off()
    assert distance < 4 * 2.0 ** -8 and same >= 0.95
    names = ["norm_attention", "norm_experts"]
    if config.block_norms:
        names += ["behind_attention", "behind_experts", "gate_attention", "gate_experts"]
    for name in names:  # another one in its place is seen
        assert off(**{name: "norm_head"})[0] > 2 * distance, name
