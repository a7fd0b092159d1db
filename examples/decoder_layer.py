"""One MoE decoder layer on the device, for a batch of sequences over a paged cache.

    h  = x + attention(norm(x))          add_rms_norm, gemv_quant (Q, K, V, O in Q8_0),
                                         rope_append, paged_attention
    y  = h + experts(norm(h))            add_rms_norm (adds the attention's output to the
                                         residual stream), router, moe_block / moe_prefill

By its configuration the layer also has norms behind its blocks (norm_add_norm), positions of
several axes, a window with first keys that stay visible (the pages between are freed), and an
output head whose rows are scored (token_logprobs).
A prompt goes through in chunks of any length, then token by token; the calls are the
same.  Run as a program it takes prompts of ragged lengths through a layer in one chunk
and in several, and prints how far the two are apart and what a decoding step costs:

    python examples/decoder_layer.py
"""
from __future__ import annotations

import sys
from dataclasses import dataclass, field
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from freemoe_b200 import TYPE_F32, TYPE_Q4_K, TYPE_Q8_0, attention, hotpath  # noqa: E402


@dataclass
class Config:
    d_model: int = 1024
    heads: int = 16
    kv_heads: int = 4
    head_dim: int = 64
    experts: int = 8
    top_k: int = 2
    ffn: int = 1024
    page_size: int = 16
    rope_base: float = 10000.0
    epsilon: float = 1e-5
    window: int = 0
    sinks: int = 0            # first keys that stay visible behind the window
    sections: tuple = ()      # rotated pairs of each axis, where positions have several
    block_norms: bool = False # norms behind the blocks too, with a gate by channels
    block_scale: float = 1.0  # of a block's normed output
    vocab: int = 0            # rows of an output head


@dataclass
class Layer:
    """Weights of one layer (seeded, in the GGUF block types of the hot path)."""
    config: Config
    weights: dict = field(default_factory=dict)
    experts: list = field(default_factory=list)
    axes: torch.Tensor | None = None  # of the rotated pairs, where positions have several

    @classmethod
    def synthetic(cls, config: Config, seed: int = 0) -> "Layer":
        c, layer = config, cls(config)
        qkv = (c.heads + 2 * c.kv_heads) * c.head_dim
        shapes = {"qkv": (TYPE_Q8_0, qkv, c.d_model), "out": (TYPE_Q8_0, c.d_model, c.heads * c.head_dim),
                  "router": (TYPE_F32, c.experts, c.d_model)}
        for i, (name, (kind, rows, cols)) in enumerate(shapes.items()):
            layer.weights[name] = (kind, hotpath.synth_weights(kind, rows, cols, seed + i, 0.05), rows, cols)
        for e in range(c.experts):
            parts = [hotpath.synth_weights(TYPE_Q4_K, rows, cols, seed + 100 + 3 * e + i, 0.05)
                     for i, (rows, cols) in enumerate(((c.ffn, c.d_model), (c.ffn, c.d_model), (c.d_model, c.ffn)))]
            layer.experts.append(torch.cat(parts))
        g = torch.Generator(device="cuda").manual_seed(seed + 1000)
        for name in ("norm_attention", "norm_experts", "norm_head", "behind_attention", "behind_experts", "gate_attention",
                     "gate_experts"):
            layer.weights[name] = 1 + 0.1 * torch.randn(c.d_model, generator=g, device="cuda")
        layer.axes = attention.rope_axes(c.sections) if c.sections else None
        if c.vocab:
            head = hotpath.synth_weights(TYPE_Q8_0, c.vocab, c.d_model, seed + 50, 0.05)
            layer.weights["head"] = (TYPE_Q8_0, head, c.vocab, c.d_model)
        return layer

    def product(self, name: str, x: torch.Tensor) -> torch.Tensor:
        kind, w, rows, cols = self.weights[name]
        return hotpath.gemv_quant(kind, w, x, rows, cols)


class Cache:
    """The layer's pages, and which of them belong to which sequence."""

    def __init__(self, config: Config, pages: int, sequences: int, max_len: int):
        c = config
        shape = (pages, c.kv_heads, c.page_size, c.head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.page_size = c.page_size
        self.table = torch.full((sequences, -(-max_len // c.page_size)), -1, dtype=torch.int32)
        self.lens = [0] * sequences
        self.free = list(range(pages))[::-1]
        self.window, self.sinks, self.n_axes = c.window, c.sinks, len(c.sections)

    def axes(self, positions: torch.Tensor) -> torch.Tensor:
        """With several axes: every other 16 tokens are an image's, four to a row of it."""
        if not self.n_axes:
            return positions
        image, inside = positions // 16 % 2 == 1, positions % 16
        start = positions - inside
        return torch.stack([torch.where(image, start + d, positions) for d in
                            (0 * inside, inside // 4, inside % 4)[:self.n_axes]]).contiguous()

    def extend(self, new_tokens: list[int]):
        """Room for each sequence's new tokens; what the layer's calls need to know of them."""
        positions, slots, starts = [], [], [0]
        for b, n in enumerate(new_tokens):
            for p in range(self.lens[b], self.lens[b] + n):
                page, row = divmod(p, self.page_size)
                if row == 0:
                    self.table[b, page] = self.free.pop()
                positions.append(p)
                slots.append(int(self.table[b, page]) * self.page_size + row)
            if self.window and self.sinks:
                # what no row from here on sees is freed: behind the first keys, before the windows
                gone = max(0, self.lens[b] - self.window + 1) // self.page_size
                for i in range(-(-self.sinks // self.page_size), gone):
                    if self.table[b, i] >= 0:
                        self.free.append(int(self.table[b, i]))
                        self.table[b, i] = -1
            self.lens[b] += n
            starts.append(starts[-1] + n)
        return {
            "positions": self.axes(torch.tensor(positions, dtype=torch.int32).cuda()),
            "slots": torch.tensor(slots, dtype=torch.int64).cuda(),
            "page_table": self.table.cuda(),
            "q_start": torch.tensor(starts, dtype=torch.int32).cuda(),
            "kv_len": torch.tensor(self.lens, dtype=torch.int32).cuda(),
            "max_q_len": max(new_tokens), "max_kv_len": max(self.lens),
        }


def decoder_layer(layer: Layer, cache: Cache, x: torch.Tensor, step: dict, inv_freq: torch.Tensor,
                  attention_factor: float = 1.0):
    """The residual stream ``x`` [tokens, d_model] bf16 through the layer, and the experts that
    its tokens took; ``step`` from ``Cache.extend``."""
    c, w, tokens = layer.config, layer.weights, x.shape[0]
    normed, _ = attention.add_rms_norm(x, w["norm_attention"], epsilon=c.epsilon)
    qkv = layer.product("qkv", normed).view(tokens, c.heads + 2 * c.kv_heads, c.head_dim)
    q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), dim=1)
    q = attention.rope_append(q, k, v, step["positions"], inv_freq, cache.k, cache.v, step["slots"],
                              attention_factor=attention_factor, axes=layer.axes)
    o = attention.paged_attention(q, cache.k, cache.v, step["page_table"], step["q_start"], step["kv_len"],
                                  max_q_len=step["max_q_len"], max_kv_len=step["max_kv_len"], window=c.window,
                                  sinks=c.sinks)
    o = layer.product("out", o.view(tokens, -1))
    if c.block_norms:
        normed, h = attention.norm_add_norm(o, w["behind_attention"], x, w["norm_experts"], gate=w["gate_attention"],
                                            scale=c.block_scale, epsilon=c.epsilon, out_dtype=torch.bfloat16)
    else:
        normed, h = attention.add_rms_norm(o, w["norm_experts"], residual=x, epsilon=c.epsilon, out_dtype=torch.bfloat16)
    experts = hotpath.moe_block if tokens <= 64 else hotpath.moe_prefill
    y, ids, _ = experts(normed, layer.product("router", normed), layer.experts, top_k=c.top_k, ffn=c.ffn,
                        gate_type=TYPE_Q4_K, return_routing=True)
    if c.block_norms:
        _, out = attention.norm_add_norm(y, w["behind_experts"], h, None, gate=w["gate_experts"], scale=c.block_scale,
                                         epsilon=c.epsilon)
        return out, ids
    return (h.float() + y).to(torch.bfloat16), ids


def score(layer: Layer, x: torch.Tensor, following: torch.Tensor, top: int = 5):
    """The log probabilities of the tokens that follow the rows of the stream ``x``, the entropy, and the most
    probable tokens."""
    normed, _ = attention.add_rms_norm(x, layer.weights["norm_head"], epsilon=layer.config.epsilon)
    return hotpath.token_logprobs(layer.product("head", normed), following, top=top)


def run(config: Config, lens: list[int], steps: int = 4, chunk: int | None = None, seed: int = 0):
    """Prompts of ragged lengths, in one chunk or in chunks of ``chunk`` tokens, then
    ``steps`` single tokens each; the stream after the layer and the experts taken,
    sequence by sequence."""
    hotpath.init(torch.cuda.current_device())
    layer = Layer.synthetic(config, seed)
    total = [n + steps for n in lens]
    pages = sum(-(-n // config.page_size) for n in total)
    cache = Cache(config, pages, len(lens), max(total))
    g = torch.Generator(device="cuda").manual_seed(seed)
    streams = [torch.randn(n, config.d_model, generator=g, device="cuda").to(torch.bfloat16) for n in total]
    inv_freq, factor = attention.rope_frequencies(config.head_dim, config.rope_base)
    outs, taken = [[] for _ in lens], [[] for _ in lens]
    done = [0] * len(lens)
    while any(d < t for d, t in zip(done, total)):
        new = [min(chunk or n, n - d) if d < n else min(1, t - d) for n, d, t in zip(lens, done, total)]
        x = torch.cat([s[d:d + n] for s, d, n in zip(streams, done, new)])
        y, ids = decoder_layer(layer, cache, x, cache.extend(new), inv_freq, factor)
        at = 0
        for b, n in enumerate(new):
            outs[b].append(y[at:at + n])
            taken[b].append(ids[at:at + n])
            at += n
            done[b] += n
    if hotpath.device_status():
        raise RuntimeError("the device status is set")
    return [torch.cat(o) for o in outs], [torch.cat(t) for t in taken]


def main() -> None:
    config, lens = Config(), [300, 17, 128, 1]
    (whole, took), (parts, took2) = run(config, lens), run(config, lens, chunk=50)
    same = torch.cat([(a == b).all(1) for a, b in zip(took, took2)])
    a, b = torch.cat(whole).float(), torch.cat(parts).float()
    off = float((a - b)[same].norm() / a[same].norm())
    print(f"prompts of {lens} tokens and 4 steps: whole against chunks of 50, relative difference {off:.1e} over "
          f"{int(same.sum())} of {same.numel()} rows (the others took another expert: a tie within rounding)")
    layer = Layer.synthetic(config)
    cache = Cache(config, 64 * 64, 64, 1024)
    cache.extend([1000] * 64)
    step = cache.extend([1] * 64)
    inv_freq, _ = attention.rope_frequencies(config.head_dim, config.rope_base)
    x = torch.randn(64, config.d_model, device="cuda").to(torch.bfloat16)
    for _ in range(3):
        decoder_layer(layer, cache, x, step, inv_freq)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(20):
        decoder_layer(layer, cache, x, step, inv_freq)
    end.record()
    torch.cuda.synchronize()
    print(f"a decoding step of 64 sequences behind 1000 keys: {begin.elapsed_time(end) / 20 * 1e3:.0f} us")
    config = Config(window=100, sinks=8, sections=(8, 12, 12), block_norms=True, block_scale=0.5, vocab=32000)
    (whole, _), layer = run(config, lens), Layer.synthetic(config)
    following = torch.zeros(whole[0].shape[0], dtype=torch.int32, device="cuda")
    logprobs, entropy, _, _ = score(layer, whole[0], following)
    print(f"with norms behind the blocks, three axes and a window with first keys: mean log probability of a fixed token "
          f"{float(logprobs.mean()):.2f}, mean entropy {float(entropy.mean()):.2f}")


if __name__ == "__main__":
    main()
