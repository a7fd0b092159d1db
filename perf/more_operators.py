"""More workloads of a decoder layer and of what follows its last one: the norms around a block with
its gate and residual scale, rotary positions of several axes (time, height, width) with the write into a
paged K/V cache, attention over a sliding window and a few first tokens that stay visible, and log
probabilities of given tokens with entropy and the most probable alternatives.

``listed()`` names the workloads, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes the
inputs of one from a seed, ``run`` takes one pass (the plain torch form, or with ``own`` the
framework's kernels), ``exact`` is the definition in 64 bits and ``work`` the bytes and operations
that a pass cannot do without.
"""
import math

import torch

own = False

FP8_GROUP = 128
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # a layer's second norm pair while one sequence decodes: latency alone
        _norms("norms one token", 1, 4096, "f32", "bf16", "bf16", gate="channel"),
        # the same for a prompt batch
        _norms("norms prompt", 8192, 4096, "bf16", "bf16", "bf16", gate="channel"),
        # gated token by token, odd width, to 8-bit rows for the next product or exchange
        _norms("norms odd width to 8 bits", 777, 2050, "f32", "f16", "e4m3", gate="token", residual_scale=0.8),
        # 16 decoding sequences behind images, q/k/v as the quantised products leave them (f32)
        _axes("axes 16 decoding", 16, 32, 8, 128, (16, 24, 24), "blocks", "f32", "bf16", page=16, far=True),
        # a prompt of text and images, three axes in blocks of pairs
        _axes("axes prompt", 8192, 32, 8, 128, (16, 24, 24), "blocks", "bf16", "bf16", page=64),
        # one sequence decodes far behind its window: latency
        _attn("sinks decode one", "bf16", 1, 1, 20011, 32, 8, 128, 16, window=1024, sinks=4),
        # 64 sequences of ragged lengths decode together: the serving batch, most pages long freed
        _attn("sinks decode 64 ragged", "bf16", 64, 1, 32768, 32, 8, 128, 16, window=4096, sinks=64, ragged=True),
        # a whole prompt at once
        _attn("sinks prompt 8192", "bf16", 1, 8192, 8192, 32, 8, 128, 64, window=2048, sinks=16),
        # a chunk beside decoding sequences, smaller heads, token-major pages, first tokens past a tile
        _attn("sinks chunk and decodes", "f16", 8, 510, 12001, 28, 4, 64, 48, window=1000, sinks=130, ragged=True,
              mixed=True, layout="nhd"),
        # the next token of one sequence, a large vocabulary, f32 as the output head leaves it: latency
        _probs("probabilities one token", 1, 151936, "f32", 20),
        # a prompt's tokens scored
        _probs("probabilities prompt", 4096, 128256, "bf16", 5, scale=0.7),
        # ragged batch of odd width, half of the vocabulary ruled out by a grammar
        _probs("probabilities masked", 333, 32003, "f16", 32, masked=True),
    ]


def _norms(name, tokens, dim, x, residual, out, gate="none", residual_scale=1.0, scale=0.5):
    return {"name": name, "op": "norms", "tokens": tokens, "dim": dim, "x": x, "residual": residual, "out": out,
            "gate": gate, "scale": scale, "residual_scale": residual_scale}


def _axes(name, tokens, heads, kv_heads, dim, sections, order, x, out, page, far=False, interleaved=False):
    return {"name": name, "op": "axes", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "sections": "/".join(map(str, sections)), "order": order, "x": x, "out": out, "page": page, "far": far,
            "interleaved": interleaved}


def _attn(name, dtype, seqs, q_len, kv_len, heads, kv_heads, dim, page, window, sinks, ragged=False, mixed=False,
          layout="hnd"):
    return {"name": name, "op": "attention", "x": dtype, "seqs": seqs, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "sinks": sinks, "ragged": ragged,
            "mixed": mixed, "layout": layout}


def _probs(name, tokens, vocab, dtype, top, scale=1.0, masked=False):
    return {"name": name, "op": "probs", "tokens": tokens, "vocab": vocab, "x": dtype, "top": top, "scale": scale,
            "masked": masked}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norms", "axes", "attention", "attention", "probs"])
    if op == "norms":
        case = _norms("", _log(rng, 1, 8192), _log(rng, 64, 8192), rng.choice(["f32", "bf16", "f16"]),
                      rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["bf16", "f16", "f32", "e4m3"]),
                      gate=rng.choice(["none", "channel", "token", "full"]),
                      residual_scale=rng.choice([1.0, 1.0, round(rng.uniform(0.2, 1.5), 3)]))
        while case["tokens"] * case["dim"] > 1 << 24 and "f32" in (case["x"], case["residual"]):
            case["tokens"] //= 2
    elif op == "axes":
        heads, kv_heads = rng.choice([(32, 8), (16, 16), (28, 4), (64, 4), (16, 1), (8, 2)])
        dim = rng.choice([64, 80, 96, 128])
        pairs = rng.choice([dim // 2, dim // 4, rng.randrange(4, dim // 2)])
        cuts = sorted(rng.randrange(1, pairs) for _ in range(rng.choice([1, 2, 2, 3])))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        case = _axes("", _log(rng, 1, 8192), heads, kv_heads, dim, sections, rng.choice(["blocks", "turn"]),
                     rng.choice(["f32", "bf16", "f16"]), rng.choice(["bf16", "f16"]),
                     rng.choice([8, 16, 32, 48, 64, 128]), far=rng.random() < 0.5, interleaved=rng.random() < 0.3)
        while case["tokens"] * heads * dim > 1 << 25:
            case["tokens"] //= 2
    elif op == "probs":
        while True:
            case = _probs("", _log(rng, 1, 4096), _log(rng, 256, 262144), rng.choice(["f32", "bf16", "f16"]),
                          rng.choice([0, 1, 5, 20, rng.randrange(33)]), scale=rng.choice([1.0, round(rng.uniform(0.3, 2.0), 3)]),
                          masked=rng.random() < 0.3)
            if case["tokens"] * case["vocab"] * _SIZE[case["x"]] <= 1 << 30:
                break
    else:
        heads, kv_heads = rng.choice([(32, 8), (16, 16), (28, 4), (64, 4), (16, 1), (8, 2)])
        while True:
            kind = rng.choice(["decode", "prompt", "chunk"])
            seqs = _log(rng, 1, {"decode": 128, "prompt": 8, "chunk": 16}[kind])
            q_len = 1 if kind == "decode" else _log(rng, 1, 4096 if kind == "prompt" else 1024)
            kv_len = q_len if kind == "prompt" else _log(rng, q_len, 131072 if kind == "decode" else 16384)
            dim, window, sinks = rng.choice([64, 80, 96, 128]), _log(rng, 1, 8192), _log(rng, 1, 256)
            width = min(kv_len, q_len + window + sinks)
            # the plain form's scores and keys stay within a few GB, the work within the listed prompt's
            if seqs * heads * q_len * width <= 1 << 29 and seqs * width * kv_heads * dim <= 1 << 28:
                break
        case = _attn("", rng.choice(["bf16", "f16"]), seqs, q_len, kv_len, heads, kv_heads, dim,
                     rng.choice([8, 16, 32, 48, 64, 128, 256]), window, sinks, ragged=rng.random() < 0.6,
                     mixed=kind == "chunk" and rng.random() < 0.4, layout=rng.choice(["hnd", "nhd"]))
    del case["name"]
    return case


def _lens(case):
    """The case's new tokens and cache lengths, sequence by sequence."""
    n = case["seqs"]
    q, kv = [], []
    for b in range(n):
        part = ((5 * b + 3) % n + 1) / n if case["ragged"] else 1.0
        ql = 1 if case["mixed"] and b != n // 2 else case["q_len"]
        if case["ragged"] and ql > 1:
            ql = max(1, int(ql * (0.5 + 0.5 * part)))
        q.append(ql)
        kv.append(max(ql, int(case["kv_len"] * part)))
    return q, kv


def _visible(q_len, kv_len, window, sinks):
    """How many keys the rows of a chunk see in all, and how many keys any of them sees."""
    total = 0
    for position in range(kv_len - q_len, kv_len):
        first = max(0, position - window + 1)
        total += position + 1 - first + min(sinks, first)
    first = max(0, kv_len - q_len - window + 1)
    return total, kv_len - first + min(sinks, first)


def work(case):
    if case["op"] == "norms":
        t, d = case["tokens"], case["dim"]
        size = _SIZE[case["x"]] + 2 * _SIZE[case["residual"]] + _SIZE[case["out"]]
        gate = {"none": 0, "channel": 4 * d, "token": 4 * t, "full": _SIZE[case["residual"]] * t * d}[case["gate"]]
        scales = 4 * t * -(-d // FP8_GROUP) if case["out"] == "e4m3" else 0
        return {"bytes": t * d * size + gate + 8 * d + scales, "flops": 9 * t * d}
    if case["op"] == "axes":
        sections = [int(n) for n in case["sections"].split("/")]
        rows = case["tokens"] * (case["heads"] + 2 * case["kv_heads"])
        turned = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": rows * case["dim"] * (_SIZE[case["x"]] + _SIZE[case["out"]]) +
                (8 + 4 * len(sections)) * case["tokens"] + 5 * sum(sections), "flops": 6 * turned * sum(sections)}
    if case["op"] == "probs":
        t, v = case["tokens"], case["vocab"]
        return {"bytes": t * v * _SIZE[case["x"]] + 12 * t + 8 * t * case["top"], "flops": 6 * t * v}
    q, kv = _lens(case)
    seen = [_visible(a, b, case["window"], case["sinks"]) for a, b in zip(q, kv)]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": 2 * dim * (2 * sum(q) * heads + 2 * sum(s[1] for s in seen) * kv_heads),
            "flops": 4 * dim * heads * sum(s[0] for s in seen)}


# ----------------------------------------------------------------------------------------- inputs

def _axis_of_pair(case):
    """The axis whose position turns each pair: sections one after the other, or the pairs dealt out in turn."""
    left = [int(n) for n in case["sections"].split("/")]
    if case["order"] == "blocks":
        return [a for a, n in enumerate(left) for _ in range(n)]
    out, a = [], 0
    while any(left):
        if left[a]:
            left[a] -= 1
            out.append(a)
        a = (a + 1) % len(left)
    return out


def _positions(case, axes):
    """Spans of text, where all axes agree, and images, whose axes count frames, rows and columns."""
    t = torch.arange(case["tokens"], device="cuda")
    span, inside = t // 300, t % 300
    start = 1000 + span * 310 + (100000 if case["far"] else 0)
    image = (span % 2 == 1)[None]
    grid = torch.stack([torch.zeros_like(t)] + [inside // 17 if a == 1 else inside % (16 + a) for a in range(1, axes)])
    return torch.where(image, start + grid, (start + inside).expand(axes, -1)).to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}

    def normal(*shape, dtype, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(_TYPES[dtype])

    if case["op"] == "norms":
        t, d = case["tokens"], case["dim"]
        # a block's output: a few channels stand out, rows differ in size
        channel = 1.0 + 9.0 * (torch.rand(d, generator=g, device="cuda") > 0.99)
        row = torch.rand(t, 1, generator=g, device="cuda") + 0.5
        s["x"] = (torch.randn(t, d, generator=g, device="cuda") * channel * row).to(_TYPES[case["x"]])
        s["residual"] = normal(t, d, dtype=case["residual"], scale=2.0)
        s["post"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
        s["pre"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
        shape = {"none": None, "channel": (d,), "token": (t, 1), "full": (t, d)}[case["gate"]]
        s["gate"] = None
        if shape:
            s["gate"] = torch.sigmoid(torch.randn(*shape, generator=g, device="cuda"))
            if case["gate"] == "full":
                s["gate"] = s["gate"].to(_TYPES[case["residual"]])
        s["eps"] = 1e-5
        return s
    if case["op"] == "axes":
        t, page, kvh, dim = case["tokens"], case["page"], case["kv_heads"], case["dim"]
        pages = -(-t // page) + 3
        axis = _axis_of_pair(case)
        s["q"] = normal(t, case["heads"], dim, dtype=case["x"])
        s["k"] = normal(t, kvh, dim, dtype=case["x"])
        s["v"] = normal(t, kvh, dim, dtype=case["x"])
        s["positions"] = _positions(case, 1 + max(axis))
        s["axes"] = torch.tensor(axis, dtype=torch.uint8, device="cuda")
        at = torch.randperm(pages, generator=g, device="cuda")
        token = torch.arange(t, device="cuda")
        s["slots"] = at[token // page] * page + token % page
        s["inv_freq"] = (1e6 ** (-torch.arange(len(axis), dtype=torch.float64) / len(axis))).float().cuda()
        s["k_cache"] = normal(pages, kvh, page, dim, dtype=case["out"])
        s["v_cache"] = normal(pages, kvh, page, dim, dtype=case["out"])
        return s
    if case["op"] == "probs":
        t, v = case["tokens"], case["vocab"]
        s["logits"] = torch.empty(t, v, dtype=_TYPES[case["x"]], device="cuda")
        for at in range(0, t, 256):
            n = min(256, t - at)
            z = torch.randn(n, v, generator=g, device="cuda").mul_(2.0)
            # some tokens are likely, more in one row than in another
            likely = torch.randint(0, v, (n, 16), generator=g, device="cuda")
            sure = 12.0 * torch.rand(n, 1, generator=g, device="cuda")
            z.scatter_add_(1, likely, sure * torch.rand(n, 16, generator=g, device="cuda"))
            if case["masked"]:
                z[torch.rand(n, v, generator=g, device="cuda") < 0.5] = -math.inf
                z[:, v - v // 8:] = -math.inf
                z[:, 0] = 0.0
            s["logits"][at:at + n] = z.to(s["logits"].dtype)
        s["tokens"] = torch.randint(0, v, (t,), generator=g, device="cuda", dtype=torch.int32)
        return s
    q_len, kv_len = _lens(case)
    page, dim, sinks = case["page"], case["dim"], case["sinks"]
    need = [-(-n // page) for n in kv_len]
    width = max(need)
    # a sequence holds the pages of its first tokens and of its rows' windows; the others are freed, and unused
    # entries of the table hold -1, as an allocator leaves them
    table = torch.full((len(need), width), -1, dtype=torch.int32)
    pages = 0
    for b, (n, m) in enumerate(zip(q_len, kv_len)):
        first = max(0, m - n - case["window"] + 1) // page
        held = [i for i in range(need[b]) if i >= first or i * page < sinks]
        table[b, held] = torch.arange(pages, pages + len(held), dtype=torch.int32)
        pages += len(held)
    at = torch.randperm(pages + 2, generator=g, device="cuda").to(torch.int32)
    table = table.cuda()
    s["table"] = torch.where(table >= 0, at[table.clamp(min=0).long()], table).contiguous()
    pages += 2
    shape = (pages, page, case["kv_heads"], dim) if case["layout"] == "nhd" else (pages, case["kv_heads"], page, dim)
    for name in ("k_cache", "v_cache"):
        c = torch.empty(shape, dtype=_TYPES[case["x"]], device="cuda").normal_(generator=g)
        s[name] = c.permute(0, 2, 1, 3) if case["layout"] == "nhd" else c
    s["q"] = normal(sum(q_len), case["heads"], dim, dtype=case["x"], scale=1.5)
    starts = [0]
    for n in q_len:
        starts.append(starts[-1] + n)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    s["max_q"], s["max_kv"] = max(q_len), max(kv_len)
    s["scale"] = 1.0 / math.sqrt(dim)
    return s


# ------------------------------------------------------------------------------------------- runs

def run(s):
    case = s["case"]
    if not own:
        return {"norms": _plain_norms, "axes": _plain_axes, "attention": _plain_attention, "probs": _plain_probs}[case["op"]](s)
    from freemoe_b200 import attention, hotpath

    if case["op"] == "norms":
        how = dict(gate=s["gate"], scale=case["scale"], residual_scale=case["residual_scale"], epsilon=s["eps"])
        if case["out"] == "e4m3":
            codes, scales, h = attention.norm_add_norm_fp8(s["x"], s["post"], s["residual"], s["pre"], **how)
            return {"codes": codes, "scales": scales, "h": h}
        y, h = attention.norm_add_norm(s["x"], s["post"], s["residual"], s["pre"], out_dtype=_TYPES[case["out"]], **how)
        return {"y": y, "h": h}
    if case["op"] == "axes":
        q = attention.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"],
                                  s["slots"], axes=s["axes"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "probs":
        chosen, entropy, top, ids = hotpath.token_logprobs(s["logits"], s["tokens"], top=case["top"], scale=case["scale"])
        return {"chosen": chosen, "entropy": entropy, "top": top, "ids": ids}
    return attention.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["q_start"], s["kv_len"],
                                     max_q_len=s["max_q"], max_kv_len=s["max_kv"], scale=s["scale"],
                                     window=case["window"], sinks=case["sinks"])


def _plain_norms(s):
    case = s["case"]
    x = s["x"].float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * s["post"] * case["scale"]
    if s["gate"] is not None:
        x = x * s["gate"].float()
    h = s["residual"].float() * case["residual_scale"] + x
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * s["pre"]
    kept = h.to(s["residual"].dtype)
    if case["out"] != "e4m3":
        return {"y": y.to(_TYPES[case["out"]]), "h": kept}
    t, d = y.shape
    groups = -(-d // FP8_GROUP)
    y = torch.nn.functional.pad(y, (0, groups * FP8_GROUP - d)).view(t, groups, FP8_GROUP)
    scales = y.abs().amax(-1).clamp(min=1e-10) / 448.0
    codes = (y / scales[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return {"codes": codes.view(t, -1)[:, :d].contiguous(), "scales": scales, "h": kept}


def _plain_axes(s):
    case = s["case"]
    out, rot = _TYPES[case["out"]], 2 * s["inv_freq"].shape[0]
    angle = s["positions"][s["axes"].long()].t().double() * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]

    def turn(x):
        x = x.float()
        head, rest = x[..., :rot], x[..., rot:]
        if case["interleaved"]:
            a, b = head[..., 0::2], head[..., 1::2]
            head = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = head[..., : rot // 2], head[..., rot // 2:]
            head = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((head, rest), -1).to(out)

    page, offset = s["slots"] // case["page"], s["slots"] % case["page"]
    s["k_cache"][page, :, offset] = turn(s["k"])
    s["v_cache"][page, :, offset] = s["v"].to(out)
    return {"q": turn(s["q"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    case = s["case"]
    seqs, heads, kvh, dim, page = (case[n] for n in ("seqs", "heads", "kv_heads", "dim", "page"))
    q, q_start, kv_len = s["q"], s["q_start"].long(), s["kv_len"].long()
    dev, tokens, max_q = q.device, q.shape[0], s["max_q"]
    q_len = q_start[1:] - q_start[:-1]
    # the keys that any row of a sequence may see: its first ones and, behind them, those from the first row's window on
    first = (kv_len - q_len - case["window"] + 1).clamp(min=0)
    kept = first.clamp(max=case["sinks"])
    width = min(s["max_kv"], max_q + case["window"] + case["sinks"])
    column = torch.arange(width, device=dev)
    key = torch.where(column < kept[:, None], column, column - kept[:, None] + first[:, None])
    here = key < kv_len[:, None]
    at = torch.where(here, key, 0)
    where = s["table"].gather(1, at // page).clamp(min=0).long()
    k = s["k_cache"][where, :, at % page].permute(0, 2, 1, 3).float()
    v = s["v_cache"][where, :, at % page].permute(0, 2, 1, 3).float()
    row = torch.arange(max_q, device=dev)
    padded = q[(q_start[:-1, None] + row).clamp(max=tokens - 1)].float()  # [seqs, max_q, heads, dim]
    padded = padded.view(seqs, max_q, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, -1, dim)
    position = ((kv_len - q_len)[:, None] + row)[..., None]  # of each row among its keys
    seen = (key[:, None] <= position) & here[:, None]
    seen &= (key[:, None] > position - case["window"]) | (key < case["sinks"])[:, None]
    score = (padded @ k.transpose(-1, -2)).mul_(s["scale"]).view(seqs, kvh, heads // kvh, max_q, width)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(-1)
    o = (weight.view(seqs, kvh, -1, width) @ v).view(seqs, kvh, heads // kvh, max_q, dim)
    o = o / torch.where(total == 0, 1.0, total)[..., None]
    token = torch.arange(tokens, device=dev)
    seq = torch.searchsorted(q_start[1:], token, right=True)
    return o[seq, :, :, token - q_start[seq]].reshape(tokens, heads, dim).to(q.dtype)


def _plain_probs(s):
    case, k = s["case"], s["case"]["top"]
    parts = []
    index = torch.arange(case["vocab"], device=s["logits"].device)
    for at in range(0, case["tokens"], 512):  # some GB of scores at a time
        raw = s["logits"][at:at + 512].float()
        z = raw * case["scale"]
        high = z.amax(-1, keepdim=True)
        e = (z - high).exp()
        total = e.sum(-1, keepdim=True)
        log_total = high + total.log()
        entropy = log_total[:, 0] - torch.where(e > 0, z * (e / total), 0.0).sum(-1)
        chosen = (z.gather(1, s["tokens"][at:at + 512, None].long()) - log_total)[:, 0]
        # one whole number an entry: larger values first, among equal ones the lower index
        bits = (raw + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2 ** 22 - index
        ids = order.topk(k, -1).indices
        parts.append((chosen, entropy, z.gather(1, ids) - log_total, ids.int()))
    return dict(zip(("chosen", "entropy", "top", "ids"), (torch.cat(p) for p in zip(*parts))))


# ------------------------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norms":
        return _exact_norms(s)
    if case["op"] == "axes":
        return _exact_axes(s)
    if case["op"] == "probs":
        return _exact_probs(s)
    q_len, kv_len = _lens(case)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    for n, m, pages in zip(q_len, kv_len, s["table"].long()):
        low = max(0, m - n + 1 - case["window"])
        key = torch.tensor([i for i in range(m) if i >= low or i < case["sinks"]], device="cuda")
        where, offset = pages[key // page], key % page
        back = torch.arange(m - n, m, device="cuda")[:, None] - key  # how far behind its row a key lies
        hidden = (back < 0) | ((back >= case["window"]) & (key >= case["sinks"]))
        for h in range(case["kv_heads"]):
            k, v = s["k_cache"][where, h, offset].double(), s["v_cache"][where, h, offset].double()
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][begin:begin + n, j].double() @ k.T) * s["scale"]
                out[begin:begin + n, j] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
        begin += n
    return out


def _exact_norms(s):
    case, eps = s["case"], s["eps"]
    x = s["x"].double()
    x = torch.einsum("td,d,t->td", x, s["post"].double(), (torch.einsum("td,td->t", x, x) / case["dim"] + eps) ** -0.5)
    gate = torch.ones((), dtype=torch.float64, device="cuda") if s["gate"] is None else s["gate"].double()
    h = case["residual_scale"] * s["residual"].double() + case["scale"] * (gate * x)
    y = torch.einsum("td,d,t->td", h, s["pre"].double(), (torch.einsum("td,td->t", h, h) / case["dim"] + eps) ** -0.5)
    if case["out"] != "e4m3":
        return {"y": y, "h": h}
    codes, scales = torch.empty_like(y), []
    for c in range(0, case["dim"], FP8_GROUP):
        part = y[:, c:c + FP8_GROUP]
        scale = part.abs().max(dim=1).values.clamp(min=1e-10) / 448.0
        # e4m3: 3 bits behind the leading one, the smallest step 2^-9
        z = part / scale[:, None]
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        codes[:, c:c + FP8_GROUP] = torch.round(z / step) * step
        scales.append(scale)
    return {"codes": codes, "scales": torch.stack(scales, 1), "h": h}


def _exact_axes(s):
    case, half = s["case"], s["inv_freq"].shape[0]
    first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    got = {}
    for name in ("q", "k"):
        x = s[name].double()
        z = torch.complex(x[..., first], x[..., second])
        for axis in range(s["positions"].shape[0]):
            mine = s["axes"] == axis
            turn = s["positions"][axis].double()[:, None] * s["inv_freq"][mine].double()
            z[..., mine] *= torch.polar(torch.ones_like(turn), turn)[:, None]
        x[..., first], x[..., second] = z.real.clone(), z.imag.clone()
        got[name] = x
    caches = []
    for cache, new in (("k_cache", got["k"]), ("v_cache", s["v"].double())):
        flat = s[cache].double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
        flat.index_copy_(0, s["slots"], new)
        caches.append(flat.view(-1, case["page"], case["kv_heads"], case["dim"]).transpose(1, 2).contiguous())
    return {"q": got["q"], "k_cache": caches[0], "v_cache": caches[1]}


def _exact_probs(s):
    case = s["case"]
    parts = []
    for at in range(0, case["tokens"], 128):
        logits = s["logits"][at:at + 128]
        log_p = torch.log_softmax(logits.double() * case["scale"], -1)
        values, order = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
        ids = order[:, :case["top"]]
        chosen = log_p.gather(1, s["tokens"][at:at + 128, None].long())[:, 0]
        parts.append((chosen, torch.special.entr(log_p.exp()).sum(-1), log_p.gather(1, ids), ids.int()))
    return dict(zip(("chosen", "entropy", "top", "ids"), (torch.cat(p) for p in zip(*parts))))
