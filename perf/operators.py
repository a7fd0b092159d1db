"""The attention side of a decoder layer, as workloads: RMS norm with the residual's addition (and an
8-bit output), rotary positions with the write into a paged K/V cache, and attention of new tokens
over that cache.

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
        # the norm before a block while one sequence decodes: latency alone
        {"name": "norm one token", "op": "norm", "tokens": 1, "dim": 4096, "x": "bf16", "residual": True, "out": "bf16"},
        # the same norm for a prompt batch whose next product or exchange takes 8-bit rows
        {"name": "norm prompt to 8 bits", "op": "norm", "tokens": 8192, "dim": 4096, "x": "bf16", "residual": True,
         "out": "e4m3"},
        # a final norm of an odd width, f32 out for the output head
        {"name": "norm odd width", "op": "norm", "tokens": 777, "dim": 2050, "x": "f16", "residual": False, "out": "f32"},
        # 16 decoding sequences, far positions, q/k/v as the quantised products leave them (f32)
        {"name": "rope 16 decoding", "op": "rope", "tokens": 16, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "x": "f32", "out": "bf16", "interleaved": False, "scaled": False, "page": 16, "far": True},
        # a prompt chunk of 8192 tokens, interleaved pairs, frequencies scaled for a long context
        {"name": "rope prompt interleaved", "op": "rope", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "x": "bf16", "out": "bf16", "interleaved": True, "scaled": True, "page": 64, "far": False},
        # part of a head of 80 rotated, ragged count of tokens
        {"name": "rope part of a head", "op": "rope", "tokens": 1001, "heads": 28, "kv_heads": 4, "dim": 80, "rot": 32,
         "x": "f16", "out": "f16", "interleaved": False, "scaled": False, "page": 48, "far": False},
        # one short sequence decodes one token: latency
        _attn("decode one short", "bf16", 1, 1, 777, 32, 8, 128, 16),
        # 64 sequences of ragged lengths decode together: the serving batch
        _attn("decode 64 ragged", "bf16", 64, 1, 8192, 32, 8, 128, 16, ragged=True),
        # one very long sequence, few key heads: the long axis has to be split
        _attn("decode one long", "f16", 1, 1, 131071, 64, 4, 128, 64),
        # a whole prompt at once
        _attn("prompt 8192", "bf16", 1, 8192, 8192, 32, 8, 128, 64),
        # prompt chunks behind contexts of ragged lengths, odd group of heads, smaller heads, token-major pages
        _attn("chunks on contexts", "f16", 4, 500, 12000, 28, 4, 64, 48, ragged=True, layout="nhd"),
        # one chunk beside seven decoding sequences, sliding window
        _attn("chunk and decodes, window", "bf16", 8, 510, 4099, 16, 16, 128, 32, ragged=True, mixed=True, window=1000),
    ]


def _attn(name, dtype, seqs, q_len, kv_len, heads, kv_heads, dim, page, ragged=False, mixed=False, window=0,
          layout="hnd"):
    return {"name": name, "op": "attention", "x": dtype, "seqs": seqs, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged, "mixed": mixed, "window": window,
            "layout": layout}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "rope", "attention", "attention"])
    if op == "norm":
        return {"op": op, "tokens": _log(rng, 1, 8192), "dim": _log(rng, 64, 8192), "x": rng.choice(["bf16", "f16", "f32"]),
                "residual": rng.random() < 0.7, "out": rng.choice(["bf16", "f16", "f32", "e4m3"])}
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128])
        heads, kv_heads = rng.choice([(32, 8), (16, 16), (28, 4), (64, 4), (16, 1), (8, 2)])
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim // 2, 2 * rng.randrange(1, dim // 2)]), "x": rng.choice(["f32", "bf16", "f16"]),
                "out": rng.choice(["bf16", "f16"]), "interleaved": rng.random() < 0.5, "scaled": rng.random() < 0.5,
                "page": rng.choice([8, 16, 32, 48, 64, 128]), "far": rng.random() < 0.5}
    heads, kv_heads = rng.choice([(32, 8), (16, 16), (28, 4), (64, 4), (16, 1), (8, 2)])
    while True:
        kind = rng.choice(["decode", "prompt", "chunk"])
        seqs = _log(rng, 1, {"decode": 128, "prompt": 8, "chunk": 16}[kind])
        q_len = 1 if kind == "decode" else _log(rng, 1, 4096 if kind == "prompt" else 1024)
        kv_len = q_len if kind == "prompt" else _log(rng, q_len, 65536 if kind == "decode" else 16384)
        dim = rng.choice([64, 80, 96, 128])
        # the plain form's scores and caches stay within a few GB, the work within the listed prompt's
        if seqs * heads * q_len * kv_len <= 1 << 30 and seqs * kv_len * kv_heads * dim <= 1 << 29:
            break
    case = _attn("", rng.choice(["bf16", "f16"]), seqs, q_len, kv_len, heads, kv_heads, dim,
                 rng.choice([8, 16, 32, 48, 64, 128, 256]), ragged=rng.random() < 0.6,
                 mixed=kind == "chunk" and rng.random() < 0.4, window=rng.choice([0, 0, 0, _log(rng, 1, kv_len)]),
                 layout=rng.choice(["hnd", "nhd"]))
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


def _visible(q_len, kv_len, window):
    """How many keys the rows of a causal chunk see in all, and how many keys any of them sees."""
    first = kv_len - q_len + 1
    if not window:
        return q_len * (first + kv_len) // 2, kv_len
    return sum(min(window, first + i) for i in range(q_len)), min(kv_len, window + q_len - 1)


def work(case):
    if case["op"] == "norm":
        t, d = case["tokens"], case["dim"]
        size = _SIZE[case["x"]] * (3 if case["residual"] else 1) + _SIZE[case["out"]]
        scales = 4 * t * -(-d // FP8_GROUP) if case["out"] == "e4m3" else 0
        return {"bytes": t * d * size + 4 * d + scales, "flops": 5 * t * d}
    if case["op"] == "rope":
        rows = case["tokens"] * (case["heads"] + 2 * case["kv_heads"])
        turned = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": rows * case["dim"] * (_SIZE[case["x"]] + _SIZE[case["out"]]) + 12 * case["tokens"] + 2 * case["rot"],
                "flops": 3 * turned * case["rot"]}
    q, kv = _lens(case)
    seen = [_visible(a, b, case["window"]) for a, b in zip(q, kv)]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": 2 * dim * (2 * sum(q) * heads + 2 * sum(s[1] for s in seen) * kv_heads),
            "flops": 4 * dim * heads * sum(s[0] for s in seen)}


# ----------------------------------------------------------------------------------------- inputs

def _frequencies(rot, scaled):
    """Rotary frequencies of base 500000; `scaled`: the slow ones divided by 8, a ramp between, as contexts are stretched."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = 500000.0 ** (-2.0 * i / rot)
    if scaled:
        turns = 8192.0 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / 8.0
    return f.float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}

    def normal(*shape, dtype, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(_TYPES[dtype])

    if case["op"] == "norm":
        t, d = case["tokens"], case["dim"]
        # hidden states: a few channels stand out, rows differ in size
        channel = 1.0 + 9.0 * (torch.rand(d, generator=g, device="cuda") > 0.99)
        row = torch.rand(t, 1, generator=g, device="cuda") + 0.5
        s["x"] = (torch.randn(t, d, generator=g, device="cuda") * channel * row).to(_TYPES[case["x"]])
        s["residual"] = normal(t, d, dtype=case["x"], scale=2.0) if case["residual"] else None
        s["weight"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
        s["eps"] = 1e-5
        return s
    if case["op"] == "rope":
        t, page, kvh, dim = case["tokens"], case["page"], case["kv_heads"], case["dim"]
        pages = -(-t // page) + 3
        s["q"] = normal(t, case["heads"], dim, dtype=case["x"])
        s["k"] = normal(t, kvh, dim, dtype=case["x"])
        s["v"] = normal(t, kvh, dim, dtype=case["x"])
        if case["far"]:
            s["positions"] = torch.randint(0, 131072, (t,), generator=g, device="cuda", dtype=torch.int32)
        else:
            s["positions"] = torch.arange(1000, 1000 + t, device="cuda", dtype=torch.int32)
        at = torch.randperm(pages, generator=g, device="cuda")
        token = torch.arange(t, device="cuda")
        s["slots"] = at[token // page] * page + token % page
        s["inv_freq"] = _frequencies(case["rot"], case["scaled"]).cuda()
        s["factor"] = 1.2 if case["scaled"] else 1.0
        s["k_cache"] = normal(pages, kvh, page, dim, dtype=case["out"])
        s["v_cache"] = normal(pages, kvh, page, dim, dtype=case["out"])
        return s
    q_len, kv_len = _lens(case)
    page, dim = case["page"], case["dim"]
    need = [-(-n // page) for n in kv_len]
    width = max(need)
    pages = sum(need) + 2
    at = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    # unused entries of the table hold -1, as an allocator leaves them
    first = torch.tensor([sum(need[:b]) for b in range(len(need))], device="cuda")[:, None]
    col = torch.arange(width, device="cuda")[None, :]
    used = col < torch.tensor(need, device="cuda")[:, None]
    s["table"] = torch.where(used, at[(first + col).clamp(max=pages - 1)], torch.full_like(at[:1], -1)).contiguous()
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
    if own:
        from freemoe_b200 import attention

        if case["op"] == "norm":
            if case["out"] == "e4m3":
                codes, scales, h = attention.add_rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], epsilon=s["eps"])
                return {"codes": codes, "scales": scales, "h": h}
            y, h = attention.add_rms_norm(s["x"], s["weight"], residual=s["residual"], epsilon=s["eps"],
                                          out_dtype=_TYPES[case["out"]])
            return {"y": y, "h": h}
        if case["op"] == "rope":
            q = attention.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"],
                                      s["slots"], interleaved=case["interleaved"], attention_factor=s["factor"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return attention.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["q_start"], s["kv_len"],
                                         max_q_len=s["max_q"], max_kv_len=s["max_kv"], scale=s["scale"],
                                         window=case["window"])
    return {"norm": _plain_norm, "rope": _plain_rope, "attention": _plain_attention}[case["op"]](s)


def _plain_norm(s):
    case = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"]
    kept = h.to(s["x"].dtype) if s["residual"] is not None else None
    if case["out"] != "e4m3":
        return {"y": y.to(_TYPES[case["out"]]), "h": kept}
    t, d = y.shape
    groups = -(-d // FP8_GROUP)
    y = torch.nn.functional.pad(y, (0, groups * FP8_GROUP - d)).view(t, groups, FP8_GROUP)
    scales = y.abs().amax(-1).clamp(min=1e-10) / 448.0
    codes = (y / scales[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return {"codes": codes.view(t, -1)[:, :d].contiguous(), "scales": scales, "h": kept}


def _turn(x, cos, sin, rot, interleaved):
    x = x.float()
    cos, sin = cos[:, None, :], sin[:, None, :]
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = head[..., : rot // 2], head[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1)


def _plain_rope(s):
    case = s["case"]
    out = _TYPES[case["out"]]
    angle = s["positions"].float()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle) * s["factor"], torch.sin(angle) * s["factor"]
    q = _turn(s["q"], cos, sin, case["rot"], case["interleaved"]).to(out)
    k = _turn(s["k"], cos, sin, case["rot"], case["interleaved"]).to(out)
    page, offset = s["slots"] // case["page"], s["slots"] % case["page"]
    s["k_cache"][page, :, offset] = k
    s["v_cache"][page, :, offset] = s["v"].to(out)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    case = s["case"]
    seqs, heads, kvh, dim, page = (case[n] for n in ("seqs", "heads", "kv_heads", "dim", "page"))
    q, q_start, kv_len = s["q"], s["q_start"].long(), s["kv_len"].long()
    dev, tokens, width, max_q = q.device, q.shape[0], s["table"].shape[1] * page, s["max_q"]
    at = s["table"].clamp(min=0).long()
    k = s["k_cache"][at].transpose(1, 2).reshape(seqs, kvh, width, dim).float()
    v = s["v_cache"][at].transpose(1, 2).reshape(seqs, kvh, width, dim).float()
    key = torch.arange(width, device=dev)
    v = torch.where((key < kv_len[:, None])[:, None, :, None], v, 0.0)
    row = torch.arange(max_q, device=dev)
    q_len = q_start[1:] - q_start[:-1]
    padded = q[(q_start[:-1, None] + row).clamp(max=tokens - 1)].float()  # [seqs, max_q, heads, dim]
    padded = padded.view(seqs, max_q, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, -1, dim)
    position = (kv_len - q_len)[:, None] + row  # of each row among its keys
    seen = (key <= position[..., None]) & (key < kv_len[:, None, None])
    if case["window"]:
        seen &= key > position[..., None] - case["window"]
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


# ------------------------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if case["residual"] else 0.0)
        root = torch.sqrt(torch.einsum("td,td->t", h, h) / case["dim"] + s["eps"])
        y = torch.einsum("td,d,t->td", h, s["weight"].double(), 1.0 / root)
        kept = h if case["residual"] else None
        if case["out"] != "e4m3":
            return {"y": y, "h": kept}
        codes, scales = torch.empty_like(y), []
        for c in range(0, case["dim"], FP8_GROUP):
            part = y[:, c:c + FP8_GROUP]
            scale = part.abs().max(dim=1).values.clamp(min=1e-10) / 448.0
            # e4m3: 3 bits behind the leading one, the smallest step 2^-9
            z = part / scale[:, None]
            step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
            codes[:, c:c + FP8_GROUP] = torch.round(z / step) * step
            scales.append(scale)
        return {"codes": codes, "scales": torch.stack(scales, 1), "h": kept}
    if case["op"] == "rope":
        rot, half = case["rot"], case["rot"] // 2
        turn = torch.polar(torch.full((case["tokens"], half), float(s["factor"]), dtype=torch.float64, device="cuda"),
                           s["positions"].double()[:, None] * s["inv_freq"].double())
        first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        got = {}
        for name in ("q", "k"):
            x = s[name].double()
            z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
            x[..., first], x[..., second] = z.real.clone(), z.imag.clone()
            got[name] = x
        caches = []
        for cache, new in (("k_cache", got["k"]), ("v_cache", s["v"].double())):
            flat = s[cache].double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
            flat.index_copy_(0, s["slots"], new)
            caches.append(flat.view(-1, case["page"], case["kv_heads"], case["dim"]).transpose(1, 2).contiguous())
        return {"q": got["q"], "k_cache": caches[0], "v_cache": caches[1]}
    q_len, kv_len = _lens(case)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (n, m) in enumerate(zip(q_len, kv_len)):
        key = torch.arange(m, device="cuda")
        where, offset = s["table"][b].long()[key // page], key % page
        back = (torch.arange(m - n, m, device="cuda")[:, None] - key)  # how far behind its row a key lies
        hidden = (back < 0) | (back >= case["window"]) if case["window"] else back < 0
        for h in range(case["kv_heads"]):
            k, v = s["k_cache"][where, h, offset].double(), s["v_cache"][where, h, offset].double()
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][begin:begin + n, j].double() @ k.T) * s["scale"]
                out[begin:begin + n, j] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
        begin += n
    return out
