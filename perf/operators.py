"""Cases of the decoder-layer operators: block planning, the 4-bit paged KV cache, attention over it, and the residual
RMS norm with 8-bit output.  `run` computes them with elementary torch operations, or, where `own` is true, through
`dracomancer_llmengine_b200.decoder`."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TILE = 16      # tokens of one cache tile
GROUP = 32     # channels that share a scale


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a serving batch: every request grows by one token, some need a page
        {"name": "blocks decode", "op": "blocks", "requests": 64, "ctx": 4096, "new": 1, "page": 16, "spare": 3},
        # a step that mixes prefill chunks and decode over many requests
        {"name": "blocks mixed", "op": "blocks", "requests": 1000, "ctx": 16384, "new": 255, "page": 32, "spare": 100},
        # the new tokens of one decode step go into the cache and are read back
        {"name": "append decode", "op": "append", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16"},
        # a prefill chunk of fp32 activations, as the library's projections produce them
        {"name": "append prefill", "op": "append", "tokens": 8192, "kv_heads": 4, "dim": 128, "page": 64, "type": "f32"},
        # one user, a short odd context, fp32: latency
        attn_case("attend one", 1, 1001, 1, 32, 4, 128, 16, "f32"),
        # a decode batch with ragged contexts
        attn_case("attend batch", 64, 4096, 1, 64, 8, 128, 16, "bf16"),
        # a few users with very long contexts
        attn_case("attend long", 4, 131001, 1, 32, 8, 128, 64, "bf16", lse=True),
        # a sliding-window layer with its first tokens kept visible, wide heads
        attn_case("attend window", 48, 32768, 1, 16, 2, 256, 32, "f16", window=4096, sinks=4),
        # chunks of prefill that attend to what is cached and to themselves
        attn_case("attend chunk", 4, 8192, 512, 32, 4, 128, 32, "bf16"),
        # one decode token of the widest configuration, scales per 256 as the 8-bit activations of the experts
        {"name": "norm decode", "op": "norm", "tokens": 1, "hidden": 7168, "type": "f32", "code": "int8", "group": 256,
         "residual": True, "y": True},
        # a prefill chunk, scales per 128
        {"name": "norm prefill", "op": "norm", "tokens": 4096, "hidden": 4096, "type": "bf16", "code": "e4m3",
         "group": 128, "residual": True, "y": True},
        # an odd number of tokens, one scale per token, codes alone
        {"name": "norm row scale", "op": "norm", "tokens": 8191, "hidden": 2048, "type": "f16", "code": "int8",
         "group": 0, "residual": False, "y": False},
    ]


def attn_case(name, requests, ctx, new, heads, kv_heads, dim, page, kind, window=0, sinks=0, lse=False, empty=False):
    return {"name": name, "op": "attend", "requests": requests, "ctx": ctx, "new": new, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "type": kind, "window": window, "sinks": sinks, "lse": lse,
            "empty": empty}


def _log(rng, lo, hi):
    """An odd number, or now and then an even one, spread over the logarithm of [lo, hi]."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    return v if rng.random() < 0.25 and v & (v - 1) == 0 else max(lo, min(hi, v | 1))


def draw(rng):
    op = rng.choice(["blocks", "append", "attend", "attend", "attend", "norm", "norm"])
    if op == "blocks":
        return {"op": op, "requests": _log(rng, 1, 1000), "ctx": _log(rng, 1, 16384), "new": _log(rng, 1, 255),
                "page": rng.choice([16, 32, 64, 128]), "spare": rng.choice([-2, 0, 1, 100])}
    if op == "append":
        kv, dim = rng.choice([(8, 128), (4, 128), (2, 256), (1, 128), (8, 64), (5, 64)])
        return {"op": op, "tokens": _log(rng, 1, 4097), "kv_heads": kv, "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["f32", "f16", "bf16"])}
    if op == "norm":
        hidden = rng.choice([2048, 4096, 7168, 5120, 896, 1023])
        group = 0 if hidden == 1023 else rng.choice([0, 32, 64, 128] + ([256] if hidden % 256 == 0 else []))
        return {"op": op, "tokens": _log(rng, 1, 4095 if hidden > 4096 else 8191), "hidden": hidden,
                "type": rng.choice(["f32", "f16", "bf16"]) if hidden <= 4096 else rng.choice(["f16", "bf16"]),
                "code": rng.choice(["int8", "e4m3"]), "group": group, "residual": rng.random() < 0.7,
                "y": rng.random() < 0.6}
    heads, kv, dim = rng.choice([(32, 4, 128), (64, 8, 128), (16, 2, 256), (32, 8, 64), (40, 8, 128), (8, 8, 128),
                                 (12, 1, 128), (20, 5, 64)])
    if rng.random() < 0.25:   # a chunk of prefill
        new, requests = _log(rng, 5, 512), _log(rng, 1, 4)
        ctx = _log(rng, new, 8192)
    else:                     # single tokens, or a few drafted ones
        new, requests = rng.choice([1, 1, 1, 2, 4]), _log(rng, 1, 64)
        ctx = _log(rng, max(8, new), min(65536, 2 ** 30 // (2 * requests * kv * dim)))
    windowed = rng.random() < 0.35
    c = attn_case("", requests, ctx, new, heads, kv, dim, rng.choice([16, 32, 64, 128]),
                  rng.choice(["f32", "f16", "bf16"]) if new <= 4 else rng.choice(["f16", "bf16"]),
                  window=_log(rng, 1, max(2, ctx)) if windowed else 0, sinks=rng.choice([0, 1, 4, 17]) if windowed else 0,
                  lse=rng.random() < 0.3, empty=rng.random() < 0.15 and requests > 1)
    del c["name"]
    return c


def _ragged(n, lo, hi, salt):
    """n whole numbers in [lo, hi], the first one hi: the same for every seed, so that a case's work is fixed."""
    return [hi if i == 0 else lo + ((i + salt) * 2654435761 >> 7) % (hi - lo + 1) for i in range(n)]


def _attn_lens(c):
    new = _ragged(c["requests"], max(1, c["new"] // 2), c["new"], 3)
    ctx = [max(n, v) for n, v in zip(new, _ragged(c["requests"], max(1, c["ctx"] // 4), c["ctx"], 11))]
    if c["empty"]:
        ctx[-1] = 0   # a request with a query and nothing in the cache
    return new, ctx


def _block_lens(c):
    new = _ragged(c["requests"], 1 if c["new"] == 1 else 0, c["new"], 5)
    ctx = _ragged(c["requests"], 0, c["ctx"], 7)
    return new, ctx


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- the cache's layout
# pages: uint8 [pages][kv heads][page/16 tiles][20*D]; a tile of 16 tokens holds, one after the other,
#   K codes  [16 tokens][4][D/32][4 bytes]: byte b of (token, q, g) has channels g*32 + q*8 + 2b (low nibble), + 1
#   K scales [8 token pairs][D/32][2 tokens] fp16, K minima [16 tokens][D/32] fp16
#   V codes  [8 token pairs][8][D/32][2 tokens][2 bytes]: byte b of (pair, n, g, h) has channels g*32 + n*4 + 2b, + 1
#   V scales [8 token pairs][D/32][2 tokens] fp16, V middles likewise
# K value = scale * code + minimum, V value = scale * (code - 8) + middle
def _parts(pages, d):
    """Views of the parts of pages [..., 20*D]."""
    lead, g = pages.shape[:-1], d // GROUP
    half = lambda a, b: pages[..., a * d:b * d].view(torch.float16)  # noqa: E731
    return (pages[..., :8 * d].view(*lead, 8, 2, 4, g, 4), half(8, 9).view(*lead, 8, g, 2), half(9, 10).view(*lead, 8, 2, g),
            pages[..., 10 * d:18 * d].view(*lead, 8, 8, g, 2, 2), half(18, 19).view(*lead, 8, g, 2),
            half(19, 20).view(*lead, 8, g, 2))


def _codes(x, value):
    """Codes, scales and offsets of x [..., D] in groups of 32: value 0 for K (the minimum), 8 for V (the middle)."""
    x = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi - lo) * (1.0 / 15.0)).half()
    m = (lo + s.float() * value).half()
    inv = torch.where(s > 0, 1.0 / s.float(), torch.zeros_like(lo))
    c = ((x - m.float()[..., None]) * inv[..., None]).round() + value
    return c.clamp(0, 15).to(torch.uint8), s, m


def _nibbles(c):
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _k_bytes(c):
    """[..., D/32, 32] codes as K bytes [..., 4, D/32, 4]."""
    return _nibbles(c).unflatten(-1, (4, 4)).transpose(-2, -3)


def _v_bytes(c):
    """[..., D/32, 32] codes as V bytes [..., 8, D/32, 2]."""
    return _nibbles(c).unflatten(-1, (8, 2)).transpose(-2, -3)


def _decode(pages, d, to=torch.float32):
    """K and V values [..., 16, D] of pages [..., 20*D]."""
    kc, ks, km, vc, vs, vm = _parts(pages, d)
    lead, g = pages.shape[:-1], d // GROUP
    split = lambda b: torch.stack((b & 15, b >> 4), -1)  # noqa: E731
    k = split(kc).transpose(-3, -4).reshape(*lead, 16, g, GROUP).to(to)                      # 8,2,[g,4,4,2]
    k = k * ks.transpose(-1, -2).reshape(*lead, 16, g, 1).to(to) + km.reshape(*lead, 16, g, 1).to(to)
    n = len(lead)
    v = split(vc).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4, n + 5).reshape(*lead, 16, g, GROUP).to(to) - 8
    v = v * vs.transpose(-1, -2).reshape(*lead, 16, g, 1).to(to) + vm.transpose(-1, -2).reshape(*lead, 16, g, 1).to(to)
    return k.flatten(-2), v.flatten(-2)


def _random_pages(n_pages, kv_heads, page, d, gen):
    """Pages filled with quantised random keys (with an offset for each channel) and values."""
    pages = torch.empty(n_pages, kv_heads, page // TILE, 20 * d, dtype=torch.uint8, device=DEV)
    kc, ks, km, vc, vs, vm = _parts(pages, d)
    off = torch.randn(kv_heads, 1, d, device=DEV, generator=gen)
    step = max(1, (1 << 27) // (kv_heads * page * d))
    for a in range(0, n_pages, step):
        b = min(n_pages, a + step)
        shape = (b - a, kv_heads, page // TILE * TILE, d)
        c, s, m = _codes(torch.randn(shape, device=DEV, generator=gen) + 0.5 * off, 0)
        kc[a:b] = _k_bytes(c).reshape(kc[a:b].shape)
        ks[a:b] = s.reshape(b - a, kv_heads, page // TILE, 8, 2, -1).transpose(-1, -2)
        km[a:b] = m.reshape(km[a:b].shape)
        c, s, m = _codes(torch.randn(shape, device=DEV, generator=gen), 8)
        vc[a:b] = _v_bytes(c).reshape(b - a, kv_heads, page // TILE, 8, 2, 8, d // GROUP, 2).permute(0, 1, 2, 3, 5, 6, 4, 7)
        vs[a:b] = s.reshape(b - a, kv_heads, page // TILE, 8, 2, -1).transpose(-1, -2)
        vm[a:b] = m.reshape(b - a, kv_heads, page // TILE, 8, 2, -1).transpose(-1, -2)
    return pages


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    return {"blocks": _prepare_blocks, "append": _prepare_append, "attend": _prepare_attend,
            "norm": _prepare_norm}[case["op"]](case, _gen(seed))


def _prepare_blocks(c, gen):
    new, ctx = _block_lens(c)
    page = c["page"]
    held = [_ceil(v, page) for v in ctx]
    need = sum(_ceil(v + n, page) for v, n in zip(ctx, new)) - sum(held)
    total = sum(held) + need + max(0, c["spare"])
    ids = torch.randperm(total, device=DEV, generator=gen).int()
    width = _ceil(c["ctx"] + c["new"], page)
    first = torch.cumsum(_ints([0] + held[:-1]), 0)
    col = torch.arange(width, device=DEV)
    table = torch.where(col < _ints(held)[:, None], ids[(first[:, None] + col).clamp(max=total - 1)], -1).int()
    free = ids[sum(held):].contiguous()
    n_free = max(0, need + c["spare"])   # a negative spare: the last requests get nothing
    s = {"op": "blocks", "ctx": _ints(ctx), "new": _ints(new), "table": table, "free": free, "n_free": _ints([n_free]),
         "page": page, "cap": sum(new) + 7}
    if own:
        from dracomancer_llmengine_b200 import decoder
        s["plan"] = decoder.BlockPlan(c["requests"], s["cap"], DEV)
    return s


def _prepare_append(c, gen):
    kind, n, hkv, d, page = TYPES[c["type"]], c["tokens"], c["kv_heads"], c["dim"], c["page"]
    n_pages = _ceil(n, page) + 3
    # keys and values as the two last parts of one projection's rows
    qkv = torch.randn(n, 3 * hkv, d, device=DEV, generator=gen)
    qkv[:, hkv:2 * hkv] += 3 * torch.randn(hkv, d, device=DEV, generator=gen)
    qkv = qkv.to(kind)
    slots = torch.randperm(n_pages * page, device=DEV, generator=gen)[:n].int()
    s = {"op": "append", "k": qkv[:, hkv:2 * hkv], "v": qkv[:, 2 * hkv:], "slots": slots, "page": page, "d": d,
         "pages": torch.zeros(n_pages, hkv, page // TILE, 20 * d, dtype=torch.uint8, device=DEV),
         "k_out": torch.empty(n, hkv, d, dtype=kind, device=DEV), "v_out": torch.empty(n, hkv, d, dtype=kind, device=DEV)}
    if own:
        from dracomancer_llmengine_b200 import decoder
        s["cache"] = decoder.KV4Cache(s["pages"], page, d)
    return s


def _prepare_attend(c, gen):
    kind, page, d = TYPES[c["type"]], c["page"], c["dim"]
    new, ctx = _attn_lens(c)
    held = [_ceil(v, page) for v in ctx]
    n_pages = sum(held) + 1
    width = max(held)
    ids = torch.randperm(n_pages, device=DEV, generator=gen).int()
    first = torch.cumsum(_ints([0] + held[:-1]), 0)
    col = torch.arange(width, device=DEV)
    table = torch.where(col < _ints(held)[:, None], ids[(first[:, None] + col).clamp(max=n_pages - 1)], -1).int()
    n = sum(new)
    q = (2 * torch.randn(n, c["heads"], d, device=DEV, generator=gen)).to(kind)
    s = {"op": "attend", "q": q, "table": table, "page": page, "d": d, "max_q": max(new), "max_seq": max(ctx),
         "cu_q": _ints([sum(new[:i]) for i in range(len(new) + 1)]), "seq_len": _ints(ctx), "window": c["window"],
         "sinks": c["sinks"], "pages": _random_pages(n_pages, c["kv_heads"], page, d, gen), "out": torch.empty_like(q),
         "lse": torch.empty(n, c["heads"], device=DEV) if c["lse"] else None}
    if own:
        from dracomancer_llmengine_b200 import decoder
        s["cache"] = decoder.KV4Cache(s["pages"], page, d)
    return s


def _prepare_norm(c, gen):
    kind, n, h = TYPES[c["type"]], c["tokens"], c["hidden"]
    x = torch.randn(n, h, device=DEV, generator=gen)
    x *= torch.exp(torch.randn(h, device=DEV, generator=gen))    # channels of unlike size, as hidden states have
    r = (4 * torch.randn(n, h, device=DEV, generator=gen)).to(kind) if c["residual"] else None
    group = c["group"] or h
    return {"op": "norm", "x": x.to(kind), "r": r, "w": 1 + 0.2 * torch.randn(h, device=DEV, generator=gen), "eps": 1e-6,
            "group": c["group"], "h": torch.empty_like(r) if r is not None else None,
            "y": torch.empty(n, h, dtype=kind, device=DEV) if c["y"] else None,
            "q": torch.empty(n, h, dtype=torch.int8 if c["code"] == "int8" else torch.float8_e4m3fn, device=DEV),
            "scales": torch.empty(n, h // group, device=DEV)}


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        return {"blocks": _own_blocks, "append": _own_append, "attend": _own_attend, "norm": _own_norm}[s["op"]](s)
    return {"blocks": _plain_blocks, "append": _plain_append, "attend": _plain_attend, "norm": _plain_norm}[s["op"]](s)


def _own_blocks(s):
    from dracomancer_llmengine_b200 import decoder
    p = s["plan"]
    decoder.plan_blocks(s["ctx"], s["new"], s["table"], s["free"], s["n_free"], s["page"], p)
    return {"table": s["table"], "slots": p.slots, "positions": p.positions, "cu": p.cu_new, "seq": p.seq_len,
            "n_free": p.n_free, "refused": p.refused}


def _own_append(s):
    s["cache"].append(s["k"], s["v"], s["slots"])
    s["cache"].read(s["slots"], s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"]}


def _own_attend(s):
    s["cache"].attend(s["q"], s["out"], s["cu_q"], s["seq_len"], s["table"], s["max_q"], s["max_seq"],
                      window=s["window"], sinks=s["sinks"], lse=s["lse"])
    return {"out": s["out"]} if s["lse"] is None else {"out": s["out"], "lse": s["lse"]}


def _own_norm(s):
    from dracomancer_llmengine_b200 import decoder
    decoder.rmsnorm_q8(s["x"], s["w"], s["eps"], s["q"], s["scales"], residual=s["r"], h=s["h"], y=s["y"],
                       group=s["group"])
    return _norm_outputs(s["h"], s["y"], s["q"], s["scales"])


def _norm_outputs(h, y, q, scales):
    o = {"q": q, "scales": scales}
    if h is not None:
        o["h"] = h
    if y is not None:
        o["y"] = y
    return o


def _plain_blocks(s):
    ctx, new, table, page, n_free = s["ctx"], s["new"], s["table"], s["page"], s["n_free"]
    held = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page - held
    pre = torch.cumsum(need, 0)
    ok = (need == 0) | (pre <= n_free)
    j = torch.arange(table.shape[1], device=DEV) - held[:, None]
    gets = ok[:, None] & (j >= 0) & (j < need[:, None])
    at = (n_free - 1 - (pre - need)[:, None] - j).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(gets, s["free"][at], table))
    cu = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0)).int()
    tok = torch.arange(s["cap"], device=DEV)
    req = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    real = req < ctx.numel()
    req = req.clamp(max=ctx.numel() - 1)
    pos = torch.where(real, ctx[req] + tok - cu[req], -1).int()
    entry = table[req, (pos // page).clamp(0, table.shape[1] - 1).long()]
    slots = torch.where(real & ok[req], entry * page + pos % page, -1).int()
    return {"table": table, "slots": slots, "positions": pos, "cu": cu, "seq": torch.where(ok, ctx + new, ctx),
            "n_free": (n_free - (need * ok).sum()).int(), "refused": (~ok).sum().int().reshape(1)}


def _plain_append(s):
    d, page, slots = s["d"], s["page"], s["slots"].long()
    kc, ks, km, vc, vs, vm = _parts(s["pages"], d)
    at, tile, pair, odd = slots // page, slots % page // TILE, slots % TILE // 2, slots % 2
    c, sc, m = _codes(s["k"], 0)
    kc[at, :, tile, pair, odd] = _k_bytes(c)
    ks[at, :, tile, pair, :, odd] = sc
    km[at, :, tile, pair, odd] = m
    c, sc, m = _codes(s["v"], 8)
    vc[at, :, tile, pair, :, :, odd] = _v_bytes(c)
    vs[at, :, tile, pair, :, odd] = sc
    vm[at, :, tile, pair, :, odd] = m
    k, v = _decode(s["pages"], d)                     # [pages, heads, tiles, 16, D]
    tok = slots % TILE
    return {"k": k[at, :, tile, tok].to(s["k"].dtype), "v": v[at, :, tile, tok].to(s["v"].dtype)}


def _plain_attend(s):
    q, d, seq, cu, page = s["q"], s["d"], s["seq_len"].long(), s["cu_q"].long(), s["page"]
    n, heads = q.shape[:2]
    reqs, hkv = seq.numel(), s["pages"].shape[1]
    rows = s["max_q"]
    # the cache, one row of keys and values for each request
    k, v = _decode(s["pages"][s["table"].long().clamp(min=0)], d)     # [requests, width, heads, tiles, 16, D]
    k = k.transpose(1, 2).reshape(reqs, hkv, -1, d)
    v = v.transpose(1, 2).reshape(reqs, hkv, -1, d)
    i = torch.arange(rows, device=DEV)
    qlen = cu[1:] - cu[:-1]
    qp = q[(cu[:-1, None] + i).clamp(max=n - 1)].float()              # [requests, rows, heads, D]
    qp = qp.unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4).reshape(reqs, hkv, -1, d)
    score = (qp @ k.transpose(-1, -2)) * (d ** -0.5)
    score = score.unflatten(2, (-1, rows))                            # [requests, kv heads, group, rows, keys]
    pos = (seq - qlen)[:, None, None] + i[:, None]
    key = torch.arange(k.shape[2], device=DEV)
    sees = (key <= pos) & (key < seq[:, None, None])
    if s["window"]:
        sees = sees & ((pos - key < s["window"]) | (key < s["sinks"]))
    sees = sees[:, None, None]
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < seq[:, None])[:, None, :, None], v, 0.0)
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, rows)) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    tok = torch.arange(n, device=DEV)
    req = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    at = tok - cu[req]
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[req, at].to(q.dtype)
    return {"out": out} if s["lse"] is None else {"out": out, "lse": lse.permute(0, 3, 1, 2).flatten(2)[req, at]}


def _plain_norm(s):
    x, w = s["x"], s["w"]
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(x.dtype)
    f = h.float()
    rstd = torch.rsqrt((f * f).mean(-1, keepdim=True) + s["eps"])
    y = (f * rstd * w).to(x.dtype) if s["y"] is not None else None
    u = (f * w).unflatten(-1, (-1, s["group"] or f.shape[-1]))
    top = u.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, 127.0 if s["q"].dtype == torch.int8 else 448.0)
    tiny = top < 2.0 ** -100
    code = u * torch.where(tiny, 0.0, most / torch.where(tiny, 1.0, top))
    code = (code.round() if s["q"].dtype == torch.int8 else code).to(s["q"].dtype).flatten(-2)
    scales = torch.where(tiny, 0.0, top / most * rstd[..., None]).squeeze(-1)
    return _norm_outputs(None if s["r"] is None else h, y, code, scales)


# ---------------------------------------------------------------- what a pass cannot do without
def _seen(new, ctx, window, sinks):
    """(keys that some query of the request sees, pairs of a query and a key that it sees)."""
    pairs, low = 0, ctx
    for i in range(new):
        p = ctx - new + i
        if p < 0:
            continue
        first = max(0, p - window + 1) if window else 0
        low = min(low, first)
        pairs += p + 1 - first + min(sinks, first)
    return (ctx - low + min(sinks, low) if ctx else 0), pairs


def work(c):
    if c["op"] == "blocks":
        new, ctx = _block_lens(c)
        pages = sum(_ceil(v + n, c["page"]) - _ceil(v, c["page"]) for v, n in zip(ctx, new))
        return {"bytes": 16 * c["requests"] + 8 * pages + 8 * (sum(new) + 7), "flops": 0}
    if c["op"] == "append":   # written once, read once
        values = c["tokens"] * c["kv_heads"] * c["dim"]
        return {"bytes": values * (4 * SIZE[c["type"]] + 2 * 1.25) + 8 * c["tokens"], "flops": 8 * values}
    if c["op"] == "norm":
        values = c["tokens"] * c["hidden"]
        per = SIZE[c["type"]] * (1 + 2 * c["residual"] + c["y"]) + 1
        scales = c["tokens"] * (c["hidden"] // c["group"] if c["group"] else 1)
        return {"bytes": values * per + 4 * scales + 4 * c["hidden"], "flops": 8 * values}
    seen = [_seen(n, v, c["window"], c["sinks"]) for n, v in zip(*_attn_lens(c))]
    rows = sum(_attn_lens(c)[0]) * c["heads"]
    keys, pairs = sum(v[0] for v in seen), sum(v[1] for v in seen)
    return {"bytes": 1.25 * keys * c["kv_heads"] * c["dim"] + rows * (2 * SIZE[c["type"]] * c["dim"] + 4 * c["lse"]),
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"blocks": lambda s: None, "append": _exact_append, "attend": _exact_attend, "norm": _exact_norm}[case["op"]](s)


def _exact_append(s):
    """Each value from its own group's range: nothing goes through the cache's bytes."""
    def back(x, middle):
        x = x.double().unflatten(-1, (-1, GROUP))
        lo = x.min(-1, keepdim=True).values
        step = ((x.max(-1, keepdim=True).values - lo) / 15).half().double()
        base = (lo + middle * step).half().double()
        code = torch.clamp(torch.round((x - base) / torch.where(step > 0, step, 1.0)) + middle, 0, 15)
        return (step * (code - middle) + base).flatten(-2)
    return {"k": back(s["k"], 0), "v": back(s["v"], 8)}


def _exact_attend(s):
    """Request by request and key/value head by head, in 64 bits."""
    if s["table"].numel() * s["page"] * s["max_q"] > 2 ** 27:
        return None
    d, page = s["d"], s["page"]
    heads, hkv = s["q"].shape[1], s["pages"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    cu, seq = s["cu_q"].tolist(), s["seq_len"].tolist()
    for r, length in enumerate(seq):
        rows = cu[r + 1] - cu[r]
        if not length or not rows:
            continue
        pages = s["pages"][s["table"][r, :_ceil(length, page)].long()]
        per = heads // hkv
        pos = torch.arange(length - rows, length, device=DEV)[:, None]
        key = torch.arange(length, device=DEV)[None]
        hidden = key > pos
        if s["window"]:
            hidden |= (key <= pos - s["window"]) & (key >= s["sinks"])
        for h in range(hkv):
            k, v = _decode(pages[:, h], d, torch.float64)
            k, v = k.reshape(-1, d)[:length], v.reshape(-1, d)[:length]
            q = s["q"][cu[r]:cu[r + 1], h * per:(h + 1) * per].double()
            a = torch.einsum("rgd,kd->grk", q, k) / math.sqrt(d)
            a = a.masked_fill(hidden, -math.inf)
            z = torch.logsumexp(a, -1)
            w = torch.exp(a - torch.where(torch.isinf(z), 0.0, z)[..., None])
            out[cu[r]:cu[r + 1], h * per:(h + 1) * per] = torch.einsum("grk,kd->rgd", w, v)
            lse[cu[r]:cu[r + 1], h * per:(h + 1) * per] = z.T
    return {"out": out} if s["lse"] is None else {"out": out, "lse": lse}


def _exact_norm(s):
    x = s["x"].double()
    total = x if s["r"] is None else x + s["r"].double()
    h = total.to(s["x"].dtype).double()        # the norm is that of the stored sum
    rms = torch.sqrt(h.pow(2).sum(-1, keepdim=True) / h.shape[-1] + s["eps"])
    u = h * s["w"].double()
    whole = s["q"].dtype == torch.int8
    most = 127.0 if whole else 448.0
    top = u.unflatten(-1, (-1, s["group"] or u.shape[-1])).abs().max(-1).values
    code = u.unflatten(-1, (top.shape[-1], -1)) / top[..., None] * most
    return _norm_outputs(None if s["r"] is None else total, None if s["y"] is None else u / rms,
                         None if whole else code.flatten(-2), top / most / rms)
