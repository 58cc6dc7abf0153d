"""Cases of the 8-bit products: projections and expert products of e4m3 rows and weights with block scales, gate/up
products with SwiGLU and 8-bit output, the plan that sorts a batch by expert, and the weighted sum of the experts' rows.
`run` computes them with elementary torch operations, or, where `own` is true, through
`dracomancer_llmengine_b200.decoder`."""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 128    # values of a row, rows of a weight, that share a scale
TINY = 2.0 ** -100


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the query/key/value projection of one decoded token: latency
        linear_case("linear one", 1, 2048, 5120, "bf16"),
        # a ragged chunk into a head of an odd width, the inner size not a whole number of blocks
        linear_case("linear odd", 1003, 2064, 1001, "f32"),
        # a prefill chunk of the widest configuration
        linear_case("linear prefill", 8192, 7168, 7168, "bf16"),
        # the down products of a decode batch: one or two rows an expert, every weight read once
        experts_case("experts decode", 64, 8, 384, 2048, 7168, "bf16"),
        # the down products of a prefill chunk whose routing is skewed: experts with thousands of rows and with none
        experts_case("experts skewed", 8192, 8, 384, 2048, 7168, "bf16", skew=1.2),
        # the shared expert's gate and up products of one decoded token
        swiglu_case("swiglu one", 1, 0, 0, 7168, 2048),
        # the routed experts' gate and up products of a decode batch
        swiglu_case("swiglu decode", 64, 8, 384, 7168, 2048),
        # a prefill chunk over small experts
        swiglu_case("swiglu prefill", 4096, 8, 256, 2048, 512),
        # a decode batch sorted by expert
        plan_case("plan decode", 64, 8, 384),
        # a prefill chunk, of which this GPU has an eighth of the experts
        plan_case("plan slice", 8192, 8, 384, first=48, count=48, skew=1.2),
        # the experts' rows of one decoded token
        combine_case("combine one", 1, 8, 2048, "f32", add=True),
        # a prefill chunk with the shared expert's rows
        combine_case("combine prefill", 4096, 8, 7168, "bf16", add=True),
    ]


def linear_case(name, tokens, k, n, kind):
    return {"name": name, "op": "linear", "tokens": tokens, "k": k, "n": n, "type": kind}


def experts_case(name, tokens, used, experts, k, n, kind, skew=0.0, gather=False):
    return {"name": name, "op": "experts", "tokens": tokens, "used": used, "experts": experts, "k": k, "n": n,
            "type": kind, "skew": skew, "gather": gather}


def swiglu_case(name, tokens, used, experts, k, inter, skew=0.0):
    return {"name": name, "op": "swiglu", "tokens": tokens, "used": used, "experts": experts, "k": k, "inter": inter,
            "skew": skew}


def plan_case(name, tokens, used, experts, first=0, count=None, skew=0.0):
    return {"name": name, "op": "plan", "tokens": tokens, "used": used, "experts": experts, "first": first,
            "count": experts if count is None else count, "skew": skew}


def combine_case(name, tokens, used, hidden, kind, add=False, skipped=False):
    return {"name": name, "op": "combine", "tokens": tokens, "used": used, "hidden": hidden, "type": kind, "add": add,
            "skipped": skipped}


def _log(rng, lo, hi):
    """An odd number, or now and then an even one, spread over the logarithm of [lo, hi]."""
    v = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v if rng.random() < 0.4 else max(lo, min(hi, v | 1))


def draw(rng):
    op = rng.choice(["linear", "linear", "experts", "experts", "swiglu", "swiglu", "plan", "combine"])
    kind, skew = rng.choice(["f32", "f16", "bf16"]), rng.choice([0.0, 0.0, 1.2])
    if op == "linear":
        c = linear_case("", _log(rng, 1, 8192), rng.choice([512, 768, 1024, 2048, 2064, 4096, 7168]),
                        rng.choice([512, 1001, 2048, 2049, 4096, 7168]), kind)
    elif op == "experts":
        e, k, n = rng.choice([(32, 512, 2048), (128, 768, 2048), (256, 512, 2048), (384, 2048, 7168), (64, 1408, 2048),
                              (16, 1040, 1001)])
        gather = rng.random() < 0.3
        c = experts_case("", _log(rng, 1, 8191 if e < 384 or not gather else 4095), rng.choice([1, 2, 4, 8]), e, k, n,
                         kind if e < 384 else "bf16", skew, gather)
    elif op == "swiglu":
        e, k, f = rng.choice([(0, 7168, 2048), (0, 2048, 768), (32, 2048, 512), (128, 2048, 768), (256, 2048, 512),
                              (384, 7168, 2048), (64, 2048, 1408), (8, 1040, 200)])
        c = swiglu_case("", _log(rng, 1, 4095 if e < 384 else 2047), rng.choice([1, 2, 4, 8]) if e else 0, e, k, f,
                        skew if e else 0.0)
    elif op == "plan":
        e = rng.choice([16, 32, 128, 256, 384, 1000])
        count = rng.choice([e, e, e // 2, e // 8])
        c = plan_case("", _log(rng, 1, 8192), rng.choice([1, 2, 4, 8]), e, rng.randrange(0, e - count + 1), count, skew)
    else:
        c = combine_case("", _log(rng, 1, 4095), rng.choice([1, 2, 4, 8]), rng.choice([1001, 2048, 4096, 7168]), kind,
                         rng.random() < 0.5, rng.random() < 0.4)
        if kind == "f32":
            c["tokens"] = min(c["tokens"], 2047)
    del c["name"]
    return c


@functools.lru_cache(maxsize=64)
def _order(tokens, used, experts, skew):
    """Experts of each token, distinct, [tokens, used]: as a top-k router picks them, of equal or of Zipf popularity.  The
    same for every seed, so that a case's work is fixed; a seed permutes the tokens and renames the experts."""
    r = np.random.default_rng(20)
    score = r.gumbel(size=(tokens, experts)).astype(np.float32) - np.float32(skew) * np.log(np.arange(1, experts + 1, dtype=np.float32))
    return np.argsort(-score, axis=1, kind="stable")[:, :used].astype(np.int32)


def _counts(c):
    return np.bincount(_order(c["tokens"], c["used"], c["experts"], c["skew"]).ravel(), minlength=c["experts"])


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _rows(tokens, k, gen):
    """Rows of hidden states in e4m3 with a scale for each block of 128, as the norm writes them."""
    codes = torch.empty(tokens, k, dtype=torch.float8_e4m3fn, device=DEV)
    scales = torch.empty(tokens, _ceil(k, BLOCK), device=DEV)
    width = torch.exp(0.7 * _randn(gen, k))
    for b in range(scales.shape[1]):
        at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        x = _randn(gen, tokens, at.stop - at.start) * width[at]
        scales[:, b] = x.abs().amax(1) / 448
        codes[:, at] = (x / scales[:, b:b + 1]).to(codes.dtype)
    return codes, scales


def _weights(lead, n, k, gen):
    """Weights [*lead, n, k] in e4m3 with a scale for each block of 128 x 128: the largest of 16384 normal values is about
    four standard deviations, and takes the code 448."""
    codes = torch.empty(math.prod(lead), n, k, dtype=torch.float8_e4m3fn, device=DEV)
    step = max(1, (1 << 28) // (n * k))
    for a in range(0, codes.shape[0], step):
        part = codes[a:a + step]
        part.copy_(torch.empty(part.shape, dtype=torch.bfloat16, device=DEV).normal_(0, 112, generator=gen).clamp_(-448, 448))
    scales = 0.02 * torch.exp(0.3 * _randn(gen, *lead, _ceil(n, BLOCK), _ceil(k, BLOCK))) / 112
    return codes.view(*lead, n, k), scales


def _routing(c, gen):
    """This seed's routing: (order [tokens, used] on the GPU, rows of each expert on the host)."""
    shift = int(torch.randint(c["experts"], (1,), device=DEV, generator=gen))
    order = torch.from_numpy(_order(c["tokens"], c["used"], c["experts"], c["skew"])).to(DEV)
    order = (order[torch.randperm(c["tokens"], device=DEV, generator=gen)] + shift) % c["experts"]
    return order.int().contiguous(), np.roll(_counts(c), shift).tolist()


def _sorted(s, order, counts):
    """What the plan gives: offsets of the experts' rows, and the token of each."""
    s["counts"] = counts
    s["offsets"] = torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device=DEV)
    s["rows"] = (torch.argsort(order.flatten(), stable=True) // order.shape[1]).int()


def prepare(case, seed):
    return {"linear": _prepare_linear, "experts": _prepare_experts, "swiglu": _prepare_swiglu, "plan": _prepare_plan,
            "combine": _prepare_combine}[case["op"]](case, _gen(seed))


def _prepare_linear(c, gen):
    s = {"op": "linear", "out": torch.empty(c["tokens"], c["n"], dtype=TYPES[c["type"]], device=DEV)}
    s["x"], s["xs"] = _rows(c["tokens"], c["k"], gen)
    s["w"], s["ws"] = _weights((), c["n"], c["k"], gen)
    return s


def _prepare_experts(c, gen):
    rows = c["tokens"] * c["used"]
    s = {"op": "experts", "out": torch.empty(rows, c["n"], dtype=TYPES[c["type"]], device=DEV)}
    _sorted(s, *_routing(c, gen))
    if not c["gather"]:
        s["rows"] = None      # the rows are in the experts' order already
    s["x"], s["xs"] = _rows(c["tokens"] if c["gather"] else rows, c["k"], gen)
    s["w"], s["ws"] = _weights((c["experts"],), c["n"], c["k"], gen)
    return s


def _prepare_swiglu(c, gen):
    rows, f = c["tokens"] * max(1, c["used"]), c["inter"]
    s = {"op": "swiglu", "codes": torch.empty(rows, f, dtype=torch.float8_e4m3fn, device=DEV),
         "scales": torch.empty(rows, _ceil(f, BLOCK), device=DEV), "offsets": None, "rows": None}
    if c["experts"]:
        _sorted(s, *_routing(c, gen))
    s["x"], s["xs"] = _rows(c["tokens"], c["k"], gen)
    s["w"], s["ws"] = _weights((c["experts"], 2) if c["experts"] else (2,), f, c["k"], gen)
    return s


def _prepare_plan(c, gen):
    order, _ = _routing(c, gen)
    s = {"op": "plan", "order": order, "first": c["first"], "count": c["count"],
         "tail": torch.zeros(order.numel(), dtype=torch.int32, device=DEV)}
    if own:
        from dracomancer_llmengine_b200 import decoder
        s["plan"] = decoder.ExpertPlan(c["tokens"], c["used"], c["count"], DEV)
    return s


def _prepare_combine(c, gen):
    t, k, kind = c["tokens"], c["used"], TYPES[c["type"]]
    pos = torch.randperm(t * k, device=DEV, generator=gen).int().view(t, k)
    if c["skipped"]:        # experts of other GPUs
        pos = torch.where(torch.rand(t, k, device=DEV, generator=gen) < 0.5, pos, -1)
    weights = torch.rand(t, k, device=DEV, generator=gen) + 0.1
    return {"op": "combine", "y": _randn(gen, t * k, c["hidden"]).to(kind), "pos": pos,
            "weights": weights / weights.sum(1, keepdim=True),
            "add": _randn(gen, t, c["hidden"]).to(kind) if c["add"] else None,
            "out": torch.empty(t, c["hidden"], dtype=kind, device=DEV)}


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        return {"linear": _own_product, "experts": _own_product, "swiglu": _own_swiglu, "plan": _own_plan,
                "combine": _own_combine}[s["op"]](s)
    return {"linear": _plain_linear, "experts": _plain_experts, "swiglu": _plain_swiglu, "plan": _plain_plan,
            "combine": _plain_combine}[s["op"]](s)


def _own_product(s):
    from dracomancer_llmengine_b200 import decoder
    decoder.linear_q8(s["x"], s["xs"], s["w"], s["ws"], s["out"], offsets=s.get("offsets"), rows=s.get("rows"))
    return {"out": s["out"]}


def _own_swiglu(s):
    from dracomancer_llmengine_b200 import decoder
    decoder.swiglu_q8(s["x"], s["xs"], s["w"], s["ws"], s["codes"], s["scales"], offsets=s["offsets"], rows=s["rows"])
    return {"codes": s["codes"], "scales": s["scales"]}


def _own_plan(s):
    from dracomancer_llmengine_b200 import decoder
    p = s["plan"]
    decoder.plan_experts(s["order"], p, first=s["first"])
    return {"offsets": p.offsets, "rows": p.rows, "pos": p.pos}


def _own_combine(s):
    from dracomancer_llmengine_b200 import decoder
    decoder.combine_experts(s["y"], s["pos"], s["weights"], s["out"], add=s["add"])
    return {"out": s["out"]}


def _values(codes, scales, rows=1):
    """Codes [n, k] as fp32, times the scale of each block of `rows` x 128."""
    col = torch.arange(codes.shape[1], device=DEV) // BLOCK
    scales = scales[:, col]
    if rows > 1:
        scales = scales[torch.arange(codes.shape[0], device=DEV) // rows]
    return codes.float() * scales


def _plain_linear(s):
    return {"out": (_values(s["x"], s["xs"]) @ _values(s["w"], s["ws"], BLOCK).T).to(s["out"].dtype)}


def _plain_experts(s):
    x, out, at = _values(s["x"], s["xs"]), s["out"], 0
    if s["rows"] is not None:
        x = x[s["rows"]]
    for e, n in enumerate(s["counts"]):     # each expert has another number of rows
        if n:
            out[at:at + n] = x[at:at + n] @ _values(s["w"][e], s["ws"][e], BLOCK).T
            at += n
    return {"out": out}


def _silu_mul(x, w, ws):
    gate, up = (x @ _values(w[i], ws[i], BLOCK).T for i in (0, 1))
    return gate / (1 + torch.exp(-gate)) * up


def _plain_swiglu(s):
    x = _values(s["x"], s["xs"])
    if s["offsets"] is None:
        u = _silu_mul(x, s["w"], s["ws"])
    else:
        x, parts, at = x[s["rows"]], [], 0
        for e, n in enumerate(s["counts"]):
            if n:
                parts.append(_silu_mul(x[at:at + n], s["w"][e], s["ws"][e]))
                at += n
        u = torch.cat(parts)
    f, groups = u.shape[1], s["scales"].shape[1]
    u = torch.nn.functional.pad(u, (0, groups * BLOCK - f)).unflatten(1, (groups, BLOCK))
    top = u.abs().amax(2)
    inv = torch.where(top < TINY, 0.0, 448 / top.clamp(min=TINY))
    codes = (u * inv[..., None]).flatten(1)[:, :f].to(torch.float8_e4m3fn)
    return {"codes": codes, "scales": torch.where(top < TINY, 0.0, top / 448)}


def _plain_plan(s):
    order, count = s["order"], s["count"]
    local = order.flatten() - s["first"]
    local = torch.where((local >= 0) & (local < count), local, count).long()
    per = torch.zeros(count + 1, dtype=torch.int64, device=DEV).scatter_add_(0, local, torch.ones_like(local))
    offsets = torch.nn.functional.pad(torch.cumsum(per[:-1], 0), (1, 0)).int()
    by_expert = torch.argsort(local, stable=True)
    at = torch.arange(local.numel(), device=DEV)
    rows = torch.where(at < offsets[-1], by_expert // order.shape[1], s["tail"]).int()
    pos = torch.empty_like(local)
    pos[by_expert] = at
    return {"offsets": offsets, "rows": rows, "pos": torch.where(local < count, pos, -1).int().view(order.shape)}


def _plain_combine(s):
    there = s["pos"] >= 0
    y = s["y"][s["pos"].clamp(min=0)].float() * torch.where(there, s["weights"], 0.0)[..., None]
    out = y.sum(1)
    if s["add"] is not None:
        out = out + s["add"].float()
    return {"out": out.to(s["out"].dtype)}


# ---------------------------------------------------------------- what a pass cannot do without
def work(c):
    op, t = c["op"], c["tokens"]
    if op == "plan":
        kept = int(_counts(c)[c["first"]:c["first"] + c["count"]].sum())
        return {"bytes": 8 * t * c["used"] + 4 * kept + 4 * (c["count"] + 1), "flops": 0}
    if op == "combine":
        rows = t * c["used"] * (0.5 if c["skipped"] else 1)
        return {"bytes": SIZE[c["type"]] * c["hidden"] * (rows + t * (1 + c["add"])) + 8 * t * c["used"],
                "flops": 2 * rows * c["hidden"]}
    rows = t * max(1, c.get("used", 1))
    weights = int((_counts(c) > 0).sum()) if c.get("experts") else 1
    k, blocks = c["k"], _ceil(c["k"], BLOCK)
    if op == "swiglu":
        n, out, x_rows = 2 * c["inter"], rows * (c["inter"] + 4 * _ceil(c["inter"], BLOCK)), t
        w_blocks = 2 * _ceil(c["inter"], BLOCK) * blocks
    else:
        n, out, x_rows = c["n"], rows * c["n"] * SIZE[c["type"]], t if c.get("gather") else rows
        w_blocks = _ceil(n, BLOCK) * blocks
    index = (4 * rows if op == "swiglu" and c["experts"] or c.get("gather") else 0) + 4 * (c.get("experts", 0) + 1)
    return {"bytes": x_rows * (k + 4 * blocks) + weights * (n * k + 4 * w_blocks) + out + index, "flops": 2 * rows * n * k}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "experts": _exact_experts, "swiglu": _exact_swiglu, "plan": lambda s: None,
            "combine": _exact_combine}[case["op"]](s)


def _exact_product(x, xs, w, ws):
    """Block by block of the inner size: the codes' product times the two scales."""
    total = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    of = torch.arange(w.shape[0], device=DEV).div(BLOCK, rounding_mode="floor")
    for b in range(xs.shape[1]):
        part = slice(b * BLOCK, (b + 1) * BLOCK)
        total += torch.einsum("mk,nk->mn", x[:, part].double() * xs[:, b, None].double(),
                              w[:, part].double() * ws[of, b, None].double())
    return total


def _exact_linear(s):
    return {"out": _exact_product(s["x"], s["xs"], s["w"], s["ws"])}


def _groups(s):
    """(expert, its places, its rows of x) for the experts that have rows."""
    ends = s["offsets"].tolist()
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if b > a:
            yield e, slice(a, b), slice(a, b) if s["rows"] is None else s["rows"][a:b].long()


def _take(x, at):
    """Rows of 8-bit values, which index as bytes."""
    return x.view(torch.uint8)[at].view(x.dtype)


def _exact_experts(s):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for e, place, at in _groups(s):
        out[place] = _exact_product(_take(s["x"], at), s["xs"][at], s["w"][e], s["ws"][e])
    return {"out": out}


def _exact_swiglu(s):
    u = torch.zeros(s["codes"].shape, dtype=torch.float64, device=DEV)
    if s["offsets"] is None:
        todo = [(slice(None), slice(None), s["w"], s["ws"])]
    else:
        todo = [(place, at, s["w"][e], s["ws"][e]) for e, place, at in _groups(s)]
    for place, at, w, ws in todo:
        gate, up = (_exact_product(_take(s["x"], at), s["xs"][at], w[i], ws[i]) for i in (0, 1))
        u[place] = gate * torch.sigmoid(gate) * up
    codes, scales = torch.empty_like(u), torch.empty(s["scales"].shape, dtype=torch.float64, device=DEV)
    for g in range(scales.shape[1]):
        part = slice(g * BLOCK, (g + 1) * BLOCK)
        scales[:, g] = u[:, part].abs().max(1).values / 448
        codes[:, part] = u[:, part] / scales[:, g, None]
    return {"codes": codes, "scales": scales}


def _exact_combine(s):
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for k in range(s["pos"].shape[1]):
        at = s["pos"][:, k]
        some = (at >= 0).nonzero()[:, 0]
        out[some] += s["y"][at[some].long()].double() * s["weights"][some, k, None].double()
    return {"out": out if s["add"] is None else out + s["add"].double()}
