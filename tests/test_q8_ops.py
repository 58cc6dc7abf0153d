"""The 8-bit products with block scales, the plan by expert and the weighted sum of the experts' rows, against plain
computations in 64 bits.

Tolerances.  Products of two e4m3 codes are exact in fp32.  A block's 128 of them are added in fp32 in an unknown order, by
adders that may cut instead of round (2^-23 of the running sum at most); its two scales are multiplied (one rounding) and the
blocks are added by fused multiply-adds.  With S the sum of the magnitudes of all terms the error is below
(128 + blocks + 4) * 2^-23 * S, and the output's own rounding adds half a step."""
import pytest
import torch

import dracomancer_llmengine_b200 as dm
from dracomancer_llmengine_b200 import decoder

pytestmark = pytest.mark.gpu
E4M3, TYPES = torch.float8_e4m3fn, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
DEV = "cuda"


@pytest.fixture(autouse=True)
def _gpu(dlib):
    yield
    dlib.draco_b200_test_q8_form(0)


# the forms that a call can take: chosen by sizes, for few rows, for any address, on the tensor cores by columns a tile
FORMS = [0, 1, 2, 32, 64, 128, 256]
# 1024 times the blocks of threads that share a tile's inner size
SPLITS = [2048 + 32, 4096 + 64, 8192 + 64, 2048 + 128, 8192 + 128, 4096 + 256, 8192 + 256]


def gen_of(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def codes_of(shape, gen):
    return (60 * torch.randn(shape, device=DEV, generator=gen)).clamp(-448, 448).to(E4M3)


def scales_of(shape, gen):
    return torch.exp(torch.randn(shape, device=DEV, generator=gen)) / 64


def cdiv(a, b):
    return -(-a // b)


def operands(rows, k, n, gen, lead=()):
    x, xs = codes_of((rows, k), gen), scales_of((rows, cdiv(k, 128)), gen)
    return x, xs, codes_of((*lead, n, k), gen), scales_of((*lead, cdiv(n, 128), cdiv(k, 128)), gen)


def wide(codes, scales, rows=1):
    """Values in 64 bits of codes [n, k] with a scale for each `rows` x 128."""
    s = scales.double().repeat_interleave(rows, 0)[:codes.shape[0]].repeat_interleave(128, 1)[:, :codes.shape[1]]
    return codes.double() * s


def plain(x, xs, w, ws):
    """(product, bound of the kernel's error before the output's rounding)"""
    a, b = wide(x, xs), wide(w, ws, 128)
    return a @ b.T, (a.abs() @ b.abs().T) * (128 + xs.shape[1] + 4) * 2.0 ** -23


def same(got, want, bound, kind):
    err = (got.double() - want).abs()
    tiny = 2.0 ** -25 if kind == "f16" else 0.0       # half a step of fp16's subnormals
    assert got.dtype is TYPES[kind] and bool((err <= bound + (want.abs() + bound) * HALF_STEP[kind] + tiny).all()), float(err.max())


SHAPES = [(1, 128, 16), (1, 2048, 130), (1, 7168, 2048), (3, 16, 1), (2, 1, 1), (5, 40, 33), (17, 272, 257), (32, 4096, 640),
          (48, 7168, 1040), (33, 512, 100), (64, 2048, 2048), (128, 1024, 128), (129, 144, 255), (257, 2064, 513), (1000, 384, 1536), (700, 7168, 384)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear(rows, k, n, kind):
    x, xs, w, ws = operands(rows, k, n, gen_of(rows + k + n))
    out = torch.full((rows, n), float("nan"), dtype=TYPES[kind], device=DEV)
    assert decoder.linear_q8(x, xs, w, ws, out) is out
    want, bound = plain(x, xs, w, ws)
    if kind == "f16":       # within its range
        top = float(want.abs().max()) / 1000
        xs /= top
        decoder.linear_q8(x, xs, w, ws, out)
        want, bound = plain(x, xs, w, ws)
    same(out, want, bound, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("form", FORMS[1:] + SPLITS)
@pytest.mark.parametrize("rows,k,n", [(1, 128, 16), (9, 1040, 130), (33, 2064, 257), (130, 640, 1001), (500, 512, 768)])
def test_linear_forms(rows, k, n, form, kind, dlib):
    """Every form on sizes that it would not be chosen for."""
    x, xs, w, ws = operands(rows, k, n, gen_of(rows + k + n))
    dlib.draco_b200_test_q8_form(form)
    same(decoder.linear_q8(x, xs, w, ws, torch.full((rows, n), float("nan"), dtype=TYPES[kind], device=DEV)), *plain(x, xs, w, ws), kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("off", [16, 3])
def test_linear_strides(kind, off):
    """Parts of wider tensors: rows that start on 16 bytes, and rows that do not; what is around the output stays."""
    rows, k, n, gen = 70, 256, 200, gen_of(off)
    x, xs, w, ws = operands(rows, k, n, gen)
    wide_x = torch.zeros(rows, k + 2 * off, device=DEV).to(E4M3)
    wide_x[:, off:off + k] = x
    wide_s = torch.full((rows, 7), float("nan"), device=DEV)
    wide_s[:, 3:5] = xs
    wide_out = torch.full((rows + 1, n + 2 * off), 7.0, device=DEV).to(TYPES[kind])
    out = wide_out[:rows, off:off + n]
    xs *= 2.0 ** -8
    wide_s[:, 3:5] = xs
    decoder.linear_q8(wide_x[:, off:off + k], wide_s[:, 3:5], w, ws, out)
    same(out, *plain(x, xs, w, ws), kind)
    assert bool((wide_out[:, :off] == 7).all() and (wide_out[:, off + n:] == 7).all() and (wide_out[rows:] == 7).all())


def test_linear_one_row_for_all():
    """A row that is repeated by a stride of 0."""
    x, xs, w, ws = operands(1, 128, 64, gen_of(1))
    out = torch.empty(9, 64, device=DEV)
    decoder.linear_q8(x.expand(9, 128), xs.expand(9, 1), w, ws, out)
    same(out, *plain(x.expand(9, 128), xs.expand(9, 1), w, ws), "f32")


@pytest.mark.parametrize("form", FORMS + SPLITS)
@pytest.mark.parametrize("rows,k,n", [(1, 128, 64), (40, 256, 300), (200, 512, 256)])
def test_not_finite_stays_in_its_row(rows, k, n, form, dlib):
    """A NaN code or scale, or an infinite scale, reaches its own row, or its own column, alone."""
    gen = gen_of(rows)
    dlib.draco_b200_test_q8_form(form)
    x, xs, w, ws = operands(rows, k, n, gen)
    clean = decoder.linear_q8(x, xs, w, ws, torch.empty(rows, n, device=DEV)).clone()
    bad = rows // 2
    for change in ("code", "scale", "inf"):
        x2, xs2 = x.clone(), xs.clone()
        if change == "code":
            x2.view(torch.uint8)[bad, k - 1] = 127
        else:
            xs2[bad, 0] = float("nan") if change == "scale" else float("inf")
        got = decoder.linear_q8(x2, xs2, w, ws, torch.empty(rows, n, device=DEV))
        assert not got[bad].isfinite().any()
        keep = torch.arange(rows, device=DEV) != bad
        assert torch.equal(got[keep], clean[keep])
    w2 = w.clone()
    w2.view(torch.uint8)[n - 1, 0] = 255
    got = decoder.linear_q8(x, xs, w2, ws, torch.empty(rows, n, device=DEV))
    assert got[:, n - 1].isnan().all() and torch.equal(got[:, :n - 1], clean[:, :n - 1])


COUNTS = {"mixed": [5, 0, 1, 128, 129, 0, 300, 31, 32, 33, 0], "empty ends": [0, 0, 7, 0], "one": [64], "nothing": [0, 0, 0],
          "decode": [1, 2, 0, 1, 1, 3, 0, 0, 1, 1, 2, 1] * 4, "large": [700, 3, 1025, 0, 257],
          "few and some": [33, 0, 1, 0, 64, 2, 0, 17, 0, 0, 65], "tens": [20, 64, 0, 65, 33, 70, 31, 1, 16]}


def group_args(counts, k, n, gather, seed, lead=()):
    gen, total = gen_of(seed), sum(counts)
    n_x = max(1, total // 2) if gather else total
    x, xs, w, ws = operands(n_x, k, n, gen, (len(counts), *lead))
    offsets = torch.nn.functional.pad(torch.tensor(counts, device=DEV).cumsum(0), (1, 0)).int()
    rows = torch.randint(n_x, (total,), device=DEV, generator=gen).int() if gather else None
    return x, xs, w, ws, offsets, rows


def of_row(x, rows, a, b):
    at = torch.arange(a, b, device=DEV) if rows is None else rows[a:b].long()
    return x.view(torch.uint8)[at].view(E4M3) if x.dtype is E4M3 else x[at]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("k,n", [(512, 256), (272, 1001), (40, 33), (128, 2048)])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("form", FORMS)
def test_grouped(counts, k, n, gather, kind, form, dlib):
    dlib.draco_b200_test_q8_form(form)
    counts = COUNTS[counts]
    x, xs, w, ws, offsets, rows = group_args(counts, k, n, gather, k + n)
    total, behind = sum(counts), 3
    out = torch.full((total + behind, n), 5.0, dtype=TYPES[kind], device=DEV)
    if rows is None:        # rows behind the last group belong to no group
        x, xs = torch.cat([x.view(torch.uint8), x.new_zeros(behind, k).view(torch.uint8)]).view(E4M3), torch.cat([xs, xs.new_ones(behind, xs.shape[1])])
        decoder.linear_q8(x, xs, w, ws, out, offsets=offsets)
    else:
        decoder.linear_q8(x, xs, w, ws, out, offsets=offsets, rows=torch.cat([rows, ints(0, 0, 0)]))
    assert bool((out[total:] == 5).all())
    at = 0
    for e, c in enumerate(counts):
        if c:
            want, bound = plain(of_row(x, rows, at, at + c), of_row(xs, rows, at, at + c), w[e], ws[e])
            same(out[at:at + c], want, bound, kind)
            at += c


@pytest.mark.parametrize("k", [256, 40])
@pytest.mark.parametrize("form", FORMS + SPLITS)
def test_rows_outside_x_give_zeros(k, form, dlib):
    dlib.draco_b200_test_q8_form(form)
    x, xs, w, ws = operands(4, k, 130, gen_of(3))
    x.view(torch.uint8)[0, 0] = 127       # the row that a careless kernel would read instead
    rows = ints(1, -1, 4, 2, -2147483648, 2147483647, 3)
    out = decoder.linear_q8(x, xs, w, ws, torch.full((7, 130), 9.0, device=DEV), rows=rows)
    assert not out[[1, 2, 4, 5]].any()
    want, bound = plain(of_row(x, ints(1, 2, 3), 0, 3), xs[1:4], w, ws)
    same(out[[0, 3, 6]], want, bound, "f32")
    f = 130
    w2, ws2 = torch.stack([w.view(torch.uint8)] * 2).view(E4M3), torch.stack([ws] * 2)
    codes, scales = torch.full((7, f), 9.0, device=DEV).to(E4M3), torch.full((7, 2), 9.0, device=DEV)
    decoder.swiglu_q8(x, xs, w2, ws2, codes, scales, rows=rows)
    assert not codes.float()[[1, 2, 4, 5]].any() and not scales[[1, 2, 4, 5]].any() and scales[[0, 3, 6]].all()


def test_no_rows_of_x():
    _, _, w, ws = operands(1, 256, 64, gen_of(4))
    x, xs = torch.empty(0, 256, device=DEV).to(E4M3), torch.empty(0, 2, device=DEV)
    out = decoder.linear_q8(x, xs, w, ws, torch.full((3, 64), 9.0, device=DEV), rows=ints(0, 1, -1))
    assert not out.any()
    assert decoder.linear_q8(x, xs, w, ws, torch.empty(0, 64, device=DEV)).numel() == 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("values", [(0, 40, 20, 60), (-5, 10, 20, 30), (0, 1000, 10, 5000), (50, 40, 30, 20), (7, 7, 7, 7)])
def test_offsets_out_of_order_stay_inside(values, form, dlib):
    """Such rows mean nothing, but nothing outside the output is touched."""
    x, xs, w, ws = operands(64, 128, 64, gen_of(5), (3,))
    dlib.draco_b200_test_q8_form(form)
    buf = torch.full((66, 64), 3.0, device=DEV)
    decoder.linear_q8(x, xs, w, ws, buf[1:65], offsets=ints(*values))
    assert bool((buf[0] == 3).all() and (buf[65] == 3).all())


def test_many_groups():
    """As many groups as a call takes, most without rows."""
    counts = [0] * 1024
    counts[0], counts[511], counts[1023] = 3, 140, 1
    x, xs, w, ws, offsets, _ = group_args(counts, 128, 40, False, 6)
    out = decoder.linear_q8(x, xs, w, ws, torch.empty(144, 40, device=DEV), offsets=offsets)
    for e, a, b in ((0, 0, 3), (511, 3, 143), (1023, 143, 144)):
        same(out[a:b], *plain(of_row(x, None, a, b), xs[a:b], w[e], ws[e]), "f32")
    with pytest.raises(dm.DracoError, match="1024"):
        decoder.linear_q8(x, xs, torch.cat([w.view(torch.uint8)] * 2).view(E4M3), torch.cat([ws] * 2), out,
                          offsets=torch.zeros(2049, dtype=torch.int32, device=DEV))


def check_swiglu(codes, scales, x, xs, w, ws):
    """exp and the quotient are within 2^-21 together; |silu'| <= 1.1.  Codes: half a step (2^-4 of the value, 2^-10 below
    the normal range) beside what the value and the scale are off."""
    (g, eg), (u, eu) = plain(x, xs, w[0], ws[0]), plain(x, xs, w[1], ws[1])
    act = g * torch.sigmoid(g)
    h, f = act * u, g.shape[1]
    eh = 1.1 * eg * (u.abs() + eu) + act.abs() * eu + 2.0 ** -21 * h.abs()
    for b in range(scales.shape[1]):
        part = slice(128 * b, min(f, 128 * b + 128))
        a, off = h[:, part].abs().amax(1, keepdim=True), eh[:, part].amax(1, keepdim=True)
        assert bool(((scales[:, b:b + 1].double() - a / 448).abs() <= (off + a * 2.0 ** -23) / 448).all())
        v = h[:, part] / a * 448
        tol = v.abs() * 2.0 ** -4 + 2.0 ** -10 + 1.1 * 448 / a * (eh[:, part] + off * h[:, part].abs() / a + 2.0 ** -22 * h[:, part].abs())
        assert bool(((codes[:, part].double() - v).abs() <= tol).all())
        assert bool((codes[:, part].double().abs().amax(1) == 448).all())


@pytest.mark.parametrize("form", [0, 1, 64, 128, 256, 2048 + 256, 4096 + 256, 8192 + 256])
@pytest.mark.parametrize("rows,k,f", [(1, 7168, 2048), (1, 128, 128), (2, 256, 200), (7, 144, 16), (33, 512, 512), (3, 40, 33),
                                      (130, 2048, 768), (500, 1024, 129), (1000, 272, 640)])
def test_swiglu(rows, k, f, form, dlib):
    dlib.draco_b200_test_q8_form(form)
    x, xs, w, ws = operands(rows, k, f, gen_of(rows + f), (2,))
    ws /= 500 * k ** 0.5
    codes, scales = torch.zeros(rows, f, device=DEV).to(E4M3), torch.full((rows, cdiv(f, 128)), 9.0, device=DEV)
    assert decoder.swiglu_q8(x, xs, w, ws, codes, scales) == (codes, scales)
    check_swiglu(codes, scales, x, xs, w, ws)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("k,f", [(512, 256), (272, 200), (40, 33), (128, 1024)])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("form", [0, 1, 64, 128, 256])
def test_swiglu_grouped(counts, k, f, gather, form, dlib):
    dlib.draco_b200_test_q8_form(form)
    counts = COUNTS[counts]
    x, xs, w, ws, offsets, rows = group_args(counts, k, f, gather, k + f, (2,))
    ws /= 500 * k ** 0.5
    total = sum(counts)
    buf, sbuf = torch.full((total + 2, f + 16), 7.0, device=DEV).to(E4M3), torch.full((total + 2, cdiv(f, 128) + 1), 7.0, device=DEV)
    codes, scales = buf[:total, :f], sbuf[:total, :-1]
    decoder.swiglu_q8(x, xs, w, ws, codes, scales, offsets=offsets, rows=rows)
    at = 0
    for e, c in enumerate(counts):
        if c:
            check_swiglu(codes[at:at + c], scales[at:at + c], of_row(x, rows, at, at + c), of_row(xs, rows, at, at + c), w[e], ws[e])
            at += c
    assert bool((buf[total:].float() == 7).all() and (buf[:, f:].float() == 7).all() and (sbuf[total:] == 7).all() and (sbuf[:, -1] == 7).all())


@pytest.mark.parametrize("form", [0, 1, 2, 64, 128, 256])
def test_swiglu_extremes(form, dlib):
    """Gates of both signs beyond exp's range, products of nothing, of tiny and of infinite size."""
    dlib.draco_b200_test_q8_form(form)
    k, f = 128, 128
    x, w = torch.zeros(6, k, device=DEV), torch.zeros(2, f, k, device=DEV)
    x[:, 0], x[0, 0] = 1, 0
    w[:, :, 0] = 1
    w[0, 1, 0] = -1
    xs = torch.tensor([[1.0], [1000.0], [2.0 ** -60], [3e38], [float("nan")], [30.0]], device=DEV)
    codes, scales = torch.empty(6, f, device=DEV).to(E4M3), torch.empty(6, 1, device=DEV)
    decoder.swiglu_q8(x.to(E4M3), xs, w.to(E4M3), torch.ones(2, 1, 1, device=DEV), codes, scales)
    c = codes.float()
    assert not c[0].any() and float(scales[0]) == 0                         # nothing
    assert float(c[1, 0]) == 448 and float(c[1, 1]) == 0 and abs(float(scales[1]) / (1e6 / 448) - 1) < 1e-6
    assert not c[2].any() and float(scales[2]) == 0                         # 2^-121 is below 2^-100
    assert scales[3].isnan() and scales[4].isnan()
    assert abs(float(scales[5]) / (900 / 448) - 1) < 1e-6 and float(c[5, 1].abs()) < 2.0 ** -9


def reference_plan(order, first, count):
    flat = (order - first).flatten().tolist()
    places = sorted((e, i) for i, e in enumerate(flat) if 0 <= e < count)
    offsets = [sum(1 for e, _ in places if e < x) for x in range(count + 1)]
    pos = [-1] * len(flat)
    for at, (_, i) in enumerate(places):
        pos[i] = at
    return offsets, [i // order.shape[1] for _, i in places], pos


@pytest.mark.parametrize("tokens,used,experts,first,count", [
    (1, 1, 1, 0, 1), (1, 8, 384, 0, 384), (64, 8, 384, 48, 48), (33, 2, 7, 3, 4), (1000, 8, 1024, 0, 1024), (1024, 8, 64, 0, 64),
    (1025, 8, 64, 0, 64), (4000, 8, 256, 32, 32), (9000, 1, 3, 0, 3), (2731, 3, 40, -5, 50), (50, 4, 16, 20, 8)])
def test_plan(tokens, used, experts, first, count):
    gen = gen_of(tokens + first)
    order = torch.randint(-1, experts + 1, (tokens, used), device=DEV, generator=gen).int()
    order[::3] = order[0].clone()        # crowded experts
    plan = decoder.ExpertPlan(tokens + 3, used, count)
    for t in (plan.offsets, plan.rows, plan.pos):
        t.fill_(77)
    assert decoder.plan_experts(order, plan, first=first) is plan
    offsets, rows, pos = reference_plan(order, first, count)
    assert plan.offsets.tolist() == offsets
    assert plan.rows[:len(rows)].tolist() == rows and bool((plan.rows[len(rows):] == 77).all())
    assert plan.pos[:tokens].flatten().tolist() == pos and bool((plan.pos[tokens:] == 77).all())


@pytest.mark.parametrize("value", [0, 5, -1, 2147483647, -2147483648])
def test_plan_of_one_expert_or_none(value):
    order = torch.full((5000, 4), value, dtype=torch.int32, device=DEV)
    for first in (0, 2147483640, -2147483648):
        plan = decoder.plan_experts(order, decoder.ExpertPlan(5000, 4, 7), first=first)
        n, e = order.numel(), value - first
        if 0 <= e < 7:
            assert plan.offsets.tolist() == [0] * (e + 1) + [n] * (7 - e) and torch.equal(plan.pos.flatten(), torch.arange(n, device=DEV).int())
            assert torch.equal(plan.rows, torch.arange(n, device=DEV).int() // 4)
        else:
            assert not plan.offsets.any() and bool((plan.pos == -1).all()) and not plan.rows.any()


def test_plan_of_no_tokens():
    plan = decoder.ExpertPlan(4, 2, 5)
    plan.offsets.fill_(9)
    decoder.plan_experts(torch.empty(0, 2, dtype=torch.int32, device=DEV), plan)
    assert not plan.offsets.any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens,used,hidden,add", [(1, 8, 2048, True), (1, 1, 1, False), (5, 8, 1001, True), (64, 3, 40, False),
                                                    (300, 9, 7168, True), (7, 0, 64, True), (7, 0, 64, False)])
def test_combine(tokens, used, hidden, add, kind):
    """One fp32 rounding a term and the output's: (used + 1) * 2^-24 of the sum of magnitudes."""
    gen, n_y = gen_of(tokens + hidden), max(1, tokens * used // 2)
    y = torch.randn(n_y, hidden, device=DEV, generator=gen).to(TYPES[kind])
    pos = torch.randint(-2, n_y + 2, (tokens, used), device=DEV, generator=gen).int()
    weights = torch.randn(tokens, used, device=DEV, generator=gen)
    extra = torch.randn(tokens, hidden, device=DEV, generator=gen).to(TYPES[kind]) if add else None
    out = torch.full((tokens, hidden), 9.0, device=DEV).to(TYPES[kind])
    there = (pos >= 0) & (pos < n_y)
    terms = y.double()[pos.clamp(0, n_y - 1).long()] * torch.where(there, weights, 0.0).double()[..., None]
    want, size = terms.sum(1), terms.abs().sum(1)
    if add:
        want, size = want + extra.double(), size + extra.double().abs()
    assert decoder.combine_experts(y, pos, weights, out, add=extra) is out
    same(out, want, size * (used + 1) * 2.0 ** -24, kind)
    if add:     # in place
        decoder.combine_experts(y, pos, weights, extra, add=extra)
        assert torch.equal(extra, out)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("off", [8, 1])
def test_combine_strides(kind, off):
    gen, t, h = gen_of(off), 11, 256
    wide_y = torch.randn(30, h + 2 * off, device=DEV, generator=gen).to(TYPES[kind])
    wide_out = torch.full((t, h + 2 * off), 9.0, device=DEV).to(TYPES[kind])
    pos = torch.randint(30, (t, 5), device=DEV, generator=gen).int()[:, 1:4]
    weights = torch.randn(t, 6, device=DEV, generator=gen)[:, 2:5]
    y, out = wide_y[:, off:off + h], wide_out[:, off:off + h]
    decoder.combine_experts(y, pos, weights, out)
    terms = y.double()[pos.long()] * weights.double()[..., None]
    same(out, terms.sum(1), terms.abs().sum(1) * 4 * 2.0 ** -24, kind)
    assert bool((wide_out[:, :off] == 9).all() and (wide_out[:, off + h:] == 9).all())


def test_combine_places_not_finite():
    """What a place outside y would hold is not looked at; a weight of 0 on an infinity is NaN, as in any sum."""
    y = torch.full((2, 16), float("inf"), device=DEV)
    y[0] = 1
    out = decoder.combine_experts(y, ints(0, -1, 0, 1).view(2, 2), torch.tensor([[2.0, 0.0], [1.0, 0.0]], device=DEV), torch.empty(2, 16, device=DEV))
    assert bool((out[0] == 2).all() and out[1].isnan().all())


class Ffn:
    """Experts of e4m3 weights, and a pass through all the operators."""

    def __init__(self, hidden, inter, experts, used, tokens, seed=0, first=0, count=None):
        gen, count = gen_of(seed), experts if count is None else count
        self.used, self.first, self.eps = used, first, 1e-6
        self.norm = 1 + 0.1 * torch.randn(hidden, device=DEV, generator=gen)
        self.w13, self.w2 = codes_of((count, 2, inter, hidden), gen), codes_of((count, hidden, inter), gen)
        self.s13 = scales_of((count, 2, cdiv(inter, 128), cdiv(hidden, 128)), gen) / (hidden ** 0.5 / 4)
        self.s2 = scales_of((count, cdiv(hidden, 128), cdiv(inter, 128)), gen) / (inter ** 0.5 / 4)
        rows = tokens * used
        self.codes = torch.empty(tokens, hidden, device=DEV).to(E4M3)
        self.scales = torch.empty(tokens, hidden // 128, device=DEV)
        self.plan = decoder.ExpertPlan(tokens, used, count)
        self.act, self.act_scales = torch.zeros(rows, inter, device=DEV).to(E4M3), torch.zeros(rows, cdiv(inter, 128), device=DEV)
        self.down = torch.zeros(rows, hidden, device=DEV)
        self.out = torch.empty(tokens, hidden, device=DEV)

    def __call__(self, x, order, weights):
        decoder.rmsnorm_q8(x, self.norm, self.eps, self.codes, self.scales, group=128)
        decoder.plan_experts(order, self.plan, first=self.first)
        decoder.swiglu_q8(self.codes, self.scales, self.w13, self.s13, self.act, self.act_scales, offsets=self.plan.offsets, rows=self.plan.rows)
        decoder.linear_q8(self.act, self.act_scales, self.w2, self.s2, self.down, offsets=self.plan.offsets)
        decoder.combine_experts(self.down, self.plan.pos, weights, self.out)
        return self.out

    def exact(self, x, order, weights):
        h = x.double() * torch.rsqrt(x.double().square().mean(1, keepdim=True) + self.eps) * self.norm.double()
        out = torch.zeros(h.shape, dtype=torch.float64, device=DEV)
        for e in range(self.w2.shape[0]):
            t, k = (order == e + self.first).nonzero(as_tuple=True)
            if not len(t):
                continue
            g, u = (h[t] @ wide(self.w13[e, i], self.s13[e, i], 128).T for i in (0, 1))
            y = (g * torch.sigmoid(g) * u) @ wide(self.w2[e], self.s2[e], 128).T
            out.index_add_(0, t, y * weights[t, k, None].double())
        return out


def routing(tokens, used, experts, gen):
    score = torch.randn(tokens, experts, device=DEV, generator=gen)
    top = score.topk(used, 1)
    return top.indices.int(), top.values.softmax(1)


@pytest.mark.parametrize("tokens", [1, 5, 64, 700])
@pytest.mark.parametrize("first,count", [(0, 16), (4, 8)])
def test_experts_together(tokens, first, count):
    """Norm, plan, gate/up, down and sum as one feed-forward, against 64 bits without the two 8-bit roundings.  Each is off by
    at most 2^-4 of a value, evenly spread: 2^-4 / sqrt(3) = 0.036 rms at most, three times over (the gate and the up product
    and the down product see one each): 0.063 of the result."""
    gen, used = gen_of(tokens), 4
    ffn = Ffn(512, 384, 16, used, tokens, 1, first, count)
    x = torch.randn(tokens, 512, device=DEV, generator=gen)
    order, weights = routing(tokens, used, 16, gen)
    got, want = ffn(x, order, weights), ffn.exact(x, order, weights)
    assert float(want.norm()) > 0 and float((got.double() - want).norm() / want.norm()) < 0.063


def test_experts_in_a_graph_and_on_streams():
    """A captured pass replayed on other inputs gives an eager pass's bits, while eager passes run on another stream."""
    gen, tokens, used = gen_of(9), 40, 4
    ffn, other = Ffn(512, 384, 16, used, tokens, 2), Ffn(512, 384, 16, used, tokens, 2)
    sets = [(torch.randn(tokens, 512, device=DEV, generator=gen), *routing(tokens, used, 16, gen)) for _ in range(4)]
    want = [other(*s).clone() for s in sets]
    x, order, weights = (t.clone() for t in sets[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ffn(x, order, weights)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(10):
        for s, w in zip(sets, want):
            for to, of in zip((x, order, weights), s):
                to.copy_(of)
            graph.replay()
            with torch.cuda.stream(side):
                assert torch.equal(other(*sets[1]), want[1])
            assert torch.equal(ffn.out, w)
    torch.cuda.synchronize()


def test_outputs_that_are_inputs_are_refused():
    x, xs, w, ws = operands(8, 128, 128, gen_of(1), (2,))
    with pytest.raises(dm.DracoError, match="overlap"):
        decoder.swiglu_q8(x, xs, w, ws, x, torch.empty(8, 1, device=DEV))
    with pytest.raises(dm.DracoError, match="overlap"):
        decoder.swiglu_q8(x, xs, w, ws, torch.empty_like(x), xs)
    y = torch.zeros(4, 8, device=DEV)
    with pytest.raises(dm.DracoError, match="overlap"):
        decoder.combine_experts(y, ints(0, 0, 0, 0).view(4, 1), torch.ones(4, 1, device=DEV), y)


def test_larger_plan_and_buffers_than_tokens():
    """A server's buffers for its largest batch: places behind the batch's last are left as they were."""
    gen = gen_of(11)
    plan = decoder.plan_experts(torch.randint(6, (10, 2), device=DEV, generator=gen).int(), decoder.ExpertPlan(50, 2, 6))
    x, xs, w, ws = operands(10, 256, 128, gen, (6,))
    out = torch.full((100, 128), 3.0, device=DEV)
    decoder.linear_q8(x, xs, w, ws, out, offsets=plan.offsets, rows=plan.rows)
    assert bool((out[20:] == 3).all())
    for e in range(6):
        a, b = plan.offsets[e:e + 2].tolist()
        same(out[a:b], *plain(of_row(x, plan.rows, a, b), of_row(xs, plan.rows, a, b), w[e], ws[e]), "f32") if b > a else None


def test_offsets_past_32_bits():
    """Weights of more than 2^32 bytes, and a row of x beyond 2^32 bytes: the last group's and the last row's products are right."""
    gen = gen_of(12)
    k, n, groups = 4096, 4096, 260
    w = torch.zeros(groups, n, k, dtype=torch.uint8, device=DEV).view(E4M3)
    ws = torch.ones(groups, n // 128, k // 128, device=DEV)
    last = codes_of((n, k), gen)
    w[-1] = last
    big = torch.zeros(1 << 20, 4112, dtype=torch.uint8, device=DEV).view(E4M3)      # 4.3 GB of rows, of which the last are used
    x, xs = big[:, :k], torch.ones(1 << 20, k // 128, device=DEV)
    x[-40:] = codes_of((40, k), gen)
    rows = torch.arange((1 << 20) - 40, 1 << 20, device=DEV).int()
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device=DEV)
    offsets[-1] = 40
    for form in (0, 1, 2, 64, 256):
        dm.lib().draco_b200_test_q8_form(form)
        out = decoder.linear_q8(x, xs, w, ws, torch.zeros(40, n, device=DEV), offsets=offsets, rows=rows)
        same(out, *plain(x[-40:], xs[-40:], last, ws[-1]), "f32")
    dense = decoder.linear_q8(x[-40:], xs[-40:], last, ws[-1], torch.zeros(40, n, device=DEV))
    same(dense, *plain(x[-40:], xs[-40:], last, ws[-1]), "f32")


def test_stream_argument():
    x, xs, w, ws = operands(20, 256, 256, gen_of(8))
    want = decoder.linear_q8(x, xs, w, ws, torch.empty(20, 256, device=DEV)).clone()
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.Stream().cuda_stream):
        out = torch.zeros(20, 256, device=DEV)
        torch.cuda.synchronize()
        decoder.linear_q8(x, xs, w, ws, out, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("which,bits", [(1, 0x101), (2, 0x102), (3, 0x104)])
@pytest.mark.parametrize("rows,n,form", [(20, 256, 64), (20, 256, 256), (300, 512, 32), (300, 512, 64), (300, 512, 128), (300, 512, 256),
                                         (300, 512, 2048 + 64), (20, 512, 2048 + 256), (50, 512, 64), (50, 512, 128), (50, 512, 256),
                                         (50, 512, 4096 + 256)])
def test_waits_that_run_out(rows, n, form, which, bits, swiglu):
    """Barriers of the tensor-core form that expect an arrival which never comes: the call ends, its rows are NaN, the status
    says which wait it was (others may have run out with it), and the next call is right."""
    if which == 3 and (not swiglu or form > 1024):
        pytest.skip("only blocks of threads that share a scale's columns wait for one another's maxima")
    x, xs, w, ws = operands(rows, 256, n, gen_of(which), (2,) if swiglu else ())
    status = ints(0)
    a = dm.DracoLinearQ8(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), n_x=rows, n_rows=rows, n=n, k=256, n_groups=1,
                         x_stride=256, x_scales_stride=2, out_stride=n, swiglu=int(swiglu), status=status.data_ptr(), wait_limit_us=2000)
    out, scales = torch.zeros(rows, n, dtype=torch.uint8 if swiglu else torch.float32, device=DEV), torch.zeros(rows, cdiv(n, 128), device=DEV)
    a.out, a.out_scales, a.out_scales_stride = out.data_ptr(), scales.data_ptr(), scales.shape[1]
    L = dm.lib()
    torch.cuda.synchronize()
    L.draco_b200_test_q8_form(form)
    assert L.draco_b200_test_q8_barrier_extra(which) == 0
    try:
        assert L.draco_b200_linear_q8(a, None) == 0
    finally:
        assert L.draco_b200_test_q8_barrier_extra(0) == which
    torch.cuda.synchronize()
    assert int(status) & bits == bits
    assert (scales if swiglu else out).isnan().all()
    assert L.draco_b200_linear_q8(a, None) == 0
    torch.cuda.synchronize()
    assert not (scales if swiglu else out).isnan().any()
    if not swiglu:
        same(out, *plain(x, xs, w, ws), "f32")
