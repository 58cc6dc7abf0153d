"""Decoder-layer operators on the GPU (block planning, 4-bit paged KV cache, attention over it, residual RMS norm with
8-bit output) against plain implementations in 64 bits, at the sizes, strides and masks where they can go wrong."""
import math

import numpy as np
import pytest
import torch

import dracomancer_llmengine_b200 as dm
from dracomancer_llmengine_b200 import decoder

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Relative 2-norm error of rounded outputs: at most half a unit in the last place of each value (2^-24, 2^-11, 2^-8 of
# it).  fp32 results carry the operator's own arithmetic: products of 22-bit halves (2^-22 each, four roundings of a
# score of size ~16: 16 * 2^-21 = 8e-6) and fp32 sums.
TOL = {"f32": 2e-5, "f16": 2.0 ** -11 + 2e-5, "bf16": 2.0 ** -8 + 2e-5}


@pytest.fixture(autouse=True)
def _gpu(dlib):
    pass


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float(torch.linalg.norm(a - b) / max(float(torch.linalg.norm(b)), 1e-30))


# ------------------------------------------------------------------ block planning
def blocks_ref(ctx, new, table, free, n_free, page, cap):
    table, taken, gone = table.copy(), 0, 0
    cu, seq, slots, pos, refused = [0], [], [-1] * cap, [-1] * cap, 0
    width = table.shape[1]
    for r, (c, n) in enumerate(zip(ctx, new)):
        held, want = -(-c // page), -(-(c + n) // page)
        need = want - held
        fits = want <= width
        ok = fits and (need == 0 or taken + need <= n_free)
        if ok:
            for j in range(need):
                table[r, held + j] = free[n_free - 1 - taken - j]
            gone += need
        if fits:
            taken += need
        refused += not ok
        seq.append(c + n if ok else c)
        for i in range(n):
            t, p = cu[-1] + i, c + i
            if t < cap:
                pos[t] = p
                if ok:
                    slots[t] = table[r, p // page] * page + p % page
        cu.append(cu[-1] + n)
    return table, cu, seq, slots, pos, n_free - gone, refused


@pytest.mark.parametrize("n,ctx_max,new_max,page,spare,slack,narrow", [
    (1, 0, 1, 16, 0, 0, 0), (1, 100, 1, 16, 5, 3, 0), (7, 40, 3, 16, 0, 1, 0), (64, 500, 1, 16, 3, 0, 0),
    (513, 300, 9, 32, -4, 2, 0), (1000, 64, 77, 48, 10, -100, 0), (33, 200, 40, 16, 2, 5, 3), (1500, 20, 0, 16, 0, 4, 0),
    (4097, 50, 5, 16, -100, 9, 0)])
def test_blocks(n, ctx_max, new_max, page, spare, slack, narrow):
    rng = np.random.default_rng(n * 7 + new_max)
    ctx, new = rng.integers(0, ctx_max + 1, n), rng.integers(0, new_max + 1, n)
    held, need = -(-ctx // page), -(-(ctx + new) // page) - -(-ctx // page)
    width = max(1, int((held + need).max()) - narrow)
    ctx = np.minimum(ctx, width * page)
    held = -(-ctx // page)
    need = -(-(ctx + new) // page) - held
    ids = rng.permutation(int(held.sum() + need.sum()) + 8).astype(np.int32)
    table = np.full((n, width), -7, np.int32)
    k = 0
    for r in range(n):
        table[r, :held[r]] = ids[k:k + held[r]]
        k += held[r]
    free = ids[k:]
    n_free = min(len(free), max(0, int(need.sum()) + spare))
    cap = max(0, int(new.sum()) + slack)
    want = blocks_ref(ctx.tolist(), new.tolist(), table, free, n_free, page, cap)
    wide = torch.full((n, width + 3), -9, dtype=torch.int32, device="cuda")   # a view of a wider table
    wide[:, :width] = torch.from_numpy(table)
    plan = decoder.BlockPlan(n, cap)
    for t in (plan.slots, plan.positions, plan.cu_new, plan.seq_len, plan.n_free, plan.refused):
        t.fill_(-77)
    for _ in range(2):   # a second call on the same inputs changes nothing
        decoder.plan_blocks(ints(ctx.tolist()), ints(new.tolist()), wide[:, :width], torch.from_numpy(free).cuda(),
                            ints([n_free]), page, plan)
        assert np.array_equal(wide[:, :width].cpu().numpy(), want[0])
        assert bool((wide[:, width:] == -9).all())
        for got, w in ((plan.cu_new, want[1]), (plan.seq_len, want[2]), (plan.slots, want[3]), (plan.positions, want[4]),
                       (plan.n_free, [want[5]]), (plan.refused, [want[6]])):
            assert got.tolist() == w


def test_blocks_nothing():
    plan = decoder.BlockPlan(0, 5)
    e = ints([])
    decoder.plan_blocks(e, e, torch.empty(0, 4, dtype=torch.int32, device="cuda"), ints([1, 2]), ints([2]), 16, plan)
    assert plan.cu_new.tolist() == [0] and plan.slots.tolist() == [-1] * 5 and plan.positions.tolist() == [-1] * 5
    assert plan.n_free.tolist() == [2] and plan.refused.tolist() == [0]


def test_blocks_bad_values_stay_in_bounds():
    """Negative lengths count as 0, a free count beyond the list is cut to it."""
    plan = decoder.BlockPlan(3, 8)
    table = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    decoder.plan_blocks(ints([-5, 0, 2000000000]), ints([2, -3, 2000000000]), table, ints([4, 9]), ints([1 << 30]), 16, plan)
    assert plan.seq_len.tolist() == [2, 0, 2000000000] and plan.refused.tolist() == [1]
    assert table[0].tolist() == [9, -1] and plan.slots.tolist()[:2] == [144, 145] and plan.n_free.tolist() == [1]


# ------------------------------------------------------------------ the cache
def quantise_ref(x, middle):
    """Codes, scale and offset of x [..., 32] (fp32 numpy), each operation rounded to fp32 as the definition has it."""
    f = np.float32
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1), x.max(-1)
        s = np.minimum((hi - lo) * f(1.0 / 15.0), f(65504)).astype(np.float16)
        m = np.clip(lo + s.astype(f) * f(middle), f(-65504), f(65504)).astype(np.float16)
        sf = s.astype(f)
        inv = np.where(sf > 0, f(1) / np.where(sf > 0, sf, f(1)), f(0)).astype(f)
        c = np.clip(np.rint((x - m.astype(f)[..., None]) * inv[..., None]) + f(middle), 0, 15)
    bad = ~np.isfinite(x).all(-1)
    c[bad], s[bad], m[bad] = 0, np.nan, np.nan
    return c.astype(np.uint8), s, m


def tile_views(pages, d):
    """numpy views of the parts of pages [n_pages, heads, tiles, 20 d] by the documented layout."""
    g = d // 32
    lead = pages.shape[:-1]
    cut = lambda a, b, t: pages[..., a * d:b * d].view(t)  # noqa: E731
    return {"kc": cut(0, 8, np.uint8).reshape(*lead, 16, 4, g, 4), "ks": cut(8, 9, np.float16).reshape(*lead, 8, g, 2),
            "km": cut(9, 10, np.float16).reshape(*lead, 16, g), "vc": cut(10, 18, np.uint8).reshape(*lead, 8, 8, g, 2, 2),
            "vs": cut(18, 19, np.float16).reshape(*lead, 8, g, 2), "vm": cut(19, 20, np.float16).reshape(*lead, 8, g, 2)}


def write_ref(pages, page_size, d, k, v, slots):
    """Token by token into the bytes."""
    t = tile_views(pages, d)
    g = d // 32
    kq, vq = quantise_ref(k.reshape(*k.shape[:2], g, 32), 0), quantise_ref(v.reshape(*v.shape[:2], g, 32), 8)
    for i, slot in enumerate(slots):
        if slot < 0 or slot // page_size >= pages.shape[0]:
            continue
        p, tile, tok = slot // page_size, slot % page_size // 16, slot % 16
        c = kq[0][i]                                               # [heads, g, 32]: channel q*8 + 2b + nibble
        b = (c[..., 0::2] | c[..., 1::2] << 4).reshape(-1, g, 4, 4)    # [heads, g, q, b]
        t["kc"][p, :, tile, tok] = b.transpose(0, 2, 1, 3)
        t["ks"][p, :, tile, tok // 2, :, tok % 2] = kq[1][i]
        t["km"][p, :, tile, tok] = kq[2][i]
        c = vq[0][i]                                               # channel n*4 + 2b + nibble
        b = (c[..., 0::2] | c[..., 1::2] << 4).reshape(-1, g, 8, 2)
        t["vc"][p, :, tile, tok // 2, :, :, tok % 2] = b.transpose(0, 2, 1, 3)
        t["vs"][p, :, tile, tok // 2, :, tok % 2] = vq[1][i]
        t["vm"][p, :, tile, tok // 2, :, tok % 2] = vq[2][i]


def read_ref(pages, page_size, d, slots, head):
    """fp64 keys and values [slots, d] of one head from the bytes."""
    t = tile_views(pages, d)
    g = d // 32
    p, tile, tok = slots // page_size, slots % page_size // 16, slots % 16
    b = t["kc"][p, head, tile, tok].transpose(0, 2, 1, 3)          # [n, g, q, b]
    c = np.stack([b & 15, b >> 4], -1).reshape(-1, g, 32).astype(np.float64)
    k = c * t["ks"][p, head, tile, tok // 2, :, tok % 2].astype(np.float64)[..., None] + \
        t["km"][p, head, tile, tok].astype(np.float64)[..., None]
    b = t["vc"][p, head, tile, tok // 2, :, :, tok % 2].transpose(0, 2, 1, 3)
    c = np.stack([b & 15, b >> 4], -1).reshape(-1, g, 32).astype(np.float64) - 8
    v = c * t["vs"][p, head, tile, tok // 2, :, tok % 2].astype(np.float64)[..., None] + \
        t["vm"][p, head, tile, tok // 2, :, tok % 2].astype(np.float64)[..., None]
    return k.reshape(-1, d), v.reshape(-1, d)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d,heads,page,n", [(64, 3, 16, 1), (64, 8, 48, 37), (128, 1, 16, 2), (128, 4, 64, 129),
                                            (256, 2, 32, 50)])
def test_append_bytes_and_read(kind, d, heads, page, n):
    rng = np.random.default_rng(d + n)
    pages = -(-n // page) + 2
    x = torch.from_numpy(rng.standard_normal((n, 3 * heads, d + 8)).astype(np.float32)).cuda() * 3
    x[0, heads:] *= 1e4
    x = x.to(TYPES[kind])
    if n > 30:
        x[3, heads:, :32] = 0.0                      # a constant group
        x[4, heads:, 32:64] = 1.5
        x[5, heads:, 7] = float("nan")
        x[6, heads:, 40] = float("inf")
        x[7, heads:, :32] *= 1e-7                    # scales in fp16's subnormal range
        if kind != "f16":
            x[8, heads:, 1], x[8, heads:, 2] = 3e30, -3e30   # beyond fp16
    slots = rng.permutation(pages * page)[:n]
    if n > 30:
        slots[10], slots[11], slots[12] = -1, pages * page, 2 ** 31 - 1
    off = 0 if d == 64 else 1                        # channels that start off a 16-byte boundary
    k, v = x[:, heads:2 * heads, off:off + d], x[:, 2 * heads:, off:off + d]
    fill = rng.integers(0, 256, (pages, heads, page // 16, 20 * d), dtype=np.uint8)
    cache = decoder.KV4Cache(torch.from_numpy(fill).cuda(), page, d)
    cache.append(k, v, ints(slots.tolist()))
    want = fill.copy()
    write_ref(want, page, d, k.float().cpu().numpy(), v.float().cpu().numpy(), slots.tolist())
    got = cache.pages.cpu().numpy()
    a, b = tile_views(got, d), tile_views(want, d)
    for name in a:
        if a[name].dtype == np.float16:              # NaN payloads may differ, everything else not
            nan = np.isnan(b[name])
            assert np.array_equal(np.isnan(a[name]), nan), name
            assert np.array_equal(a[name][~nan].view(np.uint16), b[name][~nan].view(np.uint16)), name
        else:
            assert np.array_equal(a[name], b[name]), name
    ko = torch.full((n, heads, d), 7.0, dtype=TYPES[kind], device="cuda")
    vo = torch.full((heads, n, d), 7.0, dtype=TYPES[kind], device="cuda").transpose(0, 1)
    cache.read(ints(slots.tolist()), ko, vo)
    inside = (slots >= 0) & (slots < pages * page)
    for h in range(heads):
        kr, vr = read_ref(want, page, d, slots[inside], h)
        for o, w in ((ko, kr), (vo, vr)):
            w = torch.from_numpy(w.astype(np.float32)).to(TYPES[kind])     # one rounding: the sum is exact in 64 bits
            assert torch.equal(torch.nan_to_num(o[:, h].cpu()[inside], 123.0), torch.nan_to_num(w, 123.0))
            assert not o[:, h].cpu()[~inside].any()


# ------------------------------------------------------------------ attention
def make_cache(rng, lens, page, heads, d, spare=2, junk=True):
    """A cache with random tokens for each request, pages in random order; unused bytes are junk (NaN scales too)."""
    held = [-(-n // page) for n in lens]
    n_pages = sum(held) + spare
    if junk:
        pages = rng.integers(0, 256, (n_pages, heads, page // 16, 20 * d), dtype=np.uint8)
        t = tile_views(pages, d)
        for name in ("ks", "km", "vs", "vm"):
            t[name][...] = np.where(rng.random(t[name].shape) < 0.5, np.nan, np.inf)
    else:
        pages = np.zeros((n_pages, heads, page // 16, 20 * d), np.uint8)
    ids = rng.permutation(n_pages)
    table = np.full((len(lens), max(held + [1])), -1, np.int32)
    k = 0
    cache = decoder.KV4Cache(torch.from_numpy(pages).cuda(), page, d)
    for r, n in enumerate(lens):
        table[r, :held[r]] = ids[k:k + held[r]]
        k += held[r]
        if n:
            pos = np.arange(n)
            slots = table[r, pos // page] * page + pos % page
            kv = rng.standard_normal((2, n, heads, d)).astype(np.float32)
            kv[0] += rng.standard_normal((heads, d)).astype(np.float32)
            x = torch.from_numpy(kv).cuda()
            cache.append(x[0], x[1], ints(slots.tolist()))
    return cache, table


def attend_ref(cache, table, q, cu, lens, window, sinks, scale=None):
    """fp64, request by request."""
    pages = cache.pages.cpu().numpy()
    d, page, hkv = cache.head_dim, cache.page_size, cache.n_kv_heads
    q = q.double().cpu().numpy()
    heads = q.shape[1]
    per = heads // hkv
    out, lse = np.zeros_like(q), np.full(q.shape[:2], -np.inf)
    scale = d ** -0.5 if scale is None else scale
    for r, n in enumerate(lens):
        rows = cu[r + 1] - cu[r]
        if not rows or not n:
            continue
        pos = np.arange(n)
        ok = table[r, pos // page] >= 0
        slots = np.where(ok, table[r, pos // page], 0) * page + pos % page
        for h in range(hkv):
            k, v = read_ref(pages, page, d, slots, h)
            for i in range(rows):
                p = n - rows + i
                see = ok & (pos <= p) & ((window == 0) | (p - pos < window) | (pos < sinks))
                if not see.any():
                    continue
                s = q[cu[r] + i, h * per:(h + 1) * per] @ k[see].T * scale
                top = s.max(-1, keepdims=True)
                e = np.exp(s - top)
                out[cu[r] + i, h * per:(h + 1) * per] = e @ v[see] / e.sum(-1, keepdims=True)
                lse[cu[r] + i, h * per:(h + 1) * per] = top[:, 0] + np.log(e.sum(-1))
    return torch.from_numpy(out), torch.from_numpy(lse)


def attend_case(seed, kind, lens, q_lens, heads, hkv, d, page, window=0, sinks=0, max_seq=None, stride=False, scale=None,
                holes=False, with_lse=True):
    rng = np.random.default_rng(seed)
    cache, table = make_cache(rng, lens, page, hkv, d)
    if holes:
        table[0, 0] = -5
        table[-1, 0] = cache.pages.shape[0] + 3
    cu = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)]
    n = cu[-1]
    q = torch.from_numpy(rng.standard_normal((n, heads, d)).astype(np.float32)).cuda().to(TYPES[kind])
    if stride:   # queries and outputs as parts of wider rows, off 16-byte boundaries
        wide = torch.zeros(n, heads + 2, d + 1, dtype=TYPES[kind], device="cuda")
        wide[:, 1:-1, 1:] = q
        q = wide[:, 1:-1, 1:]
        out = torch.full((heads, n, d + 3), 5.0, dtype=TYPES[kind], device="cuda").transpose(0, 1)[..., 1:d + 1]
    else:
        out = torch.full((n, heads, d), 5.0, dtype=TYPES[kind], device="cuda")
    lse = torch.full((n, heads), 5.0, device="cuda") if with_lse else None
    cache.attend(q, out, ints(cu), ints(lens), torch.from_numpy(table).cuda(), max(q_lens), max_seq or max(lens),
                 scale=scale, window=window, sinks=sinks, lse=lse)
    seen_table = np.where((table >= 0) & (table < cache.pages.shape[0]), table, -1)
    want, want_lse = attend_ref(cache, seen_table, q, cu, lens, window, sinks, scale)
    assert torch.isfinite(out).all()
    assert rel(out, want) <= TOL[kind]
    empty = torch.isinf(want_lse)
    assert not out.cpu()[empty].any()
    if not with_lse:
        return cache, table, q, out
    assert torch.equal(torch.isinf(lse).cpu(), empty)
    # lse of size ~10: a few units in the last place of fp32
    assert float((lse.cpu().double() - want_lse)[~empty].abs().max() if (~empty).any() else 0) <= 2e-5
    return cache, table, q, out


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,hkv,d,page", [(1, 1, 64, 16), (8, 8, 128, 16), (8, 2, 128, 48), (32, 4, 128, 64),
                                              (12, 1, 128, 32), (16, 1, 64, 16), (16, 2, 256, 32), (20, 4, 256, 16)])
def test_attend_single_tokens(kind, heads, hkv, d, page):
    lens = [1, 2, 15, 16, 17, 31, 0, 130, 257, 600]
    attend_case(heads * d, kind, lens, [1] * len(lens), heads, hkv, d, page)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (16, 0), (17, 4), (100, 16), (100, 17), (64, 300),
                                          (5000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_attend_windows(kind, window, sinks):
    attend_case(window % 1000 + sinks % 1000, kind, [700, 3, 129, 40, 0], [1, 1, 3, 2, 1], 8, 2, 128, 16, window, sinks)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,hkv,d", [(4, 4, 64), (8, 1, 128), (6, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 5)])
def test_attend_chunks(kind, heads, hkv, d, window, sinks):
    # chunks that are the whole sequence, end inside a tile, are empty, or outnumber the cached tokens (rows that see
    # nothing)
    attend_case(d + window, kind, [200, 65, 300, 9, 70, 128], [200, 1, 37, 13, 0, 128], heads, hkv, d, 16, window, sinks)


@pytest.mark.parametrize("heads,hkv,d,page", [(8, 1, 128, 16), (4, 4, 64, 48), (6, 2, 128, 64), (16, 1, 64, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 5), (1, 0), (64, 200), (500, 64)])
def test_attend_bf16_chunks_without_lse(heads, hkv, d, page, window, sinks):
    """Blocks of 128 rows: whole sequences, chunks behind long contexts, single tokens beside them, no queries at all, more
    queries than cached tokens, row counts around the block's."""
    attend_case(d + window, "bf16", [200, 65, 300, 9, 70, 128, 1500, 0, 64], [200, 1, 37, 13, 0, 128, 150, 3, 16], heads, hkv, d,
                page, window, sinks, with_lse=False)


def test_attend_bf16_chunks_strides_holes_and_bounds():
    attend_case(51, "bf16", [90, 400], [80, 70], 8, 2, 128, 16, stride=True, scale=0.03, with_lse=False)
    attend_case(52, "bf16", [100, 277], [40, 100], 8, 2, 128, 16, holes=True, with_lse=False)
    attend_case(53, "bf16", [3000, 20], [70, 20], 8, 2, 128, 32, max_seq=100, with_lse=False)   # a bound that is too low
    attend_case(54, "bf16", [17], [17], 40, 8, 128, 16, with_lse=False)


def test_attend_bf16_chunks_many_requests():
    """More blocks of rows than one block scans."""
    rng = np.random.default_rng(8)
    q_lens = rng.integers(0, 70, 600).tolist()
    lens = [int(q + e) for q, e in zip(q_lens, rng.integers(0, 50, 600))]
    q_lens[5], lens[5] = 70, 90
    attend_case(55, "bf16", lens, q_lens, 4, 1, 64, 16, with_lse=False)


def test_attend_bf16_chunks_long_splits():
    """A chunk behind a long context: its tiles lie in many blocks' runs."""
    attend_case(56, "bf16", [9000, 300, 5], [33, 20, 5], 8, 2, 128, 64, with_lse=False)


@pytest.mark.parametrize("kind", TYPES)
def test_attend_strides_and_scale(kind):
    attend_case(5, kind, [90, 400], [2, 1], 8, 2, 128, 16, stride=True, scale=0.03)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attend_long_splits(kind):
    """Enough tiles that the long axis is split over many blocks, beside requests that use one split or none."""
    attend_case(6, kind, [20011, 5, 0, 9000], [1, 1, 1, 2], 8, 2, 128, 64)
    attend_case(7, kind, [20011, 5, 0, 9000], [1, 1, 1, 2], 8, 2, 128, 64, max_seq=300)   # a bound that is too low


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 3]])
def test_attend_pages_outside_the_cache(kind, q_lens):
    attend_case(8, kind, [100, 77], q_lens, 4, 2, 128, 16, holes=True)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [1, 21, 80])
@pytest.mark.parametrize("value_only", [False, True])
def test_attend_hidden_nan(kind, rows, value_only):
    """Infinities and NaN in tokens that a row does not see leave it alone, and reach every row that sees them."""
    rng = np.random.default_rng(3)
    n, window, d, hkv = 150, 20, 128, 2
    cache, table = make_cache(rng, [n], 16, hkv, d)
    bad = torch.full((1, hkv, d), float("nan"), device="cuda")
    fine = torch.ones(1, hkv, d, device="cuda")
    pos = 110      # hidden for a single token (position 149); inside the window of queries 129 .. 110 + 19
    cache.append(fine if value_only else bad, bad, ints([int(table[0, pos // 16]) * 16 + pos % 16]))
    q = torch.from_numpy(rng.standard_normal((rows, 4, d)).astype(np.float32)).cuda().to(TYPES[kind])
    out = torch.empty_like(q)
    cache.attend(q, out, ints([0, rows]), ints([n]), torch.from_numpy(table).cuda(), rows, n, window=window, sinks=3)
    p = torch.arange(n - rows, n)
    sees = (pos <= p) & (p - pos < window)
    nan = torch.isnan(out).all(-1).all(-1).cpu()
    assert torch.equal(nan, sees) and torch.equal(torch.isnan(out).any(-1).any(-1).cpu(), sees)
    want, _ = attend_ref(cache, table, q, [0, rows], [n], window, 3)
    assert rel(out[~sees.cuda()], want[~sees]) <= TOL[kind]


@pytest.mark.parametrize("factor", [1e-30, 1e-3, 1e3])
def test_attend_query_magnitudes(factor):
    """Tiny and large fp32 queries (the score's scale undoes the factor, so the result is that of factor 1)."""
    rng = np.random.default_rng(4)
    cache, table = make_cache(rng, [333], 16, 2, 128)
    q = torch.from_numpy(rng.standard_normal((1, 8, 128)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    want, _ = attend_ref(cache, table, q, [0, 1], [333], 0, 0)
    cache.attend(q * factor, out, ints([0, 1]), ints([333]), torch.from_numpy(table).cuda(), 1, 333,
                 scale=128 ** -0.5 / factor)
    assert rel(out, want) <= TOL["f32"]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 64])
def test_attend_peaked_scores(kind, rows):
    """Scores far apart (a few keys take all the weight) and nearly equal ones."""
    rng = np.random.default_rng(9)
    cache, table = make_cache(rng, [500], 16, 1, 64)
    q = torch.from_numpy(rng.standard_normal((rows, 4, 64)).astype(np.float32)).cuda().to(TYPES[kind])
    for scale in (2.0, 1e-4):
        out = torch.empty_like(q)
        cache.attend(q, out, ints([0, rows]), ints([500]), torch.from_numpy(table).cuda(), rows, 500, scale=scale)
        want, _ = attend_ref(cache, table, q, [0, rows], [500], 0, 0, scale)
        # a score of size 60 in fp32 products of 22 bits: 60 * 2^-20 = 6e-5 in the weights
        assert rel(out, want) <= TOL[kind] + 6e-5


def test_attend_no_queries():
    cache = decoder.KV4Cache.empty(2, 16, 1, 64)
    q = torch.zeros(0, 4, 64, device="cuda")
    cache.attend(q, torch.empty_like(q), ints([0, 0]), ints([5]), ints([[0]]), 0, 5)
    cache.attend(q, torch.empty_like(q), ints([0]), ints([]), torch.empty(0, 1, dtype=torch.int32, device="cuda"), 0, 0)
    torch.cuda.synchronize()


def test_cache_beyond_4_gb():
    """Byte offsets past 32 bits: pages at the end of a 5 GB cache."""
    page, heads, d = 128, 8, 128
    per = dm.lib().draco_b200_kv4_page_bytes(page, heads, d)
    n_pages = 5 * 2 ** 30 // per + 1
    pages = torch.empty(n_pages, heads, page // 16, 20 * d, dtype=torch.uint8, device="cuda")
    pages[-3:] = 0
    cache = decoder.KV4Cache(pages, page, d)
    rng = np.random.default_rng(1)
    n = 300
    table = np.array([[n_pages - 1, n_pages - 3, n_pages - 2]], np.int32)
    pos = np.arange(n)
    slots = table[0, pos // page] * page + pos % page
    x = torch.from_numpy(rng.standard_normal((2, n, heads, d)).astype(np.float32)).cuda()
    cache.append(x[0], x[1], ints(slots.tolist()))
    small = decoder.KV4Cache(pages[-3:].contiguous(), page, d)
    local = (table - (n_pages - 3)).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((1, 16, d)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    cache.attend(q, out, ints([0, 1]), ints([n]), torch.from_numpy(table).cuda(), 1, n)
    want, _ = attend_ref(small, local, q, [0, 1], [n], 0, 0)
    assert rel(out, want) <= TOL["f32"]


# ------------------------------------------------------------------ norm
def norm_run(x, w, eps, code, group, res, want_y, inplace=False, pad=0):
    n, hidden = x.shape
    rows = lambda dtype, width: torch.zeros(n, width + pad, dtype=dtype, device="cuda")[:, pad:]  # noqa: E731
    codes = rows(torch.int8, hidden)
    codes = codes if code == "int8" else codes.view(torch.float8_e4m3fn)
    scales = rows(torch.float32, hidden // (group or hidden))
    h = None if res is None else (res if inplace else rows(x.dtype, hidden))
    y = rows(x.dtype, hidden) if want_y else None
    decoder.rmsnorm_q8(x, w, eps, codes, scales, residual=res, h=h, y=y, group=group)
    return codes, scales, h, y


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("n,hidden,group", [(1, 32, 32), (3, 2048, 0), (5, 2048, 256), (200, 896, 64), (2, 7168, 256),
                                            (160, 7168, 128), (149, 4096, 32), (2, 16384, 128), (2, 20000, 32),
                                            (3, 1023, 0), (4, 1, 0), (2, 17, 0), (1, 24, 0), (0, 64, 32)])
def test_norm(kind, code, n, hidden, group):
    rng = np.random.default_rng(hidden + n)
    x = torch.from_numpy(rng.standard_normal((n, hidden)).astype(np.float32)).cuda() * 3
    x = x.to(TYPES[kind])
    r = torch.from_numpy(rng.standard_normal((n, hidden)).astype(np.float32)).cuda().to(TYPES[kind])
    w = torch.from_numpy((1 + 0.3 * rng.standard_normal(hidden)).astype(np.float32)).cuda()
    eps = 1e-5
    for res, want_y, inplace, pad in ((None, True, False, 0), (r, False, False, 0), (r.clone(), True, True, 1)):
        total = x if res is None else (x.float() + res.float()).to(x.dtype)
        codes, scales, h, y = norm_run(x, w, eps, code, group, res, want_y, inplace, pad)
        if n == 0:
            continue
        if res is not None:
            assert torch.equal(h, total)
        t = total.double()
        rstd = 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
        u = total.float() * w                       # fp32 products, as defined
        most = 127.0 if code == "int8" else 448.0
        top = u.abs().unflatten(-1, (-1, group or hidden)).amax(-1)
        inv = (torch.full_like(top, most) / top).repeat_interleave(group or hidden, -1)
        want = (u * inv).round() if code == "int8" else (u * inv).to(torch.float8_e4m3fn).float()
        assert torch.equal(codes.float(), want)     # the codes do not depend on the row's sum
        # scales: quotient, square root, reciprocal and product in fp32, a sum of `hidden` squares (2^-24 per level of
        # its tree and per sequential step of a thread, at most 64)
        assert float(((scales.double() - top.double() / most * rstd) / (top.double() / most * rstd)).abs().max()) <= 70 * 2.0 ** -24
        if want_y:
            assert rel(y, t * rstd * w.double()) <= {"f32": 70 * 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]


@pytest.mark.parametrize("hidden", [512, 515])
def test_norm_special_values(hidden):
    x = torch.ones(6, hidden, device="cuda")
    x[0] = 0.0
    x[1, :32] = 0.0
    x[2, 5] = float("nan")
    x[3, 5] = float("inf")
    x[4] *= 1e-38
    x[5] *= 1e15
    w = torch.ones(hidden, device="cuda")
    group = 32 if hidden == 512 else 0
    codes, scales, _, y = norm_run(x, w, 1e-6, "int8", group, None, True)
    assert not codes[0].any() and not scales[0].any() and not y[0].any()
    if group:
        assert not codes[1, :32].any() and scales[1, 0] == 0 and bool((codes[1, 32:] == 127).all())
    assert bool(torch.isnan(scales[2, 0])) and bool(torch.isnan(scales[3, 0])) and bool(torch.isnan(y[2]).all())
    assert not codes[4].any() and not scales[4].any()
    assert bool((codes[5] == 127).all())
    assert abs(float(scales[5, 0]) * 127 - 1) < 1e-6 and abs(float(y[5, 7]) - 1) < 1e-6


# ------------------------------------------------------------------ use
def test_streams_and_graph():
    """One decode step on a side stream, captured in a graph and replayed on new contents of the same tensors."""
    rng = np.random.default_rng(2)
    page, hkv, heads, d, n = 16, 2, 8, 128, 3
    lens = [40, 16, 5000]
    cache, table = make_cache(rng, lens, page, hkv, d, spare=6)
    used = set(table[table >= 0].tolist())
    free = ints([p for p in range(cache.pages.shape[0]) if p not in used])
    wide = torch.full((n, table.shape[1] + 1), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = torch.from_numpy(table)
    ctx, new, n_free = ints(lens), ints([1, 1, 1]), ints([free.numel()])
    plan = decoder.BlockPlan(n, n)
    kv = torch.randn(2, n, hkv, d, device="cuda")
    q, out = torch.randn(n, heads, d, device="cuda"), torch.empty(n, heads, d, device="cuda")

    def step():
        decoder.plan_blocks(ctx, new, wide, free, n_free, page, plan)
        cache.append(kv[0], kv[1], plan.slots)
        cache.attend(q, out, plan.cu_new, plan.seq_len, wide, 1, 5100)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    kv.normal_()
    q.normal_()
    graph.replay()
    torch.cuda.synchronize()
    want, _ = attend_ref(cache, wide.cpu().numpy(), q, [0, 1, 2, 3], [v + 1 for v in lens], 0, 0)
    assert plan.seq_len.tolist() == [v + 1 for v in lens] and rel(out, want) <= TOL["f32"]


def test_results_repeat():
    """Bit-equal results run after run (fixed orders of every sum)."""
    rng = np.random.default_rng(12)
    cache, table = make_cache(rng, [9000, 300], 32, 4, 128)
    q = torch.randn(2, 32, 128, device="cuda")
    outs = []
    for _ in range(5):
        out = torch.empty_like(q)
        cache.attend(q, out, ints([0, 1, 2]), ints([9000, 300]), torch.from_numpy(table).cuda(), 1, 9000)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_attend_shared_scratch():
    """Calls of unlike shapes in turn over one scratch buffer."""
    rng = np.random.default_rng(21)
    lens = [5000, 31, 700, 0, 64]
    cache, table = make_cache(rng, lens, 16, 4, 128)
    tab, seq = torch.from_numpy(table).cuda(), ints(lens)
    for rows, heads, kind in ((1, 4, "f32"), (3, 32, "bf16"), (1, 64, "f16"), (20, 8, "bf16"), (1, 8, "bf16"), (9, 4, "f32")) * 2:
        n = rows * len(lens)
        q = torch.randn(n, heads, 128, device="cuda").to(TYPES[kind])
        out = torch.empty_like(q)
        cu = list(range(0, n + 1, rows))
        cache.attend(q, out, ints(cu), seq, tab, rows, max(lens))
        want, _ = attend_ref(cache, table, q, cu, lens, 0, 0)
        assert rel(out, want) <= TOL[kind]


def test_refusals():
    cache = decoder.KV4Cache.empty(4, 16, 2, 64)
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    one = ints([0])
    for bad in (lambda: decoder.KV4Cache(torch.zeros(4, 2, 1, 1280, dtype=torch.uint8), 16, 64),
                lambda: decoder.KV4Cache(cache.pages, 32, 64), lambda: decoder.KV4Cache(cache.pages, 16, 128),
                lambda: decoder.KV4Cache.empty(4, 24, 2, 64), lambda: decoder.KV4Cache.empty(4, 16, 2, 96),
                lambda: cache.append(f(1, 2, 64), f(1, 2, 32), one), lambda: cache.append(f(1, 2, 64), f(1, 2, 64).half(), one),
                lambda: cache.append(f(1, 2, 64), f(1, 2, 64), one.long()), lambda: cache.append(f(2, 2, 64), f(2, 2, 64), one),
                lambda: cache.append(f(1, 64, 2).transpose(1, 2), f(1, 2, 64), one),
                lambda: cache.append(f(1, 2, 64).cpu(), f(1, 2, 64), one),
                lambda: cache.attend(f(1, 3, 64), f(1, 3, 64), ints([0, 1]), one, ints([[0]]), 1, 1),
                lambda: cache.attend(f(1, 4, 128), f(1, 4, 128), ints([0, 1]), one, ints([[0]]), 1, 1),
                lambda: cache.attend(f(1, 4, 64), f(1, 4, 64).half(), ints([0, 1]), one, ints([[0]]), 1, 1),
                lambda: cache.attend(f(1, 4, 64), f(1, 4, 64), ints([0]), one, ints([[0]]), 1, 1),
                lambda: cache.attend(f(1, 4, 64), f(1, 4, 64), ints([0, 1]), one, ints([[0], [0]]), 1, 1),
                lambda: cache.attend(f(1, 4, 64), f(1, 4, 64), ints([0, 1]), one, ints([[0]]), 1, 1, window=-1),
                lambda: cache.attend(f(1, 4, 64), f(1, 4, 64), ints([0, 1]), one, ints([[0]]), 1, 1, scale=0.0),
                lambda: cache.attend(f(1, 4, 64), f(1, 4, 64), ints([0, 1]), one, ints([[0]]), 1, 1, scale=float("nan")),
                lambda: cache.attend(f(1, 4, 64), f(1, 4, 64), ints([0, 1]), one, ints([[0]]), 1, 1, lse=f(1, 3)),
                lambda: decoder.rmsnorm_q8(f(2, 64), f(64), 1e-6, f(2, 64), f(2, 1)),
                lambda: decoder.rmsnorm_q8(f(2, 64), f(64), 1e-6, f(2, 64).to(torch.int8), f(2, 2)),
                lambda: decoder.rmsnorm_q8(f(2, 64), f(64), 1e-6, f(2, 64).to(torch.int8), f(2, 4), group=16),
                lambda: decoder.rmsnorm_q8(f(2, 64), f(64), 1e-6, f(2, 64).to(torch.int8), f(2, 1), residual=f(2, 64)),
                lambda: decoder.rmsnorm_q8(f(2, 64), f(64), -1.0, f(2, 64).to(torch.int8), f(2, 1)),
                lambda: decoder.rmsnorm_q8(f(2, 64), f(64).half(), 1e-6, f(2, 64).to(torch.int8), f(2, 1)),
                lambda: decoder.plan_blocks(one, one, ints([[0, 1]]), one, one, 0, decoder.BlockPlan(1, 4)),
                lambda: decoder.plan_blocks(one, one, ints([[0, 1]]), one, one, 16, decoder.BlockPlan(2, 4)),
                lambda: decoder.plan_blocks(one, ints([0, 1]), ints([[0, 1]]), one, one, 16, decoder.BlockPlan(1, 4)),
                lambda: decoder.plan_blocks(one.cpu(), one, ints([[0, 1]]), one, one, 16, decoder.BlockPlan(1, 4))):
        before = dm.lib().draco_b200_launch_count()
        with pytest.raises(dm.DracoError):
            bad()
        assert dm.lib().draco_b200_launch_count() == before
    many = decoder.BlockPlan(16385, 1)
    with pytest.raises(dm.DracoError):
        z = torch.zeros(16385, dtype=torch.int32, device="cuda")
        decoder.plan_blocks(z, z, z[:, None], one, one, 16, many)


def test_c_refusals():
    """The C entry points check for themselves: null, host and misaligned pointers, short workspaces."""
    L = dm.lib()
    cache = decoder.KV4Cache.empty(4, 16, 2, 64)
    x = torch.zeros(4, 2, 64, device="cuda")
    host = torch.zeros(4, 2, 64)
    slots = ints([0, 1, 2, 3])
    call = lambda k, v, s, t=0: L.draco_b200_kv4_append(cache._desc, t, k, 128, 64, v, 128, 64, s, 4, None)  # noqa: E731
    assert call(x.data_ptr(), x.data_ptr(), slots.data_ptr()) == 0
    assert call(None, x.data_ptr(), slots.data_ptr()) == -1 and "null" in dm.last_error()
    assert call(host.data_ptr(), x.data_ptr(), slots.data_ptr()) == -1 and "device" in dm.last_error()
    assert call(x.data_ptr() + 1, x.data_ptr(), slots.data_ptr()) == -1
    assert call(x.data_ptr(), x.data_ptr(), slots.data_ptr(), 3) == -1
    broken = dm.DracoKV4Cache(cache.pages.data_ptr() + 8, 4, 16, 2, 64)
    assert L.draco_b200_kv4_append(broken, 0, x.data_ptr(), 128, 64, x.data_ptr(), 128, 64, slots.data_ptr(), 4, None) == -1
    assert L.draco_b200_kv4_append(None, 0, x.data_ptr(), 128, 64, x.data_ptr(), 128, 64, slots.data_ptr(), 4, None) == -1
    q = torch.zeros(1, 8, 64, device="cuda")
    cu, seq, table = ints([0, 1]), ints([60]), ints([[0, 1, 2, 3]])
    a = dm.DracoKV4Attention(q.data_ptr(), q.data_ptr(), None, 512, 64, 512, 64, 0, 8, 1, 1, cu.data_ptr(), seq.data_ptr(),
                             table.data_ptr(), 4, 4, 1, 1 << 20, 0.1, 0, 0, None, 0)
    need = L.draco_b200_kv4_attention_workspace(cache._desc, a)
    assert need > 0 and L.draco_b200_kv4_attention(cache._desc, a, None) == -1 and "workspace" in dm.last_error()
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need - 1
    assert L.draco_b200_kv4_attention(cache._desc, a, None) == -1
    a.workspace_bytes = need
    out = torch.zeros_like(q)
    a.out = out.data_ptr()
    assert L.draco_b200_kv4_attention(cache._desc, a, None) == 0, dm.last_error()
    a.n_heads = 7
    assert L.draco_b200_kv4_attention(cache._desc, a, None) == -1
    assert L.draco_b200_kv4_attention(cache._desc, None, None) == -1
    assert L.draco_b200_rmsnorm_q8(None, None) == -1
    assert L.draco_b200_kv4_page_bytes(16, 2, 64) == 2 * 1280 and L.draco_b200_kv4_page_bytes(16, 2, 80) == 0
    assert math.isclose(0.0, float(out.abs().max()))
    torch.cuda.synchronize()
