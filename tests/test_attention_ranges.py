"""Attention over the 4-bit cache where the values' size, the scores' spread or the tokens' range are not those of unit normal
numbers: against 64 bits, request by request."""
import numpy as np
import pytest
import torch

from dracomancer_llmengine_b200 import decoder
from test_decoder_ops import TOL, TYPES, attend_ref, ints, rel

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(dlib):
    pass


def allowed(kind, want):
    """TOL of the result's norm; an fp16 output has besides half its smallest step (2^-24) of absolute error a value."""
    norm = float(torch.linalg.norm(want))
    return TOL[kind] * norm + (2.0 ** -25 * want.numel() ** 0.5 if kind == "f16" else 0.0)


def filled(k, v, page, spare=1, seed=0):
    """A cache with the tokens of each request (k, v: lists of fp32 [tokens, heads, d]), its table, pages in random order."""
    heads, d = k[0].shape[1:]
    lens = [t.shape[0] for t in k]
    held = [-(-n // page) for n in lens]
    cache = decoder.KV4Cache.empty(sum(held) + spare, page, heads, d)
    ids = np.random.default_rng(seed).permutation(sum(held) + spare)
    table = np.full((len(lens), max(held + [1])), -1, np.int32)
    at = 0
    for r, n in enumerate(lens):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
        pos = np.arange(n)
        if n:
            cache.append(k[r].cuda(), v[r].cuda(), ints((table[r, pos // page] * page + pos % page).tolist()))
    return cache, table, lens


def check(kind, cache, table, lens, q_lens, q, window=0, sinks=0, with_lse=False, want_cache=None):
    cu = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)]
    out = torch.full_like(q, 5.0)
    lse = torch.empty(q.shape[:2], device="cuda") if with_lse else None
    cache.attend(q, out, ints(cu), ints(lens), torch.from_numpy(table).cuda(), max(q_lens), max(lens), window=window,
                 sinks=sinks, lse=lse)
    want, want_lse = attend_ref(cache, table, q, cu, lens, window, sinks)
    assert torch.isfinite(out).all()
    for r in range(len(lens)):
        a, b = out[cu[r]:cu[r + 1]].double().cpu(), want[cu[r]:cu[r + 1]]
        assert float(torch.linalg.norm(a - b)) <= allowed(kind, b), f"request {r}: {rel(a, b)}"
    if with_lse:
        assert float((lse.cpu().double() - want_lse).abs().max()) <= 2e-5
    return out


def dominated(n, margins, value, heads, d, seed):
    """Requests whose first token is `margin` nats above the others and has values near 0 (a thousandth of theirs)."""
    gen = torch.Generator().manual_seed(seed)
    sign = torch.randn(heads, d, generator=gen).sign()
    k, v = [], []
    for m in margins:
        k.append(torch.randn(n, heads, d, generator=gen))
        v.append(value * torch.randn(n, heads, d, generator=gen))
        k[-1][0] = sign * m / d ** 0.5      # a query of ones along the signs scores m
        v[-1][0] *= 1e-3
    return k, v, sign


def queries(kind, sign, rows, per, seed):
    """Queries near the signs of their kv head: [rows, heads, d]."""
    gen = torch.Generator().manual_seed(seed)
    heads, d = sign.shape
    q = sign.repeat_interleave(per, 0) + 0.3 * torch.randn(rows, heads * per, d, generator=gen)
    return q.cuda().to(TYPES[kind])


MARGINS = [0.0, 6.0, 9.0, 12.0, 14.0]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [1e-3, 1e-2, 0.1, 1.0, 1e3])
@pytest.mark.parametrize("n,d,heads,per,window", [(4096, 128, 2, 4, 0), (4099, 128, 1, 16, 1500), (1001, 64, 2, 8, 0),
                                                  (2048, 256, 1, 8, 0)])
def test_dominating_token_single(kind, value, n, d, heads, per, window):
    """A first token that takes most of the weight and adds nothing: the result is what the small weights of the others
    give, in sums split over blocks and in whole units, visible as one of the first tokens beside a window."""
    k, v, sign = dominated(n, MARGINS, value, heads, d, 1)
    cache, table, lens = filled(k, v, 32)
    check(kind, cache, table, lens, [1] * len(lens), queries(kind, sign, len(lens), per, 2), window, 1 if window else 0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [1e-3, 0.1, 1e3])
@pytest.mark.parametrize("rows,window", [(40, 0), (70, 900)])
def test_dominating_token_chunk(kind, value, rows, window):
    """The same for chunks (bf16: the tensor-core form)."""
    n, d, heads, per = 2048, 128, 1, 4
    k, v, sign = dominated(n, MARGINS, value, heads, d, 3)
    cache, table, lens = filled(k, v, 64)
    q_lens = [rows - i for i in range(len(lens))]
    check(kind, cache, table, lens, q_lens, queries(kind, sign, sum(q_lens), per, 4), window, 2 if window else 0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [1e-2, 1.0])
def test_dominating_token_long(kind, value):
    k, v, sign = dominated(100003, [12.0, 14.0], value, 1, 128, 5)
    cache, table, lens = filled(k, v, 64)
    check(kind, cache, table, lens, [1, 1], queries(kind, sign, 2, 8, 6))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("value", [1e-3, 1e-2, 3e4])
def test_value_sizes(kind, value):
    """No token dominates; values far from 1."""
    gen = torch.Generator().manual_seed(7)
    k = [torch.randn(n, 2, 128, generator=gen) for n in (1, 2, 40, 700, 4100)]
    v = [(value * torch.randn(t.shape, generator=gen)).clamp(-6e4, 6e4) for t in k]
    cache, table, lens = filled(k, v, 16)
    q = torch.randn(len(lens), 8, 128, generator=gen).cuda().to(TYPES[kind])
    check(kind, cache, table, lens, [1] * len(lens), q)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_value_sizes_that_change(kind, order):
    """Values that grow, shrink or jump by factors of ten along the context, within what one sum of fp32 can hold."""
    gen = torch.Generator().manual_seed(8)
    n = 3000
    size = 10.0 ** torch.linspace(-3, 3, n)
    size = {"up": size, "down": size.flip(0), "mixed": size[torch.randperm(n, generator=gen)]}[order]
    k = [torch.randn(n, 2, 128, generator=gen)]
    v = [size[:, None, None] * torch.randn(n, 2, 128, generator=gen)]
    cache, table, lens = filled(k, v, 16)
    q = torch.randn(1, 8, 128, generator=gen).cuda().to(TYPES[kind])
    check(kind, cache, table, lens, [1], q)
    check(kind, cache, table, lens, [90], torch.randn(90, 4, 128, generator=gen).cuda().to(TYPES[kind]))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 300), (1, 5000), (70, 300)])
@pytest.mark.parametrize("negative", [False, True])
def test_scores_of_large_magnitude(kind, rows, n, negative):
    """Scores up to 1e32: the largest takes all the weight (they differ by far more than their rounding), whatever its size
    and sign."""
    d = 128
    gen = torch.Generator().manual_seed(10)
    sign = torch.randn(1, d, generator=gen).sign()
    k = torch.randn(n, 1, d, generator=gen)
    if negative:        # every score is below 0
        k = k - sign
    cache, table, lens = filled([k], [torch.randn(n, 1, d, generator=gen)], 32)
    q = (sign + 0.1 * torch.randn(rows, 4, d, generator=gen) if negative else torch.randn(rows, 4, d, generator=gen))
    q = q.cuda().to(TYPES[kind])
    lse = torch.empty(rows, 4, device="cuda") if kind != "bf16" or rows == 1 else None
    for scale in (1e5, 1e6, 3e7, 1e8, 1e9, 1e20, 1e30):
        out = torch.zeros_like(q)
        cache.attend(q, out, ints([0, rows]), ints(lens), torch.from_numpy(table).cuda(), rows, n, scale=scale, lse=lse)
        want, want_lse = attend_ref(cache, table, q, [0, rows], lens, 0, 0, scale)
        # rows in which the first two scores are closer than their rounding may go either way (fp16 keys: 2^-11 a channel)
        s = torch.einsum("rhd,kd->rhk", q.double().cpu(), keys(cache, table, n)) * scale
        mask = torch.arange(n) > torch.arange(n - rows, n)[:, None]
        top = s.masked_fill(mask[:, None], -np.inf).topk(2, -1).values
        clear = (top[..., 0] - top[..., 1]) > s.abs().amax() * 2.0 ** -8
        assert int(clear.sum()) >= rows * 4 // 4
        a, b = out.double().cpu()[clear], want[clear]
        assert float(torch.linalg.norm(a - b)) <= allowed(kind, b), scale
        if lse is not None:
            assert float(((lse.cpu().double() - want_lse) / want_lse).abs().max()) <= 2.0 ** -18


def keys(cache, table, n):
    """fp64 keys of the one request and head of a cache."""
    pos = np.arange(n)
    k = torch.empty(n, 1, cache.head_dim, device="cuda")
    cache.read(ints((table[0, pos // cache.page_size] * cache.page_size + pos % cache.page_size).tolist()), k, torch.empty_like(k))
    return k[:, 0].double().cpu()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 300), (1, 5000), (21, 300), (80, 300)])
@pytest.mark.parametrize("large", [1e2, 1e4])
def test_queries_of_wide_range(kind, rows, n, large):
    """Rows whose largest channels meet keys of 0, so that channels 10^3 to 10^5 times smaller make the scores."""
    d = 128
    gen = torch.Generator().manual_seed(13)
    k = 10 * torch.randn(n, 1, d, generator=gen)
    k[..., :32] = 0.0
    cache, table, lens = filled([k], [torch.randn(n, 1, d, generator=gen)], 16)
    q = 0.1 * torch.randn(rows, 4, d, generator=gen)
    q[..., :32] *= 10 * large
    check(kind, cache, table, lens, [rows], q.cuda().to(TYPES[kind]), with_lse=rows == 1)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 21, 80])
@pytest.mark.parametrize("size", [1e-44, 1e-38, 1e-30, 1e30, 2e38])
def test_queries_at_the_ends_of_their_type(kind, rows, size):
    """Rows of subnormal and of the largest numbers (keys bring the scores back to size 1 where the scale can, else to 0)."""
    n, d = 200, 64
    gen = torch.Generator().manual_seed(14)
    cache, table, lens = filled([torch.randn(n, 1, d, generator=gen)], [torch.randn(n, 1, d, generator=gen)], 16)
    q = (torch.rand(rows, 4, d, generator=gen) * 2 - 1).mul(size).to(TYPES[kind]).cuda()
    out, scale = torch.zeros_like(q), min(0.1 / size, 1e37)
    cache.attend(q, out, ints([0, rows]), ints(lens), torch.from_numpy(table).cuda(), rows, n, scale=scale)
    want, _ = attend_ref(cache, table, q, [0, rows], lens, 0, 0, scale)
    assert rel(out, want) <= TOL[kind]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 21, 80])
@pytest.mark.parametrize("size", [7e4, 4e5, 1e30])
def test_values_beyond_fp16(kind, rows, size):
    """Values that fp16 cannot hold (the cache can, up to its scale's range): rows that see the token have its part, rows that
    do not are left alone."""
    n, d, window, pos = 150, 128, 20, 110
    gen = torch.Generator().manual_seed(11)
    k, v = torch.randn(n, 1, d, generator=gen), torch.randn(n, 1, d, generator=gen)
    v[pos] = size * torch.rand(1, d, generator=gen) * torch.randn(1, d, generator=gen).sign()
    cache, table, lens = filled([k], [v], 16)
    q = torch.randn(rows, 4, d, generator=gen).cuda().to(TYPES[kind])
    out = torch.zeros_like(q)
    cache.attend(q, out, ints([0, rows]), ints(lens), torch.from_numpy(table).cuda(), rows, n, window=window)
    want, _ = attend_ref(cache, table, q, [0, rows], lens, window, 0)
    assert torch.isfinite(out).all()
    for i in range(rows):
        a, b = out[i].double().cpu(), want[i]
        assert float(torch.linalg.norm(a - b)) <= TOL[kind] * float(torch.linalg.norm(b)), (i, n - rows + i)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [1, 21, 80])
@pytest.mark.parametrize("size", [7e4, 4e5])
def test_keys_beyond_fp16(kind, rows, size):
    """Keys that fp16 cannot hold, in one token of each of three tiles, against queries that keep the scores ordinary."""
    n, d = 150, 128
    gen = torch.Generator().manual_seed(12)
    k, v = torch.randn(n, 1, d, generator=gen), torch.randn(n, 1, d, generator=gen)
    for pos in (3, 70, 110):
        k[pos, 0, 32:64] = size * torch.randn(32, generator=gen).clamp(-1.5, 1.5)
    cache, table, lens = filled([k], [v], 16)
    q = torch.randn(rows, 4, d, generator=gen)
    q[..., 32:64] *= 1e-6       # those channels' part of a score is of size 1
    check(kind, cache, table, lens, [rows], q.cuda().to(TYPES[kind]))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [1, 21, 80])
@pytest.mark.parametrize("pos", [70, 146])
def test_nan_values_with_vanishing_weight(kind, rows, pos):
    """A token whose values are NaN and whose weight is e^-60 of the row's: 0 in any number, and yet NaN times it is NaN, in
    tiles that every row sees and in those that some see a part of.  Rows that do not see it are left alone."""
    n, d = 150, 128
    gen = torch.Generator().manual_seed(9)
    sign = torch.randn(1, d, generator=gen).sign()
    k = 0.05 * torch.randn(n, 1, d, generator=gen)
    k[pos // 16 * 16] = sign * 60 / d ** 0.5       # of the same tile: one warp takes both
    v = torch.randn(n, 1, d, generator=gen)
    v[pos] = float("nan")
    cache, table, lens = filled([k], [v], 16)
    q = sign.repeat_interleave(4, 0) + 0.01 * torch.randn(rows, 4, d, generator=gen)
    q = q.cuda().to(TYPES[kind])
    out = torch.zeros_like(q)
    cache.attend(q, out, ints([0, rows]), ints(lens), torch.from_numpy(table).cuda(), rows, n)
    sees = torch.arange(n - rows, n) >= pos
    assert torch.equal(torch.isnan(out).all(-1).all(-1).cpu(), sees)
    assert torch.equal(torch.isnan(out).any(-1).any(-1).cpu(), sees)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [2, 3, 40])
def test_short_rows_behind_a_dominating_token(kind, n):
    """Rows that one or a few small weights make: a weight's rounding then is the result's, in all channels alike."""
    k, v, sign = dominated(n, [5.0 + 0.01 * i for i in range(300)], 1.0, 1, 64, 15)
    cache, table, lens = filled(k, v, 16)
    check(kind, cache, table, lens, [1] * len(lens), queries(kind, sign, len(lens), 1, 16))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [1, 21, 80])
@pytest.mark.parametrize("n", [2, 5, 300])
def test_values_with_outlier_channels(kind, rows, n):
    """Groups of values with one large channel and the rest near 0: the rest's part of the result is near 0 too."""
    gen = torch.Generator().manual_seed(17)
    k, v = [], []
    for _ in range(8):
        k.append(torch.randn(n, 1, 128, generator=gen))
        v.append(1e-3 * torch.randn(n, 1, 128, generator=gen))
        v[-1][..., 5::32] = 10 * torch.randn(n, 1, 4, generator=gen)
    cache, table, lens = filled(k, v, 16)
    q_lens = [min(rows, n)] * len(lens)
    check(kind, cache, table, lens, q_lens, torch.randn(sum(q_lens), 8, 128, generator=gen).cuda().to(TYPES[kind]))
