"""Decoder-layer operators at the ends of what their arguments allow."""
import importlib.util
import os
import threading
import time

import pytest
import torch

import dracomancer_llmengine_b200 as dm
from dracomancer_llmengine_b200 import decoder, synth
from test_decoder_ops import TYPES, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(dlib):
    pass


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,heads,max_seq,with_lse", [(1, 4, 0, True), (1, 4, 100, True), (1, 16, 100000, True), (3, 4, 5000, True),
                                                         (40, 8, 5000, True), (200, 4, 0, False), (200, 4, 100000, False)])
def test_attend_tables_without_columns(kind, rows, heads, max_seq, with_lse):
    """A table of no pages: every length is cut to 0, nothing is read from it, rows are 0 and lse -infinity."""
    cache = decoder.KV4Cache.empty(2, 16, 2, 64)
    n_req = 3
    q = torch.randn(n_req * rows, heads, 64, device="cuda").to(TYPES[kind])
    cu = ints([rows * r for r in range(n_req + 1)])
    for lens in ([0] * n_req, [5, 0, 1 << 20]):
        out = torch.full_like(q, 3.0)
        lse = torch.zeros(q.shape[:2], device="cuda") if with_lse else None
        cache.attend(q, out, cu, ints(lens), torch.empty(n_req, 0, dtype=torch.int32, device="cuda"), rows, max_seq, lse=lse)
        assert not out.any()
        if with_lse:
            assert bool((lse == -float("inf")).all())


def split_call(seed, lens, heads=8, d=128, page=16):
    """A cache and the arguments of a call whose long axis is split, over pages of random tokens."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    held = [-(-n // page) for n in lens]
    cache = decoder.KV4Cache.empty(sum(held), page, 2, d)
    slots = torch.arange(sum(held) * page, dtype=torch.int32, device="cuda")
    kv = torch.randn(2, slots.numel(), 2, d, device="cuda", generator=gen)
    cache.append(kv[0], kv[1], slots)
    table = torch.full((len(lens), max(held)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = torch.arange(at, at + n, device="cuda")
        at += n
    q = torch.randn(len(lens), heads, d, device="cuda", generator=gen)
    return cache, q, ints(list(range(len(lens) + 1))), ints(lens), table, 1, max(lens)


def test_graphs_of_one_cache_on_two_streams():
    """Two captured calls of one cache, with other requests and lengths, replayed at the same time, eager calls beside them:
    none disturbs another's partial sums."""
    cache, q, cu, seq, table, _, longest = split_call(1, [30000, 9000, 17, 24000])
    cases = []
    for part in (slice(0, 2), slice(1, 4)):
        n = part.stop - part.start
        args = (q[part].clone(), cu[:n + 1].clone(), seq[part].clone(), table[part].clone())
        want = cache.attend(args[0], torch.empty_like(args[0]), *args[1:], 1, longest).clone()
        out, graph = torch.empty_like(args[0]), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.attend(args[0], out, *args[1:], 1, longest)
        cases.append((graph, out, want, torch.cuda.Stream(), args))     # a graph reads its inputs where they were
    torch.cuda.synchronize()
    side, eager = torch.cuda.Stream(), []
    for _ in range(50):
        for graph, out, _, stream, _ in cases:
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(side):
            eager.append(cache.attend(q, torch.empty_like(q), cu, seq, table, 1, longest))
    torch.cuda.synchronize()
    for graph, out, want, _, _ in cases:
        assert torch.equal(out, want)
    assert all(torch.equal(e, eager[0]) for e in eager)
    kept = {t.data_ptr() for t in cache._kept}
    assert len(kept) == 2 and not kept & {t.data_ptr() for t in decoder._eager[cache.device.index].values()}


def test_scratch_is_shared_by_caches_and_outgrown():
    """Caches on one stream share its buffer; a larger call in between leaves the earlier results right."""
    small, large = split_call(2, [5000]), split_call(3, [40000] * 6, heads=16)
    first = [c[0].attend(c[1], torch.empty_like(c[1]), *c[2:]).clone() for c in (small, large)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = [c[0].attend(c[1], torch.empty_like(c[1]), *c[2:]).clone() for c in (small, large, small, large)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, first[i % 2]) for i, a in enumerate(again))
    assert small[0]._scratch is large[0]._scratch and stream.cuda_stream in small[0]._scratch
    assert not small[0]._kept


def test_workspace_of_the_caller():
    cache, q, cu, seq, table, rows, longest = split_call(4, [9000, 100])
    want = cache.attend(q, torch.empty_like(q), cu, seq, table, rows, longest)
    n = cache.workspace_bytes(8, 2, rows, longest, dtype=torch.float32, table_width=table.shape[1])
    assert n > 0 and cache.workspace_bytes(8, 2, 1, 100) == 0
    ws = torch.full((n + 64,), 255, dtype=torch.uint8, device="cuda")
    before = dict(decoder._eager[cache.device.index])
    got = cache.attend(q, torch.empty_like(q), cu, seq, table, rows, longest, workspace=ws[:n])
    assert torch.equal(got, want) and bool((ws[n:] == 255).all()) and decoder._eager[cache.device.index] == before
    for bad in (ws[:n - 1], ws[:n].cpu(), ws[::2], ws[1:n + 1], "x"):
        with pytest.raises(dm.DracoError):
            cache.attend(q, torch.empty_like(q), cu, seq, table, rows, longest, workspace=bad)
    for bad in (dict(n_heads=7), dict(n_heads=0), dict(max_q_len=-1), dict(dtype=torch.float64)):
        with pytest.raises(dm.DracoError):
            cache.workspace_bytes(**{**dict(n_heads=8, n_req=2, max_q_len=1, max_seq_len=100), **bad})


def test_calls_do_not_wait_for_synchronous_ones():
    """A decoder call returns while another thread is inside a synchronous call of the library, which waits for work that was
    queued before it."""
    layer = synth.make_layer(hidden=512, n_exp=8, n_used=2, inter=256)
    x = torch.randn(4, layer.hidden, device="cuda")
    out = torch.empty_like(x)
    dm.forward(layer, x, out=out)       # weights are on the GPU from here on
    plan, zero, one = decoder.BlockPlan(1, 4), ints([0]), ints([1])
    table, free, count = ints([[-1, -1]]), ints([3, 4]), ints([2])
    decoder.plan_blocks(zero, one, table, free, count, 16, plan)    # a kernel's first launch loads it, which may wait for the GPU
    torch.cuda.synchronize()
    side, inside, queued = torch.cuda.Stream(), threading.Event(), torch.cuda.Event()
    torch.cuda._sleep(1_000_000_000)    # about half a second of the default stream, which the synchronous call waits for
    queued.record()

    def synchronous():
        inside.set()
        dm.forward(layer, x, out=out)

    thread = threading.Thread(target=synchronous)
    thread.start()
    inside.wait()
    time.sleep(0.1)
    assert not queued.query()
    decoder.plan_blocks(zero, one, table, free, count, 16, plan, stream=side)
    assert not queued.query(), "the call waited for the synchronous one"
    thread.join()
    torch.cuda.synchronize()
    assert plan.slots.tolist()[:1] == [4 * 16]


@pytest.mark.parametrize("which", [1, 2, 3])
def test_a_wait_that_runs_out_is_reported(which):
    """Barriers that expect an arrival which never comes (a step's keys, weights or products), and waits of up to a
    millisecond: the kernel ends, says so, and gives NaN, not wrong numbers; the next call is right."""
    d, rows, n = 128, 300, 6000
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = decoder.KV4Cache.empty(n // 64 + 1, 64, 2, d)
    kv = torch.randn(2, n, 2, d, device="cuda", generator=gen)
    cache.append(kv[0], kv[1], torch.arange(n, dtype=torch.int32, device="cuda"))
    table = torch.arange(n // 64 + 1, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(rows, 8, d, device="cuda", generator=gen).bfloat16()
    cu, seq = ints([0, rows]), ints([n])
    want = cache.attend(q, torch.empty_like(q), cu, seq, table, rows, n)
    assert torch.isfinite(want).all() and cache.status.tolist() == [0]
    out, status = torch.zeros_like(q), ints([0])
    a = dm.DracoKV4Attention(q.data_ptr(), out.data_ptr(), None, 8 * d, d, 8 * d, d, 2, 8, 1, rows, cu.data_ptr(), seq.data_ptr(),
                             table.data_ptr(), table.shape[1], table.shape[1], rows, n, d ** -0.5, 0, 0, None, 0)
    ws = torch.empty(dm.lib().draco_b200_kv4_attention_workspace(cache._desc, a), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    call = lambda limit, word=status: dm.lib().draco_b200_kv4_attention_checked(  # noqa: E731
        cache._desc, a, word.data_ptr(), limit, torch.cuda.current_stream().cuda_stream)
    assert dm.lib().draco_b200_test_kv4_barrier_extra(which) == 0
    try:
        assert call(1000) == 0, dm.last_error()
    finally:
        assert dm.lib().draco_b200_test_kv4_barrier_extra(0) == which
    torch.cuda.synchronize()
    # 0x100 and the bits of waits; 0x80 would be products that were still in flight at the end
    assert status.item() & 0x100 and status.item() & 0x7f and not status.item() & ~0x17f
    assert torch.isnan(out).all()
    status.zero_()
    for limit in (0, 2000000):
        assert call(limit) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want) and status.item() == 0
    assert call(-1) == -1 and call(2000001) == -1 and call(0, torch.zeros(1, dtype=torch.int32)) == -1


def test_example_does_not_use_rows_of_refused_requests():
    """A step that finds no page for a request: its rows are not taken for results."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decoder_layer.py")
    spec = importlib.util.spec_from_file_location("decoder_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    layer = example.Layer(torch.bfloat16)
    server = example.Server(layer, 2, 64)
    step = lambda n: server.step(*torch.randn(2, sum(n), layer.hidden, device="cuda").bfloat16(), ints(n), max(n))  # noqa: E731
    step([30, 5])
    assert server.check() < 5e-3
    server.n_free.zero_()
    step([1, 1])        # both have room in their pages
    assert server.check() < 5e-3
    step([10, 1])
    with pytest.raises(RuntimeError, match="1 requests found no free page"):
        server.check()
    assert server.ctx.tolist() == [31, 7]
