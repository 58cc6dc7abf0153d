"""What the 8-bit products and the operators around them refuse, seen without a GPU: nothing is launched."""
import random

import pytest
import torch

import dracomancer_llmengine_b200 as dm
from dracomancer_llmengine_b200 import decoder

E4M3 = torch.float8_e4m3fn


def linear(**over):
    a = dm.DracoLinearQ8(n_x=4, n_rows=4, n=128, k=128, n_groups=1, dtype=0, x_stride=128, x_scales_stride=1, out_stride=128,
                         out_scales_stride=1)
    for name, value in over.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("over,word", [
    (dict(n=0), "n, k >= 1"), (dict(k=0), "n, k >= 1"), (dict(n_x=-1), "n_x"), (dict(n_rows=-1), "n_rows"),
    (dict(n_groups=0), "n_groups"), (dict(n_groups=1025), "1024"), (dict(dtype=3), "dtype"), (dict(n_groups=2), "offsets"),
    (dict(n_rows=5), "without rows"), (dict(k=1 << 25), "2^24"), (dict(out_stride=127), "strides"),
    (dict(x_stride=-1), "strides"), (dict(swiglu=1, out_scales_stride=0), "strides"), (dict(wait_limit_us=-1), "wait_limit"),
    (dict(wait_limit_us=2000001), "wait_limit"), (dict(), "null")])
def test_c_linear_refuses(over, word):
    assert dm.lib().draco_b200_linear_q8(linear(**over), None) == -1
    assert word in dm.last_error()


def test_c_entries_refuse():
    L = dm.lib()
    assert L.draco_b200_linear_q8(None, None) == -1
    assert L.draco_b200_linear_q8(linear(n_x=0, n_rows=0), None) == 0          # nothing to do
    assert L.draco_b200_plan_experts(None, 4, 2, 0, 8, None, None, None, None) == -1 and "null" in dm.last_error()
    for tokens, used, experts in ((-1, 2, 8), (4, 0, 8), (4, 2, 0), (4, 2, 1025), (1 << 23, 4, 8)):
        assert L.draco_b200_plan_experts(None, tokens, used, 0, experts, None, None, None, None) == -1
    assert L.draco_b200_combine_experts(None, None) == -1
    c = dict(n_y=2, n_tokens=2, n_used=1, hidden=8, dtype=0, out_stride=8)
    for over in (dict(), dict(hidden=0), dict(dtype=-1), dict(n_tokens=-1), dict(out_stride=7), dict(y_stride=-1)):
        assert L.draco_b200_combine_experts(dm.DracoCombineExperts(**{**c, **over}), None) == -1
    assert L.draco_b200_combine_experts(dm.DracoCombineExperts(**{**c, "n_tokens": 0}), None) == 0


def product(**over):
    """Arguments of a call on CPU tensors of the right shapes, which is refused last of all for where they are."""
    a = dict(x=torch.zeros(4, 256).to(E4M3), x_scales=torch.zeros(4, 2), w=torch.zeros(130, 256).to(E4M3),
             w_scales=torch.zeros(2, 2), out=torch.zeros(4, 130))
    return {**a, **over}


@pytest.mark.parametrize("over,word", [
    (dict(), "GPU"), (dict(x=None), "tensor"), (dict(x=torch.zeros(4, 256)), "float8"), (dict(x=torch.zeros(256).to(E4M3)), "x must"),
    (dict(x=torch.zeros(256, 4).to(E4M3).T), "contiguous rows"), (dict(x_scales=torch.zeros(4, 1)), "x_scales"),
    (dict(x_scales=torch.zeros(3, 2)), "x_scales"), (dict(x_scales=torch.zeros(4, 2).double()), "x_scales"),
    (dict(w=torch.zeros(130, 255).to(E4M3)), "w must"), (dict(w=torch.zeros(1, 130, 256).to(E4M3)), "w must"),
    (dict(w=torch.zeros(260, 256).to(E4M3)[::2]), "w must"), (dict(w_scales=torch.zeros(1, 2)), "w_scales"),
    (dict(w_scales=torch.zeros(2, 4)[:, ::2]), "w_scales"), (dict(out=torch.zeros(4, 129)), "column"),
    (dict(out=torch.zeros(5, 130)), "one row"), (dict(out=torch.zeros(4, 130, dtype=torch.int32)), "floating"),
    (dict(out=torch.zeros(130, 4).T), "contiguous rows"), (dict(rows=torch.zeros(3, dtype=torch.int32)), "rows must"),
    (dict(offsets=torch.zeros(2)), "offsets must")])
def test_python_linear_refuses(over, word):
    with pytest.raises(dm.DracoError, match=word):
        decoder.linear_q8(**product(**over))


def test_python_others_refuse():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    a = product(w=torch.zeros(2, 130, 256).to(E4M3), w_scales=torch.zeros(2, 2, 2))
    del a["out"]
    for codes, scales in ((torch.zeros(4, 130).to(E4M3), torch.zeros(4, 2)), (torch.zeros(4, 130), torch.zeros(4, 2)),
                          (torch.zeros(4, 130).to(E4M3), torch.zeros(4, 1)), (torch.zeros(4, 100).to(E4M3), torch.zeros(4, 1))):
        with pytest.raises(dm.DracoError):
            decoder.swiglu_q8(**a, codes=codes, scales=scales)
    with pytest.raises(dm.DracoError, match="w must"):
        decoder.swiglu_q8(**{**a, "w": torch.zeros(3, 130, 256).to(E4M3)}, codes=torch.zeros(4, 130).to(E4M3),
                          scales=torch.zeros(4, 2))
    plan = decoder.ExpertPlan(4, 2, 8, device="cpu")
    for order in (i(4, 2), i(8), i(4, 2).long(), i(5, 2), i(4, 3), i(2, 4).T):
        with pytest.raises(dm.DracoError):
            decoder.plan_experts(order, plan)
    y, w = torch.zeros(8, 16), torch.zeros(4, 2)
    for over in (dict(), dict(y=y.half()), dict(pos=i(4, 3)), dict(weights=w.half()), dict(add=torch.zeros(3, 16)),
                 dict(y=torch.zeros(8, 15)), dict(out=torch.zeros(4, 16).long())):
        with pytest.raises(dm.DracoError):
            decoder.combine_experts(**{**dict(y=y, pos=i(4, 2), weights=w, out=torch.zeros(4, 16)), **over})


@pytest.fixture
def made_up_addresses():
    """Calls look at no address where there is no GPU to launch on."""
    L = dm.lib()
    if L.draco_b200_device_count() > 0:
        pytest.skip("what is not refused would run")
    L.draco_b200_pointers_checked(1)
    yield L
    L.draco_b200_pointers_checked(0)


FAR = 1 << 40       # between buffers that have nothing to do with one another


def refused(rc):
    """Whether a call was refused for what its buffers share; else it fails at its launch."""
    assert rc in (-1, -3) and (rc != -1 or "overlap" in dm.last_error()), (rc, dm.last_error())
    return rc == -1


@pytest.mark.parametrize("reach", [300, 60])
def test_outputs_that_share_bytes_with_inputs(reach, made_up_addresses):
    """Rows of x and of the output laid out at random in one buffer, against the bytes that each has."""
    rng, L, seen = random.Random(1), made_up_addresses, [0, 0]
    for _ in range(4000):
        n_x, k, n_rows, n, elem = rng.randint(1, 6), rng.randint(1, 40), rng.randint(1, 6), rng.randint(1, 8), rng.choice([1, 2, 4])
        stride = rng.choice([0, rng.randint(1, 60), 64])
        out_stride = max(n, rng.choice([stride // elem, rng.randint(0, 20), 64 // elem]))
        at = rng.randint(-reach, reach) * 4
        a = linear(n_x=n_x, k=k, n_rows=n_rows, n=n, x_stride=stride, x_scales_stride=1, out_stride=out_stride,
                   dtype={4: 0, 2: 1, 1: 0}[elem], swiglu=int(elem == 1), x=FAR, x_scales=2 * FAR, w=3 * FAR, w_scales=4 * FAR,
                   rows=5 * FAR, out=FAR + at, out_scales=6 * FAR, out_scales_stride=1)
        mine = {at + r * out_stride * elem + i for r in range(n_rows) for i in range(n * elem)}
        theirs = {r * stride + i for r in range(n_x) for i in range(k)}
        want = bool(mine & theirs)
        assert refused(L.draco_b200_linear_q8(a, None)) == want, (n_x, k, stride, n_rows, n, elem, out_stride, at)
        seen[want] += 1
    assert min(seen) > 200


def test_what_may_not_share_bytes(made_up_addresses):
    """Each output against each input and the other outputs, by its last byte; a large call is answered at once."""
    L = made_up_addresses
    n_x, k, n_rows, n = 1 << 20, 1 << 12, 1 << 21, 1 << 9
    base = dict(n_x=n_x, k=k, n_rows=n_rows, n=n, n_groups=3, swiglu=1, x_stride=k, x_scales_stride=k // 128, out_stride=n,
                out_scales_stride=n // 128, x=FAR, x_scales=2 * FAR, w=3 * FAR, w_scales=4 * FAR, offsets=5 * FAR, rows=6 * FAR,
                out=7 * FAR, out_scales=8 * FAR, status=9 * FAR)
    sizes = dict(x=n_x * k, x_scales=n_x * k // 32, w=6 * n * k, w_scales=24 * (n // 128) * (k // 128), offsets=16, rows=4 * n_rows,
                 out=n_rows * n, out_scales=n_rows * n // 32, status=4)
    call = lambda **over: refused(L.draco_b200_linear_q8(linear(**{**base, **over}), None))  # noqa: E731
    assert not call()
    outputs = ("out", "out_scales", "status")
    for one in outputs:
        for other in sizes:
            if other != one:
                assert call(**{one: base[other] + sizes[other] - 4}) and not call(**{one: base[other] + sizes[other]}), (one, other)
                assert call(**{one: base[other] + 4 - sizes[one]}) and not call(**{one: base[other] - sizes[one]}), (one, other)
    plan = dict(order=FAR, offsets=2 * FAR, rows=3 * FAR, pos=4 * FAR)
    sizes = dict(order=4 * 400, offsets=4 * 9, rows=4 * 400, pos=4 * 400)
    call = lambda **over: refused(L.draco_b200_plan_experts(*(lambda p: (p["order"], 100, 4, 0, 8, p["offsets"], p["rows"], p["pos"], None))({**plan, **over})))  # noqa: E731
    assert not call()
    for one in plan:
        for other in plan:
            if other != one:
                assert call(**{one: plan[other] + sizes[other] - 4}) and not call(**{one: plan[other] + sizes[other]}), (one, other)
    base = dict(y=FAR, pos=2 * FAR, weights=3 * FAR, add=4 * FAR, out=5 * FAR, y_stride=16, pos_stride=2, weights_stride=2, add_stride=16,
                out_stride=16, n_y=10, n_tokens=4, n_used=2, hidden=8, dtype=0)
    call = lambda **over: refused(L.draco_b200_combine_experts(dm.DracoCombineExperts(**{**base, **over}), None))  # noqa: E731
    assert not call() and not call(add=5 * FAR) and not call(add=None)
    assert not call(out=FAR + 32) and not call(out=4 * FAR + 32)            # the other half of wider rows
    assert call(out=FAR + 28) and call(out=2 * FAR + 28) and call(out=3 * FAR) and call(out=4 * FAR + 64)
    assert call(add=5 * FAR, add_stride=8) and not call(add=5 * FAR, add_stride=8, n_tokens=1)
    assert not call(out=FAR, n_used=0)                                       # y is not read
