"""The 8-bit products where they could go wrong: waits of which some run out and some do not, copies that land in any order,
gates beyond the range of exp, inputs and outputs in one buffer."""
import pytest
import torch

import dracomancer_llmengine_b200 as dm
from dracomancer_llmengine_b200 import decoder
from test_q8_ops import DEV, E4M3, cdiv, check_swiglu, gen_of, ints, of_row, operands, plain, same

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(dlib):
    yield
    dlib.draco_b200_test_q8_form(0)
    dlib.draco_b200_test_q8_barrier_extra(0)


def c_call(rows, k, n, seed, swiglu):
    """(arguments of a C call, its tensors: x, x_scales, w, w_scales, out, scales, status)"""
    x, xs, w, ws = operands(rows, k, n, gen_of(seed), (2,) if swiglu else ())
    if swiglu:
        ws /= 500 * k ** 0.5
    out = torch.zeros(rows, n, dtype=torch.uint8 if swiglu else torch.float32, device=DEV)
    scales, status = torch.zeros(rows, cdiv(n, 128), device=DEV), ints(0)
    a = dm.DracoLinearQ8(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), n_x=rows, n_rows=rows, n=n, k=k, n_groups=1,
                         x_stride=k, x_scales_stride=xs.shape[1], out_stride=n, out_scales_stride=scales.shape[1],
                         swiglu=int(swiglu), status=status.data_ptr(), wait_limit_us=2000)
    a.out, a.out_scales = out.data_ptr(), scales.data_ptr()
    return a, (x, xs, w, ws, out, scales, status)


@pytest.mark.parametrize("swiglu,rows,split,columns", [(False, rows, split, columns) for rows in (20, 50, 300) for split in (2, 4, 8)
                                                       for columns in (128, 256)] +
                         [(True, rows, split, 256) for rows in (20, 50, 300) for split in (2, 8)])
def test_waits_that_run_out_in_some_warps(swiglu, rows, split, columns, dlib):
    """A tile's inner size shared by blocks of threads, where the product of one half of the columns never comes: the warps of
    the other half end in time.  The call ends, all rows are NaN, and the next call is right."""
    a, (x, xs, w, ws, out, scales, status) = c_call(rows, 256 * split, 512, rows + split, swiglu)
    torch.cuda.synchronize()
    dlib.draco_b200_test_q8_form(1024 * split + columns)
    dlib.draco_b200_test_q8_barrier_extra(4)
    assert dlib.draco_b200_linear_q8(a, None) == 0
    dlib.draco_b200_test_q8_barrier_extra(0)
    torch.cuda.synchronize()
    assert int(status) & 0x102 == 0x102
    assert (scales if swiglu else out).isnan().all()
    status.zero_()
    assert dlib.draco_b200_linear_q8(a, None) == 0
    torch.cuda.synchronize()
    assert int(status) == 0 and not (scales if swiglu else out).isnan().any()
    if not swiglu:
        same(out, *plain(x, xs, w, ws), "f32")


@pytest.mark.parametrize("swiglu,form", [(False, f) for f in (32, 64, 128, 256, 2048 + 64, 2048 + 256)] +
                         [(True, f) for f in (64, 128, 256, 2048 + 256)])
@pytest.mark.parametrize("rows,k,n", [(20, 4096, 256), (50, 4096, 384), (64, 7168, 130), (300, 4096, 640), (1000, 2064, 1001)])
def test_copies_that_land_in_another_order(rows, k, n, form, swiglu, dlib):
    """Every block's first operands come after all its other copies: the same bits."""
    a, (x, xs, w, ws, out, scales, status) = c_call(rows, k, n, rows + n, swiglu)
    torch.cuda.synchronize()
    dlib.draco_b200_test_q8_form(form)
    assert dlib.draco_b200_linear_q8(a, None) == 0
    torch.cuda.synchronize()
    want, want_scales = out.clone(), scales.clone()
    out.zero_(), scales.zero_()
    dlib.draco_b200_test_q8_barrier_extra(5)
    a.wait_limit_us = 0
    for _ in range(3):
        assert dlib.draco_b200_linear_q8(a, None) == 0
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(out, want) and torch.equal(scales, want_scales)
    if not swiglu:
        same(out, *plain(x, xs, w, ws), "f32")
    else:
        check_swiglu(out.view(E4M3), scales, x, xs, w, ws)


@pytest.mark.parametrize("form", [64, 128, 256])
@pytest.mark.parametrize("each", [10, 30, 100])
def test_copies_that_land_in_another_order_by_expert(each, form, dlib):
    """The same with rows by index, where rows come by other copies, and with many tiles a block."""
    gen, k, n, groups = gen_of(each), 2048, 2048, 12
    x, xs, w, ws = operands(100, k, n, gen, (groups,))
    offsets = torch.arange(groups + 1, device=DEV).int() * each
    rows = torch.randint(100, (groups * each,), device=DEV, generator=gen).int()
    dlib.draco_b200_test_q8_form(form)
    want = decoder.linear_q8(x, xs, w, ws, torch.zeros(groups * each, n, device=DEV), offsets=offsets, rows=rows)
    dlib.draco_b200_test_q8_barrier_extra(5)
    status = ints(0)
    for _ in range(3):
        got = decoder.linear_q8(x, xs, w, ws, torch.zeros(groups * each, n, device=DEV), offsets=offsets, rows=rows, status=status)
        assert int(status) == 0 and torch.equal(got, want)
    same(got[:each], *plain(of_row(x, rows, 0, each), xs[rows[:each].long()], w[0], ws[0]), "f32")


FAR = [3e38, 2.4e38, 1e30, 1000.5, 999.0, 400.0, 163.0, 104.0, 90.0, 88.7, 87.4, 80.1, 79.9, 20.0, 1.0]


@pytest.mark.parametrize("rows", [3, 40, 300])
@pytest.mark.parametrize("form", [0, 1, 2, 64, 128, 256, 2048 + 256])
def test_swiglu_of_far_gates(rows, form, dlib):
    """Gates to the ends of fp32, with ups that bring the product back into its range.  The products are exact here (one value,
    powers of two); silu and the product are within 2^-21, the scale's quotient is rounded once more; codes are off by half a step
    (2^-4 of the value, 2^-10 below the normal range) and by what value and scale are off (2^-20 together)."""
    dlib.draco_b200_test_q8_form(form)
    k, f = 256, 128
    x, w = torch.zeros(rows, k, device=DEV), torch.zeros(2, f, k, device=DEV)
    x[:, 0] = 1
    sign = torch.tensor([1.0, -1.0, 0.5, -0.5, 0.25, -0.25, 2.0 ** -6, -2.0 ** -6], device=DEV)
    w[0, :, 0], w[1, :, 0] = sign.repeat(f // 8), sign.repeat_interleave(f // 8)
    x, w = x.to(E4M3), w.to(E4M3)
    for gate in FAR + [-g for g in FAR]:
        for up in (3e38, 1e30, 1e18, 1e9, 1.0, 1e-6, 1e-30, 0.0):
            ws = torch.ones(2, 1, 2, device=DEV)
            ws[0], ws[1] = gate, up
            codes, scales = torch.empty(rows, f, device=DEV).to(E4M3), torch.empty(rows, 1, device=DEV)
            decoder.swiglu_q8(x, torch.ones(rows, 2, device=DEV), w, ws, codes, scales)
            g, u = (ws[i, 0, 0].double() * w[i, :, 0].double() for i in (0, 1))
            h = g / (1 + torch.exp(-g)) * u
            a, got = float(h.abs().max()), scales.double()
            assert bool((codes.view(torch.uint8) == codes.view(torch.uint8)[0]).all() and (got == got[0]).all() or got.isnan().all())
            if a > 3.41e38:
                assert got.isnan().all()
            elif a < 2.0 ** -101:
                assert not got.any() and not codes.float().any()
            elif a > 2.0 ** -99 and a < 3.4e38:
                assert bool(((got - a / 448).abs() <= a / 448 * 2.0 ** -20).all())
                v = h / a * 448
                assert bool(((codes.double() - v).abs() <= v.abs() * (2.0 ** -4 + 1.1 * 2.0 ** -20) + 2.0 ** -10).all())


@pytest.mark.parametrize("form", [0, 1, 2, 64, 128, 256])
def test_swiglu_of_infinite_gates(form, dlib):
    """silu(infinity) = infinity and silu(-infinity) = -infinity / infinity: the block's scale is NaN, other blocks' are not."""
    dlib.draco_b200_test_q8_form(form)
    x, w = torch.zeros(5, 128, device=DEV), torch.ones(2, 256, 128, device=DEV)
    x[:, 0] = 1
    for gate in (float("inf"), -float("inf"), float("nan")):
        ws = torch.ones(2, 2, 1, device=DEV)
        ws[0, 1] = gate
        codes, scales = torch.empty(5, 256, device=DEV).to(E4M3), torch.empty(5, 2, device=DEV)
        decoder.swiglu_q8(x.to(E4M3), torch.ones(5, 1, device=DEV), w.to(E4M3), ws, codes, scales)
        assert scales[:, 1].isnan().all() and bool((scales[:, 0] > 0).all() and (codes.float()[:, :128] == 448).all())


def test_parts_of_one_buffer():
    """Inputs and outputs side by side in the rows of one buffer are apart; ones that share a byte are refused, with nothing written."""
    buf = torch.zeros(40, 512, device=DEV).to(E4M3)
    x, xs, w, ws = operands(40, 256, 128, gen_of(2), (2,))
    buf[:, :256] = x
    want = decoder.swiglu_q8(x, xs, w, ws, torch.empty(40, 128, device=DEV).to(E4M3), torch.empty(40, 1, device=DEV))
    wide_s = torch.cat([xs, xs.new_zeros(40, 1)], 1)
    got = decoder.swiglu_q8(buf[:, :256], wide_s[:, :2], w, ws, buf[:, 256:384], wide_s[:, 2:])
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    before = buf.view(torch.uint8).clone()
    for codes, scales in ((buf[:, 255:383], wide_s[:, 2:]), (buf[:, 256:384], wide_s[:, 1:2]), (buf[:, 384:], ws.view(-1)[:1].expand(40, 1)),
                          (buf[:, 384:], buf.view(torch.float32)[:, 100:101])):
        with pytest.raises(dm.DracoError, match="overlap|strides"):
            decoder.swiglu_q8(buf[:, :256], wide_s[:, :2], w, ws, codes, scales)
    flat = torch.zeros(8192, device=DEV)
    with pytest.raises(dm.DracoError, match="overlap"):
        decoder.linear_q8(x, flat[:80].view(40, 2), w[0], ws[0], flat[79:79 + 40 * 128].view(40, 128))
    order = torch.zeros(65, 2, dtype=torch.int32, device=DEV)
    plan = decoder.ExpertPlan(64, 2, 4)
    plan.pos = order[1:]
    with pytest.raises(dm.DracoError, match="overlap"):
        decoder.plan_experts(order[:64], plan)
    y = torch.zeros(9, 16, device=DEV)
    with pytest.raises(dm.DracoError, match="overlap"):
        decoder.combine_experts(y[:8], ints(0, 1).view(2, 1), torch.ones(2, 1, device=DEV), y[7:9])
    torch.cuda.synchronize()
    assert torch.equal(buf.view(torch.uint8), before) and not flat.any() and not order.any()


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("rows,form", [(20, 128), (20, 256), (50, 128), (300, 128), (300, 256)])
def test_waits_that_run_out_leave_nothing_wrong(rows, form, swiglu, dlib):
    """Without shared tiles: what is not NaN is right, what has no product is NaN."""
    a, (x, xs, w, ws, out, scales, status) = c_call(rows, 512, 512, rows, swiglu)
    dlib.draco_b200_test_q8_form(form)
    dlib.draco_b200_test_q8_barrier_extra(4)
    torch.cuda.synchronize()
    assert dlib.draco_b200_linear_q8(a, None) == 0
    torch.cuda.synchronize()
    assert int(status) & 0x102 == 0x102
    if swiglu:
        assert scales.isnan().all()
    else:
        want, bound = plain(x, xs, w, ws)
        bad = out.isnan()
        assert bad.any() and not bad.all()
        same(torch.where(bad, 0.0, out), torch.where(bad, 0.0, want), bound, "f32")
