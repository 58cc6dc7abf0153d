"""The 8-bit products where they could go wrong: waits of which some run out and some do not."""
import pytest
import torch

import dracomancer_llmengine_b200 as dm
from test_q8_ops import DEV, cdiv, gen_of, ints, operands, plain, same

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(dlib):
    yield
    dlib.draco_b200_test_q8_form(0)
    dlib.draco_b200_test_q8_barrier_extra(0)


def c_call(rows, k, n, seed, swiglu):
    """(arguments of a C call, its tensors: x, x_scales, w, w_scales, out, scales, status)"""
    x, xs, w, ws = operands(rows, k, n, gen_of(seed), (2,) if swiglu else ())
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
