"""What the 8-bit products and the operators around them refuse, seen without a GPU: nothing is launched."""
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
