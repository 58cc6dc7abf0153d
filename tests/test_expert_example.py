"""The example that runs a feed-forward with 8-bit experts, eagerly and as a graph."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("tokens,dtype", [(1, "bf16"), (7, "f32"), (64, "f16"), (300, "bf16")])
def test_expert_layer(dlib, tokens, dtype, graph):
    """An e4m3 rounding is off by at most 2^-4 of a value, 2^-4 / sqrt(3) = 0.036 of it on average (rms) if evenly spread; the rows
    are rounded before the gate and the up product and before the down product: sqrt(3) of it, and 16-bit types' 2^-8 beside it."""
    spec = importlib.util.spec_from_file_location("expert_layer", os.path.join(ROOT, "examples", "expert_layer.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    error = example.main(["--tokens", str(tokens), "--dtype", dtype, "--steps", "2"] + (["--graph"] if graph else []))
    assert error <= 0.0625 + 2.0 ** -8
