"""The example that serves one decoder layer: prompts in chunks, then single tokens, with each step's attention checked
against 64 bits over the cache's own values."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# half a unit in the last place of the outputs' type, and the fp32 arithmetic beside it
TOL = {"f32": 2e-5, "f16": 2.0 ** -11 + 2e-5, "bf16": 2.0 ** -8 + 2e-5}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TOL)
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 4)])
def test_decoder_layer(dlib, dtype, window, sinks):
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    errors = example.main(["--requests", "5", "--steps", "3", "--dtype", dtype, "--window", str(window), "--sinks", str(sinks)])
    assert len(errors) == 5 and max(errors) <= TOL[dtype]
