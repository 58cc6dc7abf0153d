"""The decoder-layer operators on a machine without a GPU: shapes that need no device, and loud refusals instead of a
fallback."""
import pytest
import torch

import dracomancer_llmengine_b200 as dm
from dracomancer_llmengine_b200 import decoder


def test_page_bytes():
    f = dm.lib().draco_b200_kv4_page_bytes
    # 1.25 bytes for a key and a value channel
    assert f(16, 1, 64) == 16 * 64 * 5 // 4 and f(48, 3, 128) == 48 * 3 * 128 * 5 // 4 and f(128, 8, 256) == 128 * 8 * 320
    assert f(24, 1, 64) == 0 and f(0, 1, 64) == 0 and f(16, 0, 64) == 0 and f(16, 1, 96) == 0


def test_c_entries_refuse_null_and_bad_shapes():
    L = dm.lib()
    assert L.draco_b200_plan_blocks(None, None, 1, 16, None, 1, 1, None, 0, None, 0, None, None, None, None, None, None,
                                    None) == -1
    assert "null" in dm.last_error()
    assert L.draco_b200_plan_blocks(None, None, 20000, 16, None, 1, 1, None, 0, None, 0, None, None, None, None, None, None,
                                    None) == -1
    assert L.draco_b200_kv4_append(None, 0, None, 0, 0, None, 0, 0, None, 1, None) == -1
    cache = dm.DracoKV4Cache(None, 1, 16, 1, 64)
    assert L.draco_b200_kv4_read(cache, 0, None, 0, 0, None, 0, 0, None, 1, None) == -1 and "cache" in dm.last_error()
    assert L.draco_b200_kv4_attention(cache, None, None) == -1
    assert L.draco_b200_kv4_attention_workspace(cache, None) == 0
    assert L.draco_b200_rmsnorm_q8(None, None) == -1
    norm = dm.DracoNormQ8(dtype=0, fmt=0, n_rows=1, hidden=100, group=32)
    assert L.draco_b200_rmsnorm_q8(norm, None) == -1 and "group" in dm.last_error()
    norm.group = 0
    assert L.draco_b200_rmsnorm_q8(norm, None) == -1 and "null" in dm.last_error()


def test_python_refuses_cpu_tensors():
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(dm.DracoError):
        decoder.KV4Cache(torch.zeros(4, 2, 1, 1280, dtype=torch.uint8), 16, 64)
    with pytest.raises(dm.DracoError):
        decoder.plan_blocks(i(0), i(1), i(0)[:, None], i(0), i(1), 16, decoder.BlockPlan(1, 4, device="cpu"))
    with pytest.raises(dm.DracoError):
        decoder.rmsnorm_q8(torch.zeros(2, 64), torch.ones(64), 1e-6, torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2, 1))
    with pytest.raises(dm.DracoError):
        decoder.rmsnorm_q8(None, None, 1e-6, None, None)
