"""Decoder-layer operators at the ends of what their arguments allow."""
import pytest
import torch

from dracomancer_llmengine_b200 import decoder
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
