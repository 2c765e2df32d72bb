"""paged_mla_decode_fwd at the ends of the range of scales and scores."""
import pytest
import torch

import paged_cases as P
from oracle import sparse_mla_oracle as orc
from test_gpu_paged import _case, _run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("heads", [16, 96])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -96, -2.0 ** -96])
@pytest.mark.parametrize("parts", [1, 3])
def test_small_scales_and_large_queries(heads, scale, parts):
    """A scale of nothing makes all rows alike, however large the scores; a small one goes with queries that are as large."""
    q, cache, table, n, _ = _case("bf16", [300, 128], 1, heads, 64, 7)
    q = (q.float() * 2.0 ** 90).to(torch.bfloat16)                     # scores of some 2^95
    out, lse = _run(q, cache, table, n, scale, num_sm_parts=parts)
    P.check_attention(out, lse, q, cache, table, n, scale, False)
