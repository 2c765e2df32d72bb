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



@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("heads", [16, 96])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 30, 2.0 ** 40, -2.0 ** 60, 2.0 ** 100])
def test_scores_whose_own_roundings_are_large(kind, heads, size):
    """Scores of this size, whose fp32 steps are larger than any exponent: the row of the largest alone has weight, and it has all of it."""
    q, cache, table, n, scale = _case(kind, [250, 64], 1, heads, 64, 8)
    scale *= size
    out, lse = _run(q, cache, table, n, scale, num_sm_parts=1)
    rows = orc.cache_values(cache.cpu())
    for b, m in enumerate(n.tolist()):
        pos = torch.arange(m)
        k = rows[table[b].cpu().long()[pos // 64], pos % 64]
        qd = q[b, 0].cpu().double()
        s = qd @ k.T * scale
        spread = (qd.abs() @ k.abs().T).amax(dim=1) * abs(scale)
        off = q.shape[-1] * 2.0 ** -23 * spread                        # of a score: fp32 sums of the products
        top, at = s.topk(2, dim=1)
        sure = top[:, 0] - top[:, 1] > 2 * off + 300                    # 2^-300 and less: no weight
        assert float(sure.double().mean()) > 0.7
        v = k[at[:, 0], :512]
        # The weight is 2^r, where r is the rounding of the maximum, and so is the sum; w for the weight's 16 bits (2^r is none of them unless
        # r is 0), w for the output's, a step each for the product, the reciprocal and its product.
        w = P.HALF_STEP[q.dtype]
        assert bool(((out[b, 0].cpu().double() - v).abs() <= (2 * w + w * w + 2.0 ** -21) * v.abs() + 2.0 ** -24)[sure].all())
        assert bool(((lse[b, 0].cpu().double() - top[:, 0] * 1.4426950408889634).abs() <= 1.45 * off + 2.0 ** -22 * top[:, 0].abs())[sure].all())


@pytest.mark.parametrize("heads", [16, 96])
@pytest.mark.parametrize("parts", [1, 2, 5, None])
@pytest.mark.parametrize("sink", [False, True])
def test_scores_far_below_what_stands_for_nothing(heads, parts, sink):
    """Scores of some -5e32, below the -1e30 that the LSE of a row without anything has: all rows alike, so the output is the row."""
    q, cache, table, n, scale = _case("bf16", [700, 130, 0], 1, heads, 64, 9)
    row = torch.where(torch.arange(576, device=DEV) % 3 == 0, -2.0 ** 53, 2.0 ** 52).to(torch.bfloat16)
    cache[:] = row
    q[:] = -row
    sinks = torch.full((heads,), float("-inf"), device=DEV) if sink else None
    out, lse = _run(q, cache, table, n, scale, num_sm_parts=parts, attn_sink=sinks)
    s = float((row.double() * -row.double()).sum()) * scale * 1.4426950408889634
    # equal weights of 1, whole numbers of them: exact sums but for the merge's products, the division and the output's rounding
    assert s < -1e32
    assert float((out[:2].double() - row[:512].double()).abs().max()) <= (2.0 ** -8 + 700 * 2.0 ** -23) * 2.0 ** 53
    assert float((lse[:2].double() - s).abs().max()) <= 576 * 2.0 ** -23 * -s
    assert bool((out[2] == 0).all()) and bool((lse[2] == -1e30).all())
