"""paged_mla_decode_fwd where running maxima outgrow their lag after a partition's first block: the accumulator is rescaled between the
products of two blocks."""
import pytest
import torch

import paged_cases as P
from test_gpu_paged import _case, _run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rising(kind, lengths, heads, block, step, seed, s_q=1):
    """Scores that rise by `step` (base 2) from block to block of the rows: by a rotated value of every row (V has none of it; in 584-byte
    rows the 512 values are V, and it is one more value of V)."""
    q, cache, table, n, scale = _case(kind, lengths, s_q, heads, 64, seed, spare=0, std=0.5)
    q[..., -1] = torch.tensor(step / (scale * 1.4426950408889634) / 4, device=DEV).to(q.dtype)      # (fp16 queries stay in range)
    at = {"bf16": slice(575, 576), "fp16": slice(575, 576), "v32": slice(654, 656)}.get(kind)
    for b, m in enumerate(lengths):
        pos = torch.arange(m, device=DEV)
        page, row = table[b].long()[pos // 64], pos % 64
        value = (4.0 * (pos // block)).to(P.DTYPE[kind]).unsqueeze(1)
        if kind == "model1":
            flat = cache.view(cache.shape[0], -1)
            col = row.unsqueeze(1) * 576 + torch.tensor([574, 575], device=DEV)
            flat[page.unsqueeze(1), col] = value.view(torch.uint8)
        else:
            cache[page, row, 0, at] = value.view(torch.uint8) if kind == "v32" else value
    return q, cache, table, n, scale


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("heads", [16, 64, 96, 128])
@pytest.mark.parametrize("lengths,parts", [([384] * 40, None), ([300, 257, 129, 400, 511] * 6, 9), ([384, 260], 1)])
def test_every_block_rescales(kind, heads, lengths, parts):
    """Requests of a few blocks, so that what one of the rescalings loses is not scaled away by those behind it."""
    case = _rising(kind, lengths, heads, 64 if heads <= 64 or kind in ("v32", "model1") else 128, 9.0, 7 + heads)
    out, lse = _run(*case, num_sm_parts=parts)
    P.check_attention(out, lse, *case, False)
    from sparse_mla_sm120_b200 import paged
    for _ in range(100):
        again, again_lse = paged.paged_mla_decode_fwd(*case, num_sm_parts=parts)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("parts", [1, None])
def test_a_long_request_that_rises(kind, parts):
    """32768 rows, 128 heads: a rescaling in each of a partition's blocks (256 of them in one partition), the same bits each time."""
    case = _rising(kind, [32768], 128, 128, 8.5, 5)
    out, lse = _run(*case, num_sm_parts=parts)
    P.check_attention(out, lse, *case, False)
    from sparse_mla_sm120_b200 import paged
    for _ in range(300):
        again, again_lse = paged.paged_mla_decode_fwd(*case, num_sm_parts=parts)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)
