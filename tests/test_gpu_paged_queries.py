"""paged_mla_decode_fwd with queries that hold no numbers: their own outputs have none, all others keep their bits."""
import pytest
import torch

import paged_cases as P
from test_gpu_paged import _case, _run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("token", [0, -1])
@pytest.mark.parametrize("s_q,heads,parts", [(2, 16, 1), (3, 8, 5), (4, 40, None), (3, 64, None)])
def test_a_query_that_is_no_number(kind, value, token, s_q, heads, parts):
    """In one head of the first or the last token, under a causal mask: no other head or token of any request changes a bit."""
    q, cache, table, n, scale = _case(kind, [130, 64, 65, 41, 2], s_q, heads, 32, 41 + heads, width=9)
    clean, clean_lse = _run(q, cache, table, n, scale, causal=True, num_sm_parts=parts)
    P.check_attention(clean, clean_lse, q, cache, table, n, scale, True)
    bad = q.clone()
    bad[:, token, heads // 2, 77] = value
    out, lse = _run(bad, cache, table, n, scale, causal=True, num_sm_parts=parts)
    same = torch.ones(s_q, heads, dtype=torch.bool, device=DEV)
    same[token, heads // 2] = False
    assert torch.equal(out[:, same], clean[:, same]) and torch.equal(lse[:, same], clean_lse[:, same])
    mine = out[0, token, heads // 2]
    assert torch.isnan(mine).all() or not torch.equal(mine, clean[0, token, heads // 2])


@pytest.mark.parametrize("kind", ["bf16", "v32", "model1"])
@pytest.mark.parametrize("s_q,heads,parts", [(2, 16, 1), (3, 64, None)])
def test_scores_out_of_range(kind, s_q, heads, parts):
    """One head of the first token whose fp32 scores overflow: the other tokens keep their bits."""
    q, cache, table, n, scale = _case(kind, [130, 65, 41], s_q, heads, 32, 43, width=9)
    clean, clean_lse = _run(q, cache, table, n, scale, causal=True, num_sm_parts=parts)
    bad = q.clone()
    bad[:, 0, heads // 2] = 3e38
    out, lse = _run(bad, cache, table, n, scale, causal=True, num_sm_parts=parts)
    assert torch.equal(out[:, 1:], clean[:, 1:]) and torch.equal(lse[:, 1:], clean_lse[:, 1:])


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("length", [64, 65, 66, 128, 130])
def test_hidden_rows_of_every_value(kind, value, length):
    """One value of one of the newest rows is no number, in the latent part and in the rotated one: tokens that do not see the row keep
    their bits, wherever the row lies in its block."""
    s_q, heads, lat = 3, 16, P.LATENT[kind]
    q, cache, table, n, scale = _case(kind, [length], s_q, heads, 32, 45)
    clean, _ = _run(q, cache, table, n, scale, causal=True)
    for back in (1, 2):
        for rotated in (False, True):
            bad, m = cache.clone(), length - back
            page, at = int(table[0, m // 32]), m % 32
            if kind in ("bf16", "fp16"):
                bad[page, at, 0, 575 if rotated else 100] = value
            elif rotated:
                two = torch.tensor([value], dtype=torch.bfloat16, device=DEV).view(torch.uint8)
                if kind == "v32":
                    bad[page, at, 0, 654:] = two
                else:
                    bad.view(bad.shape[0], -1)[page, at * 576 + 574:at * 576 + 576] = two
            elif kind == "v32":
                bad[page, at, 0, 512:516] = torch.tensor([value], device=DEV).view(torch.uint8)       # the scale of 128 values
            else:
                bad.view(bad.shape[0], -1)[page, at * 576 + 100] = 0x7f
            out, _ = _run(q, bad, table, n, scale, causal=True)
            assert torch.equal(out[:, :s_q - back], clean[:, :s_q - back])
