"""append_kv_cache refuses a q_out whose vectors lie in one another's place, before any device work, and takes all others."""
import pytest

from sparse_mla_sm120_b200 import _lib

FAKE = 4096


def _call(tokens, heads, token, head):
    return _lib.load().smla_append_kv(FAKE, 512, FAKE, 64, FAKE, 0, 4, 64, 64 * 656, FAKE, 1, FAKE, 1, FAKE, 8, 1, FAKE, 64 * heads, 64, FAKE, token, head,
                                      tokens, heads, None)


@pytest.mark.parametrize("tokens,heads,token,head", [
    (2, 4, 256, 0), (2, 4, 0, 64), (1, 4, 0, 0), (3, 1, 0, 0), (3, 1, 56, 0), (2, 4, 248, 64), (2, 4, 256, 56), (2, 4, 64, 64), (4, 2, 64, 192), (3, 3, 128, 128),
    (2 ** 31 - 1, 128, 8128, 64)])
def test_overlaps(tokens, heads, token, head):
    assert _call(tokens, heads, token, head) == -2 and b"overlap" in _lib.load().smla_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 4), (3, 1), (5, 7)])
@pytest.mark.parametrize("layout", ["tokens outside", "heads outside", "wide"])
def test_places_of_their_own(tokens, heads, layout):
    import torch
    from sparse_mla_sm120_b200 import paged
    q = torch.randn(tokens, heads, 64, device="cuda:0").to(torch.bfloat16)
    room = {"tokens outside": (tokens, heads, 64), "heads outside": (heads, tokens, 64), "wide": (tokens, heads, 200)}[layout]
    out = torch.zeros(room, dtype=torch.bfloat16, device="cuda:0")
    out = out.transpose(0, 1) if layout == "heads outside" else out[..., 128:192] if layout == "wide" else out
    table = torch.cat([torch.ones(1, 32), torch.zeros(1, 32)], dim=1).cuda()          # nothing turns
    at = torch.zeros(tokens, dtype=torch.int64, device="cuda:0")
    z = torch.zeros(tokens, 576, dtype=torch.bfloat16, device="cuda:0")
    cache = torch.zeros(1, 64, 1, 576, dtype=torch.bfloat16, device="cuda:0")
    paged.append_kv_cache(z[:, :512], z[:, 512:], cache, torch.arange(tokens, device="cuda:0"), at, table, q_pe=q, q_out=out)
    assert torch.equal(out, q)
    if tokens > 1 and heads > 1:
        with pytest.raises(ValueError, match="overlap"):
            paged.append_kv_cache(z[:, :512], z[:, 512:], cache, torch.arange(tokens, device="cuda:0"), at, table, q_pe=q, q_out=out[:1].expand(tokens, -1, -1))
