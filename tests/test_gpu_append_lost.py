"""Tokens whose position lies outside the table, as a padded batch has them: what the append calls allocate holds zeros for them."""
import pytest
import torch

import paged_cases as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
POSITIONS = [0, -1, 7, 300, 2 ** 31 - 1, -2 ** 31, 299, -7, 5]
LOST = torch.tensor([p < 0 or p >= 300 for p in POSITIONS])


def _dirty(*shapes):
    """Leaves memory of these sizes in the allocator's hands that holds no numbers."""
    rooms = [torch.full(s, 0x7f, dtype=torch.uint8, device=DEV) for s in shapes for _ in range(4)]
    del rooms


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("heads", [1, 17, 64])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("offset,interleaved", [(0, False), (64, True)])
def test_indexer_queries(wide, heads, weighted, offset, interleaved):
    from sparse_mla_sm120_b200 import paged
    g = torch.Generator().manual_seed(heads)
    t = len(POSITIONS)
    pos = torch.tensor(POSITIONS, dtype=torch.int64 if wide else torch.int32, device=DEV)
    k, q = (torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV) for s in ((t, 128), (t, heads, 128)))
    w = torch.randn(t, heads, generator=g).to(DEV) if weighted else None
    ki = torch.full((40, 128), 1.5, device=DEV).to(torch.float8_e4m3fn)
    ks = torch.full((40,), 3.0, device=DEV)
    slots = torch.arange(3, 3 + t, device=DEV)
    cs = P.rotary_table(300).to(DEV)
    _dirty((t * heads * 128,), (t * heads * 4,))
    qi, wo = paged.append_indexer_keys(k, ki, ks, slots, pos, cs, interleaved, offset, q, w)
    assert bool((qi.view(torch.uint8)[LOST] == 0).all()) and bool((wo[LOST] == 0).all())
    assert bool((ki.float()[3:3 + t][LOST] == 1.5).all()) and bool((ks[3:3 + t][LOST] == 3).all())
    # the others as in a batch without such tokens
    keep = ~LOST
    ki2, ks2 = ki.clone(), ks.clone()
    qi2, wo2 = paged.append_indexer_keys(k[keep], ki2, ks2, slots[keep], pos[keep], cs, interleaved, offset, q[keep], None if w is None else w[keep])
    assert torch.equal(qi.view(torch.uint8)[keep], qi2.view(torch.uint8)) and torch.equal(wo[keep], wo2)
    assert torch.equal(ki.view(torch.uint8), ki2.view(torch.uint8)) and torch.equal(ks, ks2)
    # a table without positions: all are lost
    _dirty((t * heads * 128,), (t * heads * 4,))
    qi, wo = paged.append_indexer_keys(k, ki, ks, slots, pos, cs[:0], interleaved, offset, q, w)
    assert bool((qi.view(torch.uint8) == 0).all()) and bool((wo == 0).all()) and torch.equal(ki.view(torch.uint8), ki2.view(torch.uint8))


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("heads", [1, 17, 64])
@pytest.mark.parametrize("interleaved", [True, False])
def test_queries(kind, heads, interleaved):
    from sparse_mla_sm120_b200 import paged
    g = torch.Generator().manual_seed(heads)
    t, dt, lat = len(POSITIONS), P.DTYPE[kind], P.LATENT[kind]
    pos = torch.tensor(POSITIONS, device=DEV)
    down, q = (torch.randn(*s, generator=g).to(dt).to(DEV) for s in ((t, lat + 64), (t, heads, 64)))
    cache = P.make_cache(kind, 1, 64, 3).to(DEV)
    before = cache.clone()
    slots = torch.arange(t, device=DEV)
    cs = P.rotary_table(300).to(DEV)
    _dirty((t * heads * 128,))
    out = paged.append_kv_cache(down[:, :lat], down[:, lat:], cache, slots, pos, cs, interleaved, q_pe=q)
    assert bool((out[LOST] == 0).all())
    given = torch.full_like(out, 7)
    paged.append_kv_cache(down[:, :lat], down[:, lat:], cache, slots, pos, cs, interleaved, q_pe=q, q_out=given)
    assert torch.equal(given[~LOST], out[~LOST]) and bool((given[LOST] == 7).all())
    for a, b in zip(P.rows_of(cache, kind), P.rows_of(before, kind)):
        assert torch.equal(a[:t][LOST].contiguous().view(torch.uint8), b[:t][LOST].contiguous().view(torch.uint8))
