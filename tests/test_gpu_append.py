"""append_kv_cache and append_indexer_keys against 64-bit formulas: bytes where the format leaves no choice, half a rounding step elsewhere."""
import pytest
import torch

import paged_cases as P
from oracle import sparse_mla_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(kind, tokens, heads, page, pages, seed, wide=True, rows_wide=True):
    g = torch.Generator().manual_seed(seed)
    lat, dt = P.LATENT[kind], P.DTYPE[kind]
    down = (torch.randn(tokens, lat + 64 + 8, generator=g) * torch.exp(torch.randn(tokens, 1, generator=g))).to(dt)     # wider than what is used
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    pos = torch.randint(0, 500, (tokens,), generator=g)
    return dict(kv_c=down[:, :lat], k_pe=down[:, lat:lat + 64], slots=slots if wide else slots.int(), pos=pos if rows_wide else pos.int(),
                q=torch.randn(tokens, heads, 192, generator=g).to(dt), cache=P.make_cache(kind, pages, page, seed + 1))


def _check_rows(kind, before, after, slots, kv_c, k_pe, cos_sin, pos, interleaved):
    """Rows that no slot names keep their bytes; the others hold the format's bytes and rotated values within a rounding."""
    pages, page = before.shape[:2]
    lat0, sc0, pe0 = (t.cpu() for t in P.rows_of(before, kind))
    lat1, sc1, pe1 = (t.cpu() for t in P.rows_of(after, kind))
    hit = torch.zeros(pages * page, dtype=torch.bool)
    good = (slots >= 0) & (slots < pages * page)
    hit[slots[good].long()] = True
    same = lambda a, b: torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert same(lat0[~hit], lat1[~hit]) and same(sc0[~hit], sc1[~hit]) and same(pe0[~hit], pe1[~hit])
    rows, x, kp = slots[good].long(), kv_c[good], k_pe[good]
    if len(rows) == 0:
        return
    if kind in ("bf16", "fp16"):
        assert same(lat1[rows], x.contiguous())
    else:
        full = torch.cat([x, torch.zeros(len(x), 64, dtype=x.dtype)], dim=1).view(len(x), 1, 1, -1)
        packed = (orc.quantize_kv_v32 if kind == "v32" else orc.quantize_kv_model1)(full)
        lat, sc, _ = P.rows_of(packed, kind)
        assert same(lat1[rows], lat) and same(sc1[rows], sc)
    if cos_sin is None:
        assert same(pe1[rows], kp.contiguous())
        return
    ref = orc.rotate_ref(kp, cos_sin, pos[good], interleaved)
    most = kp.double().abs().amax(dim=1, keepdim=True)
    d = (pe1[rows].double() - ref).abs()
    assert bool((d <= P.HALF_STEP[kp.dtype] * ref.abs() + 2.0 ** -22 * 2 * most).all())     # one rounding; two fp32 products and their sum


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("tokens,heads,page,pages,interleaved", [(1, 1, 64, 1, True), (1, 128, 64, 3, False), (7, 5, 16, 2, True), (33, 16, 1, 40, False),
                                                                (130, 17, 48, 4, True), (513, 3, 128, 6, False)])
def test_append(kind, tokens, heads, page, pages, interleaved):
    from sparse_mla_sm120_b200 import paged
    c = _case(kind, tokens, heads, page, pages, 10 * tokens + heads, wide=tokens % 2 == 1, rows_wide=heads % 2 == 0)
    cs = P.rotary_table(500)
    dev = {k: v.to(DEV) for k, v in c.items()}
    kv = torch.cat([c["kv_c"], c["k_pe"], c["kv_c"][:, :8]], dim=1).to(DEV)            # one array, rows further apart than used
    lat = P.LATENT[kind]
    q = torch.randn(tokens, heads, lat + 64, device=DEV).to(P.DTYPE[kind])
    q0 = q.clone()
    r = paged.append_kv_cache(kv[:, :lat], kv[:, lat:lat + 64], dev["cache"], dev["slots"], dev["pos"], cs.to(DEV), interleaved,
                              q_pe=dev["q"][..., 128:], q_out=q[..., lat:])
    torch.cuda.synchronize()
    assert r.data_ptr() == q[..., lat:].data_ptr()
    _check_rows(kind, c["cache"], dev["cache"], c["slots"], c["kv_c"], c["k_pe"], cs, c["pos"], interleaved)
    assert torch.equal(q[..., :lat], q0[..., :lat])
    x = c["q"][..., 128:]
    ref = orc.rotate_ref(x, cs, c["pos"], interleaved)
    d = (q[..., lat:].cpu().double() - ref).abs()
    assert bool((d <= P.HALF_STEP[x.dtype] * ref.abs() + 2.0 ** -21 * x.double().abs().amax(dim=-1, keepdim=True)).all())
    # in place, the same bits
    p = dev["q"][..., 128:]
    again = paged.append_kv_cache(kv[:, :lat], kv[:, lat:lat + 64], dev["cache"], dev["slots"], dev["pos"], cs.to(DEV), interleaved, q_pe=p, q_out=p)
    assert torch.equal(again, q[..., lat:])


@pytest.mark.parametrize("kind", P.KINDS)
def test_append_without_rotation_matches_the_writer(kind):
    from sparse_mla_sm120_b200 import indexer, paged
    c = _case(kind, 64, 1, 64, 1, 77)
    dev = {k: v.to(DEV) for k, v in c.items()}
    assert paged.append_kv_cache(dev["kv_c"], dev["k_pe"], dev["cache"], dev["slots"]) is None
    _check_rows(kind, c["cache"], dev["cache"], c["slots"], c["kv_c"], c["k_pe"], None, None, True)
    if kind == "v32":
        packed = indexer.pack_kv_cache(torch.cat([dev["kv_c"], dev["k_pe"]], dim=1))
        assert torch.equal(dev["cache"].view(64, 656)[dev["slots"]], packed)


@pytest.mark.parametrize("kind", P.KINDS)
def test_append_leaves_out_what_has_no_place(kind):
    """Slots and positions outside: neither the cache nor q_out is touched for them; padded pages keep what lies between them."""
    from sparse_mla_sm120_b200 import paged
    c = _case(kind, 9, 4, 32, 3, 5)
    slots, pos = c["slots"].clone(), c["pos"].clone()
    slots[1], slots[3], slots[5] = -1, 96, 2 ** 40
    pos[2], pos[4], pos[6] = -1, 500, 2 ** 33
    cs = P.rotary_table(500)
    cache = P.padded(c["cache"].to(DEV), 64)
    room = cache.as_strided((3, cache.stride(0)), (cache.stride(0), 1))
    gap = room[:, c["cache"][0].numel():].clone()
    q = torch.full((9, 4, 64), 7.0, device=DEV).to(P.DTYPE[kind])
    x = c["q"][..., 128:].contiguous().to(DEV)
    paged.append_kv_cache(c["kv_c"].to(DEV), c["k_pe"].to(DEV), cache, slots.to(DEV), pos.to(DEV), cs.to(DEV), q_pe=x, q_out=q)
    torch.cuda.synchronize()
    out = (pos < 0) | (pos >= 500)
    _check_rows(kind, c["cache"], cache.cpu(), torch.where(out, -1, slots), c["kv_c"], c["k_pe"], cs, pos.clamp(0, 499), True)
    assert torch.equal(room[:, c["cache"][0].numel():].view(torch.uint8), gap.view(torch.uint8))
    assert bool((q[out.to(DEV)] == 7).all()) and not bool((q[~out.to(DEV)] == 7).any(dim=-1).any(dim=-1).any())
    before = cache.clone()
    e = torch.empty(0, dtype=torch.int64, device=DEV)
    assert paged.append_kv_cache(c["kv_c"][:0].to(DEV), c["k_pe"][:0].to(DEV), cache, e, e, cs.to(DEV), q_pe=x[:0]).shape == (0, 4, 64)
    slots[:] = torch.arange(9)                # a table without positions, and a cache without pages: nowhere to go either
    paged.append_kv_cache(c["kv_c"].to(DEV), c["k_pe"].to(DEV), cache, slots.to(DEV), pos.to(DEV), cs[:0].to(DEV))
    paged.append_kv_cache(c["kv_c"].to(DEV), c["k_pe"].to(DEV), cache[:0], slots.to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(before.contiguous().view(torch.uint8), cache.contiguous().view(torch.uint8))


@pytest.mark.parametrize("kind", ["v32", "model1"])
def test_append_scales_at_their_borders(kind):
    """Groups whose largest value is 448 times a power of two, a step more, zero, tiny and huge; NaN and infinities stay in their rows."""
    from sparse_mla_sm120_b200 import paged
    lat = P.LATENT[kind]
    x = torch.randn(24, lat, generator=torch.Generator().manual_seed(2)).clamp(-1, 1).to(torch.bfloat16)
    for i, top in enumerate([448.0, 450.0, 446.0, 1.75, 1.7578125, 0.0, 1e-30, 1e-4, 0.0448, 3e38, 28.0, 3.5]):
        x[i] = x[i] * 0 if top < 1e-3 else (x[i].float() * min(top, 1e30)).to(torch.bfloat16)
        x[i, ::16] = top
    cache = torch.zeros(1, 64, 1, P.ROW[kind], dtype=torch.uint8)
    dev = cache.to(DEV)
    slots = torch.arange(24)
    k_pe = torch.zeros(24, 64, dtype=torch.bfloat16)
    paged.append_kv_cache(x.to(DEV), k_pe.to(DEV), dev, slots.to(DEV))
    _check_rows(kind, cache, dev.cpu(), slots, x, k_pe, None, None, True)
    x[3, 5] = float("nan")
    paged.append_kv_cache(x.to(DEV), k_pe.to(DEV), dev, slots.to(DEV))
    v = orc.cache_values(dev.cpu())[0]
    assert torch.isnan(v[3, 5]) and torch.isfinite(v[:24][torch.arange(24) != 3]).all()


def test_flat_cache_and_far_rows():
    """The flat form of 656-byte rows, and rows more than 2^32 bytes from the cache's start."""
    from sparse_mla_sm120_b200 import paged
    c = _case("v32", 5, 1, 64, 1, 9)
    flat = torch.zeros(70, 1, 656, dtype=torch.uint8, device=DEV)
    paged.append_kv_cache(c["kv_c"].to(DEV), c["k_pe"].to(DEV), flat, c["slots"].to(DEV))
    _check_rows("v32", torch.zeros(1, 70, 1, 656, dtype=torch.uint8), flat.cpu().view(1, 70, 1, 656), c["slots"], c["kv_c"], c["k_pe"], None, None, True)
    big = torch.empty((65000, 64, 1, 576), dtype=torch.bfloat16, device=DEV)            # 4.8 GB
    slots = torch.tensor([65000 * 64 - 1, 64 * 64000 + 3, 0], device=DEV)
    x = c["kv_c"][:3].contiguous().to(DEV)
    paged.append_kv_cache(x, c["k_pe"][:3].to(DEV), big, slots)
    assert torch.equal(big.view(-1, 576)[slots][:, :512], x)


@pytest.mark.parametrize("tokens,heads,interleaved,offset,rotate", [(1, 64, False, 0, True), (1, 1, True, 64, True), (3, 9, True, 0, True), (70, 32, False, 64, True),
                                                                   (257, 3, False, 0, False), (5, 0, False, 0, True)])
def test_indexer_keys(tokens, heads, interleaved, offset, rotate):
    from sparse_mla_sm120_b200 import paged
    g = torch.Generator().manual_seed(tokens + heads)
    k = (torch.randn(tokens, 136, generator=g) * 3).to(torch.bfloat16)
    q = torch.randn(tokens, heads, 128, generator=g).to(torch.bfloat16)
    w = torch.randn(tokens, heads, generator=g)
    cap = 2 * tokens + 5
    slots = torch.randperm(cap, generator=g)[:tokens]
    if tokens > 4:
        slots[2], slots[4] = -1, cap
        k[1] = 0
    cs, pos = P.rotary_table(300), torch.randint(0, 300, (tokens,), generator=g)
    ki0 = torch.randn(cap, 128, generator=g).to(torch.float8_e4m3fn)
    ki, ks = ki0.to(DEV), torch.full((cap,), 3.0, device=DEV)
    rot = (pos.to(DEV), cs.to(DEV)) if rotate else (None, None)
    r = paged.append_indexer_keys(k.to(DEV)[:, :128], ki, ks, slots.to(DEV), *rot, interleaved=interleaved, rope_offset=offset, q=q.to(DEV), weights=w.to(DEV))
    torch.cuda.synchronize()

    def check(x, codes, scale):
        y = x.double()
        if rotate:
            y[..., offset:offset + 64] = orc.rotate_ref(x[..., offset:offset + 64], cs, pos[:len(x)] if x.dim() == 3 else pos[good], interleaved)
        ref = y.abs().amax(dim=-1).clamp(min=1e-4) / 448
        assert bool(((scale.double() - ref).abs() <= 2.0 ** -21 * ref).all())            # the rotation, a maximum and a division in fp32
        v = codes.double() * scale.double().unsqueeze(-1)
        # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below its normal numbers
        most = y.abs().amax(dim=-1, keepdim=True)
        assert bool(((v - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -10 * scale.double().unsqueeze(-1) + 2.0 ** -20 * most).all())
    good = (slots >= 0) & (slots < cap)
    check(k[good][:, :128], ki.cpu()[slots[good]], ks.cpu()[slots[good]])
    hit = torch.zeros(cap, dtype=torch.bool)
    hit[slots[good]] = True
    assert torch.equal(ki.cpu().view(torch.uint8)[~hit], ki0.view(torch.uint8)[~hit]) and bool((ks.cpu()[~hit] == 3).all())
    qi, wo = (t.cpu() for t in r)
    assert qi.shape == (tokens, heads, 128) and wo.shape == (tokens, heads)
    if heads:
        alone, scale = (t.cpu() for t in paged.append_indexer_keys(k.to(DEV)[:, :128], ki, ks, slots.to(DEV), *rot, interleaved=interleaved,
                                                                  rope_offset=offset, q=q.to(DEV)))
        assert torch.equal(alone.view(torch.uint8), qi.view(torch.uint8)) and torch.equal(wo, w * scale)
        check(q, qi, scale)
    assert paged.append_indexer_keys(k.to(DEV)[:, :128], ki, ks, slots.to(DEV), *rot) is None
