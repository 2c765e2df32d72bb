"""paged_mla_decode_fwd against the 64-bit formula: every cache layout, lengths, page sizes, tables, masks, sinks, partitions, streams and
graphs; and a whole step of appends and attention."""
import pytest
import torch

import paged_cases as P
from oracle import sparse_mla_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _run(q, cache, table, lengths, scale, **kw):
    from sparse_mla_sm120_b200 import paged
    from sparse_mla_sm120_b200._runtime import check_status
    r = paged.paged_mla_decode_fwd(q, cache, table, lengths, scale, **kw)
    torch.cuda.synchronize()
    check_status(torch.device(DEV))
    return r


def _case(kind, lengths, s_q, heads, page, seed, spare=2, std=1.0, width=None):
    pages = sum(-(-max(n, 0) // page) for n in lengths) + spare
    cache = P.make_cache(kind, pages, page, seed, std)
    table = P.table_of(lengths, page, pages, seed + 1, width)
    g = torch.Generator().manual_seed(seed + 2)
    d = P.LATENT[kind] + 64
    q = (0.7 * torch.randn(len(lengths), s_q, heads, d, generator=g)).to(P.DTYPE[kind])
    return q.to(DEV), cache.to(DEV), table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), d ** -0.5


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("lengths,s_q,heads,page,causal", [
    ([1], 1, 1, 64, False),
    ([64], 1, 16, 64, False),
    ([65], 1, 64, 64, False),
    ([200], 1, 128, 64, False),
    ([0, 1, 63, 64, 65, 127, 128, 129], 1, 16, 64, False),
    ([300, 0, 0, 17, 0, 1000, 2], 1, 40, 64, True),
    ([5, 130, 1, 0, 3, 64], 3, 24, 64, True),       # requests with fewer rows than queries: some queries see nothing
    ([90, 70], 5, 128, 64, True),
    ([400, 333], 2, 8, 16, True),
    ([100, 333], 1, 20, 48, False),                  # pages that end inside a block
    ([77, 61], 1, 128, 2, False),
    ([150], 2, 65, 130, False),
    ([2500, 900], 1, 128, 64, False),
])
def test_attention(kind, lengths, s_q, heads, page, causal):
    q, cache, table, n, scale = _case(kind, lengths, s_q, heads, page, len(lengths) * 100 + heads)
    out, lse = _run(q, cache, table, n, scale, causal=causal)
    P.check_attention(out, lse, q, cache, table, n, scale, causal)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "v32"])
def test_odd_pages(kind):
    """Pages of one row, of three and of seven; 584-byte rows need pages that start on 16 bytes."""
    for page in (1, 3, 7):
        q, cache, table, n, scale = _case(kind, [65, 130, 7], 1, 16, page, page)
        out, lse = _run(q, cache, table, n, scale)
        P.check_attention(out, lse, q, cache, table, n, scale, False)


def test_odd_pages_of_584_byte_rows_are_refused():
    q, cache, table, n, scale = _case("model1", [10], 1, 16, 3, 1)
    with pytest.raises(ValueError, match="aligned"):
        _run(q, cache, table, n, scale)


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("parts", [1, 2, 3, 7, 40, 148, 300])
def test_partitions(kind, parts):
    """However the rows are cut, requests within a partition and requests over many."""
    q, cache, table, n, scale = _case(kind, [700, 3, 0, 1300, 64, 65], 1, 70, 64, 11)
    sink = torch.randn(70, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    out, lse = _run(q, cache, table, n, scale, num_sm_parts=parts, attn_sink=sink)
    P.check_attention(out, lse, q, cache, table, n, scale, False, sink)
    again, _ = _run(q, cache, table, n, scale, num_sm_parts=parts, attn_sink=sink)
    assert torch.equal(out, again)


@pytest.mark.parametrize("parts", [1, None])
def test_sinks(parts):
    """No sink's weight, all of it, and sinks far above and below the scores; a request without rows has its sink as LSE."""
    sink = torch.tensor([float("-inf"), float("inf"), 200.0, -200.0, 0.0, 3.0, 88.0, -1.0], device=DEV)
    q, cache, table, n, scale = _case("bf16", [500, 0, 2], 1, 8, 64, 21)
    out, lse = _run(q, cache, table, n, scale, attn_sink=sink, num_sm_parts=parts)
    P.check_attention(out, lse, q, cache, table, n, scale, False, sink)


@pytest.mark.parametrize("kind", P.KINDS)
def test_peaked_and_large_scores(kind):
    """Scores that grow along the rows (the running maximum moves in every block) and rows whose largest score is far above the others."""
    q, cache, table, n, scale = _case(kind, [640], 1, 16, 64, 31, spare=0, std=0.2)
    rows = orc.cache_values(cache.cpu())[table.cpu()[0].long()].reshape(640, -1)
    q = (rows[[639, 5, 100, 64] * 4] * 6).view(1, 1, 16, -1).to(q.dtype).to(DEV)
    out, lse = _run(q, cache, table, n, scale * 4)
    P.check_attention(out, lse, q, cache, table, n, scale * 4, False)


@pytest.mark.parametrize("kind", P.KINDS)
@pytest.mark.parametrize("parts", [1, 5])
def test_what_is_not_seen_does_not_matter(kind, parts):
    """No-number bytes behind the rows of a request, in pages that it does not have, and in the rows that a query must not see."""
    q, cache, table, n, scale = _case(kind, [130, 65, 40], 2, 16, 32, 41, width=9)
    clean, clean_lse = _run(q, cache, table, n, scale, causal=True, num_sm_parts=parts)
    P.check_attention(clean, clean_lse, q, cache, table, n, scale, True)
    poison = cache.clone()
    used = torch.zeros(poison.shape[0], 32, dtype=torch.bool)
    for b, m in enumerate(n.tolist()):
        for j in range(m):
            used[int(table[b, j // 32]), j % 32] = True
    fill = 0x7f if poison.dtype == torch.uint8 else float("nan")
    if kind == "model1":
        flat = poison.view(poison.shape[0], -1)
        flat[:, :32 * 576].view(-1, 32, 576)[~used.to(DEV)] = fill
        flat[:, 32 * 576:].view(-1, 32, 8)[~used.to(DEV)] = 255
    else:
        poison[:, :, 0][~used.to(DEV)] = fill
    out, lse = _run(q, poison, table, n, scale, causal=True, num_sm_parts=parts)
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
    # the newest row of every request: the first query does not see it, the second has no number
    for b, m in enumerate(n.tolist()):
        page, at = int(table[b, (m - 1) // 32]), (m - 1) % 32
        if kind == "model1":
            poison.view(poison.shape[0], -1)[page, at * 576:(at + 1) * 576] = fill
        else:
            poison[page, at] = fill
    out, lse = _run(q, poison, table, n, scale, causal=True, num_sm_parts=parts)
    assert torch.equal(out[:, 0], clean[:, 0]) and torch.equal(lse[:, 0], clean_lse[:, 0])
    assert torch.isnan(out[:, 1]).all() and torch.isnan(lse[:, 1]).all()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinite_hidden_row(value):
    q, cache, table, n, scale = _case("bf16", [70], 2, 8, 64, 43)
    clean, _ = _run(q, cache, table, n, scale, causal=True)
    page, at = int(table[0, 69 // 64]), 69 % 64
    cache[page, at, 0, 100] = value
    out, _ = _run(q, cache, table, n, scale, causal=True)
    assert torch.equal(out[:, 0], clean[:, 0])


def test_pages_that_the_cache_does_not_have():
    """Entries below zero or past the cache within a request's length count as no entry."""
    q, cache, table, n, scale = _case("bf16", [300, 129], 1, 16, 32, 51)
    table[0, 2], table[0, 4], table[1, 0] = -1, cache.shape[0], -2 ** 31
    table[1, 4] = 2 ** 31 - 1
    out, lse = _run(q, cache, table, n, scale)
    P.check_attention(out, lse, q, cache, table, n, scale, False)
    table[:] = -1
    out, lse = _run(q, cache, table, n, scale)
    assert bool((out == 0).all()) and bool((lse == -1e30).all())


def test_lengths_outside_the_table():
    q, cache, table, n, scale = _case("bf16", [128, 64], 1, 16, 64, 61)
    long = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=DEV)
    out, lse = _run(q, cache, table, long, scale)
    P.check_attention(out, lse, q, cache, table, long, scale, False)


@pytest.mark.parametrize("kind", P.KINDS)
def test_strides(kind):
    """Padded pages, tables that are slices or one row for all, and a given output."""
    q, cache, table, n, scale = _case(kind, [150, 150, 150], 1, 16, 32, 71)
    wide = torch.full((3, 2 * table.shape[1] + 3), -7, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    ref, ref_lse = _run(q, cache, table, n, scale)
    P.check_attention(ref, ref_lse, q, cache, table, n, scale, False)
    out = torch.full_like(ref, 9)
    got, lse = _run(q, P.padded(cache, 64), wide[:, :table.shape[1]], n, scale, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, ref) and torch.equal(lse, ref_lse)
    shared, _ = _run(q, cache, table[:1].expand(3, -1), n, scale)
    assert torch.equal(shared[0], ref[0])
    P.check_attention(shared, _, q, cache, table[:1].expand(3, -1), n, scale, False)
    flat, flat_lse = _run(q[:, 0], cache, table, n, scale)
    assert torch.equal(flat, ref[:, 0]) and torch.equal(flat_lse, ref_lse[:, 0])


def test_nothing_to_do():
    q, cache, table, n, scale = _case("bf16", [5], 1, 16, 64, 81)
    out, lse = _run(q[:0], cache, table[:0], n[:0], scale)
    assert out.shape == (0, 1, 16, 512) and lse.shape == (0, 1, 16)
    out, lse = _run(q[:, :0], cache, table, n, scale)
    assert out.shape == (1, 0, 16, 512)
    out, lse = _run(q, cache, table[:, :0], n, scale)
    assert bool((out == 0).all()) and bool((lse == -1e30).all())
    out, lse = _run(q, cache[:0], table, n, scale)
    assert bool((out == 0).all())


def test_far_rows():
    """Rows more than 2^32 bytes from the cache's start."""
    cache = torch.empty((60000, 64, 1, 576), dtype=torch.bfloat16, device=DEV)           # 4.4 GB
    small = P.make_cache("bf16", 3, 64, 5).to(DEV)
    ids = torch.tensor([59999, 58300, 1], device=DEV)
    cache[ids] = small
    q = torch.randn(1, 16, 576, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(torch.bfloat16)
    n = torch.tensor([190], dtype=torch.int32, device=DEV)
    out, lse = _run(q, cache, ids.int().view(1, 3), n, 0.04)
    ref, ref_lse = _run(q, small, torch.arange(3, dtype=torch.int32, device=DEV).view(1, 3), n, 0.04)
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)


def test_many_requests():
    """More requests than a partition scan has threads."""
    g = torch.Generator().manual_seed(91)
    lengths = torch.randint(0, 40, (1500,), generator=g).tolist()
    q, cache, table, n, scale = _case("bf16", lengths, 1, 4, 16, 92)
    out, lse = _run(q, cache, table, n, scale)
    P.check_attention(out, lse, q, cache, table, n, scale, False)


def test_streams_and_graphs():
    """A call on a side stream, and two captured calls that replay in turn with eager ones between: no scratch is shared."""
    from sparse_mla_sm120_b200 import paged
    a = _case("bf16", [900, 700], 1, 128, 64, 101)
    b = _case("v32", [1200, 30, 400], 1, 64, 64, 102)
    ref = [_run(*x) for x in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.paged_mla_decode_fwd(*a)
        graphs, outs = [], []
        for x in (a, b):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(paged.paged_mla_decode_fwd(*x))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], ref[0][0])
    for _ in range(3):
        for o in outs:
            o[0].zero_(), o[1].zero_()
        graphs[0].replay()
        eager = paged.paged_mla_decode_fwd(*b)
        graphs[1].replay()
        torch.cuda.synchronize()
        for o, r in zip(outs + [eager], ref + [ref[1]]):
            assert torch.equal(o[0], r[0]) and torch.equal(o[1], r[1])
    # other lengths in the same buffers: the graph finds its partitions anew
    a[3][:] = torch.tensor([3, 640], dtype=torch.int32, device=DEV)
    graphs[0].replay()
    torch.cuda.synchronize()
    P.check_attention(outs[0][0], outs[0][1], *a[:4], a[4], False)


@pytest.mark.parametrize("kind", P.KINDS)
def test_a_step_through_the_flashmla_surface(kind):
    """Prompt rows appended in two chunks, then three steps: append the new token's row and query, attend over everything."""
    from sparse_mla_sm120_b200 import interface, paged
    g = torch.Generator().manual_seed(111)
    lat, dt, page, heads = P.LATENT[kind], P.DTYPE[kind], 32, 24
    cache = P.make_cache(kind, 12, page, 112).to(DEV)
    start = [70, 33]
    table = P.table_of([120, 100], page, 12, 113).to(DEV)
    cs = P.rotary_table(200).to(DEV)
    rand = lambda *s: torch.randn(*s, generator=g).to(dt).to(DEV)

    def slots(b, pos):
        return table[b].long()[pos // page] * page + pos % page
    for b, n in enumerate(start):
        for lo, hi in ((0, n // 2), (n // 2, n)):
            pos = torch.arange(lo, hi, device=DEV)
            down = rand(hi - lo, lat + 64)
            paged.append_kv_cache(down[:, :lat], down[:, lat:], cache, slots(b, pos), pos, cs)
    meta, _ = interface.get_mla_metadata()
    for step in range(3):
        lengths = torch.tensor([n + step + 1 for n in start], dtype=torch.int32, device=DEV)
        pos = lengths - 1
        down, q = rand(2, lat + 64), rand(2, 1, heads, lat + 64)
        at = torch.stack([slots(b, pos[b].long()) for b in range(2)])
        paged.append_kv_cache(down[:, :lat], down[:, lat:], cache, at, pos, cs, q_pe=rand(2, heads, 64), q_out=q[:, 0, :, lat:])
        out, lse = interface.flash_mla_with_kvcache(q, cache, table, lengths, 512, meta, causal=True, is_fp8_kvcache=kind in ("v32", "model1"))
        torch.cuda.synchronize()
        P.check_attention(out, lse.permute(0, 2, 1), q, cache, table, lengths, (lat + 64) ** -0.5, True)
        last = orc.cache_values(cache.cpu()).reshape(12 * page, -1)[at.cpu()][:, lat:]
        ref = orc.rotate_ref(down[:, lat:].cpu(), cs.cpu(), pos.cpu(), True)
        assert float((last - ref).abs().max()) <= P.HALF_STEP[dt] * float(ref.abs().max()) + 1e-5
    with pytest.raises(ValueError, match="initialised"):
        interface.flash_mla_with_kvcache(q[:1], cache, table[:1], lengths[:1], 512, meta, causal=True, is_fp8_kvcache=kind in ("v32", "model1"))


def test_an_indexed_step_on_appended_caches():
    """Keys, rows and queries appended, then indexer -> top-k -> attention: with a list as long as the context, the same as attention over
    everything, within the FP8-class kernels' bounds."""
    import helpers as H
    from sparse_mla_sm120_b200 import paged, pipeline
    g = torch.Generator().manual_seed(121)
    context, heads, ih, tokens = 512, 64, 32, 4
    cs = P.rotary_table(context).to(DEV)
    cache = torch.zeros(8, 64, 1, 656, dtype=torch.uint8, device=DEV)
    ki, ks = torch.zeros(context, 128, device=DEV).to(torch.float8_e4m3fn), torch.zeros(context, device=DEV)
    bf = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)
    pos = torch.arange(context, device=DEV)
    table = torch.randperm(8, generator=g).int().to(DEV)
    rows = table.long()[pos // 64] * 64 + pos % 64
    down = bf(context, 576)
    paged.append_kv_cache(down[:, :512], down[:, 512:], cache, rows, pos, cs)
    q = 0.5 * bf(tokens, heads, 576)
    qi, w = paged.append_indexer_keys(bf(context, 128), ki, ks, pos, pos, cs, q=bf(context, ih, 128), weights=torch.rand(context, ih, generator=g).to(DEV))
    qi, w = qi[-tokens:].contiguous(), w[-tokens:].contiguous()
    lo = torch.zeros(tokens, dtype=torch.int32, device=DEV)
    hi = torch.full((tokens,), context, dtype=torch.int32, device=DEV)
    out, lse, picked = pipeline.sparse_mla_indexed_decode_fwd(q, cache, qi, ki, ks, w, lo, hi, 576 ** -0.5, topk=context,
                                                              block_table=table.view(1, -1).expand(tokens, -1).contiguous())
    assert torch.equal(picked.sort(dim=1).values.long(), torch.arange(context, device=DEV).expand(tokens, -1))
    dense, dense_lse = _run(q, cache, table.view(1, -1).expand(tokens, -1), hi, 576 ** -0.5)
    P.check_attention(dense.unsqueeze(1), dense_lse.unsqueeze(1), q.unsqueeze(1), cache, table.view(1, -1).expand(tokens, -1), hi, 576 ** -0.5, False)
    H.compare_out(out.cpu(), dense.cpu(), H.TC_ABS, H.TC_REL, H.TC_COS)
    assert float((lse - dense_lse).abs().max()) <= H.TC_LSE * 1.45
