"""paged_mla_decode_fwd of more than 64 query rows per request over 16-bit caches, which runs on pairs of SMs: what test_gpu_paged.py asks at
fewer rows."""
import pytest
import torch

import paged_cases as P
from oracle import sparse_mla_oracle as orc
from test_gpu_paged import _case, _run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = ("bf16", "fp16")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths,s_q,heads,page,causal", [
    ([1], 1, 65, 64, False),                              # the second CTA of the pair has one query row
    ([0, 1, 127, 128, 129, 255, 256, 257], 1, 128, 64, False),
    ([500, 0, 0, 17, 0, 1000, 2], 1, 96, 64, True),
    ([130, 1, 0, 3], 3, 43, 64, True),                    # 129 query rows: the second pair has one
    ([300, 70], 5, 128, 128, True),
    ([333, 100], 2, 64, 16, True),                        # pages that end inside a block
    ([100, 333], 1, 80, 48, False),
    ([150, 9], 2, 65, 130, True),
    ([65, 130], 1, 72, 1, False),
    ([200], 1, 72, 3, False),
    ([3000, 1500], 1, 128, 64, False),
])
def test_attention(kind, lengths, s_q, heads, page, causal):
    q, cache, table, n, scale = _case(kind, lengths, s_q, heads, page, len(lengths) * 100 + heads)
    sink = torch.randn(heads, device=DEV, generator=torch.Generator(device=DEV).manual_seed(heads)) if heads % 2 else None
    out, lse = _run(q, cache, table, n, scale, causal=causal, attn_sink=sink)
    P.check_attention(out, lse, q, cache, table, n, scale, causal, sink)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parts", [1, 2, 5, 9, 74, 200])
def test_partitions(kind, parts):
    q, cache, table, n, scale = _case(kind, [1700, 3, 0, 1300, 128, 129], 2, 70, 64, 11)
    out, lse = _run(q, cache, table, n, scale, num_sm_parts=parts, causal=True)
    P.check_attention(out, lse, q, cache, table, n, scale, True)
    again, _ = _run(q, cache, table, n, scale, num_sm_parts=parts, causal=True)
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sign", [4.0, -4.0, 0.0])
def test_peaked_scores(kind, sign):
    """Scores that grow along the rows, of either sign of the scale, and a scale of nothing."""
    q, cache, table, n, scale = _case(kind, [1280], 1, 96, 64, 31, spare=0, std=0.2)
    rows = orc.cache_values(cache.cpu())[table.cpu()[0].long()].reshape(1280, -1)
    q = (rows[[1279, 5, 300, 128, 640, 1000] * 16] * 6).view(1, 1, 96, -1).to(q.dtype).to(DEV)
    out, lse = _run(q, cache, table, n, scale * sign)
    P.check_attention(out, lse, q, cache, table, n, scale * sign, False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s_q,heads", [(2, 48), (3, 128)])
@pytest.mark.parametrize("parts", [1, 5])
def test_what_is_not_seen_does_not_matter(kind, s_q, heads, parts):
    """No-number bytes behind the rows of a request, in pages that it does not have, and in the rows that a query must not see."""
    q, cache, table, n, scale = _case(kind, [258, 129, 40], s_q, heads, 32, 41, width=12)
    clean, clean_lse = _run(q, cache, table, n, scale, causal=True, num_sm_parts=parts)
    P.check_attention(clean, clean_lse, q, cache, table, n, scale, True)
    used = torch.zeros(cache.shape[0], 32, dtype=torch.bool)
    for b, m in enumerate(n.tolist()):
        for j in range(m):
            used[int(table[b, j // 32]), j % 32] = True
    poison = cache.clone()
    poison[:, :, 0][~used.to(DEV)] = float("nan")
    out, lse = _run(q, poison, table, n, scale, causal=True, num_sm_parts=parts)
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
    # the newest row of every request: only the last query sees it
    for b, m in enumerate(n.tolist()):
        poison[int(table[b, (m - 1) // 32]), (m - 1) % 32] = float("nan")
    out, lse = _run(q, poison, table, n, scale, causal=True, num_sm_parts=parts)
    assert torch.equal(out[:, :-1], clean[:, :-1]) and torch.equal(lse[:, :-1], clean_lse[:, :-1])
    assert torch.isnan(out[:, -1]).all() and torch.isnan(lse[:, -1]).all()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinite_hidden_row(value):
    q, cache, table, n, scale = _case("bf16", [130], 2, 64, 64, 43)
    clean, _ = _run(q, cache, table, n, scale, causal=True)
    page, at = int(table[0, 129 // 64]), 129 % 64
    cache[page, at, 0, 100] = value
    out, _ = _run(q, cache, table, n, scale, causal=True)
    assert torch.equal(out[:, 0], clean[:, 0])


def test_pages_that_the_cache_does_not_have():
    q, cache, table, n, scale = _case("bf16", [300, 129], 1, 100, 32, 51)
    table[0, 2], table[0, 4], table[1, 0] = -1, cache.shape[0], -2 ** 31
    table[1, 4] = 2 ** 31 - 1
    out, lse = _run(q, cache, table, n, scale)
    P.check_attention(out, lse, q, cache, table, n, scale, False)
    table[:] = -1
    out, lse = _run(q, cache, table, n, scale)
    assert bool((out == 0).all()) and bool((lse == -1e30).all())


def test_an_output_on_16_bytes_and_padded_pages():
    q, cache, table, n, scale = _case("bf16", [150, 260], 1, 128, 32, 71)
    ref, ref_lse = _run(q, cache, table, n, scale)
    room = torch.full((ref.numel() + 16,), 9, dtype=ref.dtype, device=DEV)
    out = room[8:8 + ref.numel()].view(ref.shape)
    got, lse = _run(q, P.padded(cache, 64), table, n, scale, out=out)
    assert torch.equal(got, ref) and torch.equal(lse, ref_lse)
    assert bool((room[:8] == 9).all()) and bool((room[8 + ref.numel():] == 9).all())


def test_pairs_give_what_single_sms_give():
    """The same queries in two calls of 64 heads, and in one of 128: the same within the roundings of weights and outputs."""
    q, cache, table, n, scale = _case("bf16", [900, 64, 2000], 1, 128, 64, 81)
    both, both_lse = _run(q, cache, table, n, scale)
    halves = [_run(q[:, :, i:i + 64].contiguous(), cache, table, n, scale) for i in (0, 64)]
    for i, (out, lse) in enumerate(halves):
        P.check_attention(out, lse, q[:, :, 64 * i:64 * i + 64], cache, table, n, scale, False)
        assert float((both_lse[:, :, 64 * i:64 * i + 64] - lse).abs().max()) <= 2.0 ** -14


def test_far_rows():
    """Rows more than 2^32 bytes from the cache's start."""
    cache = torch.empty((60000, 64, 1, 576), dtype=torch.bfloat16, device=DEV)           # 4.4 GB
    small = P.make_cache("bf16", 3, 64, 5).to(DEV)
    ids = torch.tensor([59999, 58300, 1], device=DEV)
    cache[ids] = small
    q = torch.randn(1, 128, 576, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(torch.bfloat16)
    n = torch.tensor([190], dtype=torch.int32, device=DEV)
    out, lse = _run(q, cache, ids.int().view(1, 3), n, 0.04)
    ref, ref_lse = _run(q, small, torch.arange(3, dtype=torch.int32, device=DEV).view(1, 3), n, 0.04)
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)


def test_many_requests():
    """More requests than a partition scan has threads."""
    g = torch.Generator().manual_seed(91)
    lengths = torch.randint(0, 40, (1200,), generator=g).tolist()
    q, cache, table, n, scale = _case("bf16", lengths, 1, 66, 16, 92)
    out, lse = _run(q, cache, table, n, scale)
    P.check_attention(out, lse, q, cache, table, n, scale, False)


@pytest.mark.parametrize("heads", [16, 128])
def test_a_scale_that_is_no_number(heads):
    q, cache, table, n, _ = _case("bf16", [70, 0], 1, heads, 64, 101)
    out, lse = _run(q, cache, table, n, float("nan"))
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert bool((out[1] == 0).all()) and bool((lse[1] == -1e30).all())


@pytest.mark.parametrize("kind", KINDS)
def test_a_captured_step(kind):
    """Appends and attention of 128 heads as one graph that replays over growing contexts."""
    from sparse_mla_sm120_b200 import paged
    g = torch.Generator().manual_seed(111)
    dt, page, heads, steps = P.DTYPE[kind], 64, 128, 4
    cache = P.make_cache(kind, 14, page, 112).to(DEV)
    lengths = torch.tensor([509, 127], dtype=torch.int32, device=DEV)
    table = P.table_of([520, 140], page, 14, 113).to(DEV)
    cs = P.rotary_table(600).to(DEV)
    rand = lambda *s: torch.randn(*s, generator=g).to(dt).to(DEV)
    down, q, q_pe = rand(2, 576), rand(2, 1, heads, 576), rand(2, heads, 64)
    slots, pos = torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)

    def step():
        paged.append_kv_cache(down[:, :512], down[:, 512:], cache, slots, pos, cs, q_pe=q_pe, q_out=q[:, 0, :, 512:])
        return paged.paged_mla_decode_fwd(q, cache, table, lengths, 576 ** -0.5)

    def place():
        pos.copy_(lengths - 1)
        slots.copy_(table.long().gather(1, (pos // page).unsqueeze(1)).squeeze(1) * page + pos % page)
    place()
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out, lse = step()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(steps):
        lengths += 1
        place()
        for buffer in (down, q, q_pe):
            buffer.copy_(torch.randn(buffer.shape, generator=g).to(dt))
        graph.replay()
        torch.cuda.synchronize()
        P.check_attention(out, lse, q, cache, table, lengths, 576 ** -0.5, False)
        turned = orc.rotate_ref(q_pe.cpu(), cs.cpu(), pos.cpu(), True)
        assert float((q[:, 0, :, 512:].cpu().double() - turned).abs().max()) <= P.HALF_STEP[dt] * float(turned.abs().max()) + 1e-5
