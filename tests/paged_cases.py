"""Inputs and error bounds shared by the tests of paged.py."""
import torch

import helpers as H
from oracle import sparse_mla_oracle as orc

KINDS = ("bf16", "fp16", "v32", "model1")
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "v32": torch.bfloat16, "model1": torch.bfloat16}
LATENT = {"bf16": 512, "fp16": 512, "v32": 512, "model1": 448}
ROW = {"bf16": 576, "fp16": 576, "v32": 656, "model1": 584}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # of a rounding, relative to the value


def make_cache(kind, pages, page, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, page, 1, LATENT[kind] + 64, generator=g) * std
    if kind in ("bf16", "fp16"):
        return x.to(DTYPE[kind])
    return (orc.quantize_kv_v32 if kind == "v32" else orc.quantize_kv_model1)(x.to(torch.bfloat16))


def padded(cache, pad):
    """The same pages, further apart: `pad` elements of something else between them."""
    n = cache[0].numel()
    room = torch.full((cache.shape[0], n + pad), 0x7f if cache.dtype == torch.uint8 else float("nan"), dtype=cache.dtype, device=cache.device)
    view = room[:, :n].view(cache.shape)
    view.copy_(cache)
    return view


def table_of(lengths, page, pages, seed, width=None):
    """A block table whose requests own shuffled pages; what lies behind a request's pages names none."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lengths]
    assert sum(need) <= pages
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), width or max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def check_attention(out, lse, q, cache, table, lengths, scale, causal, sink=None):
    """Bounds from the roundings, none of them fitted.  With w = 2^-8 (bf16) or 2^-11 (fp16) half a step relative to the value:
    output rounding w |out|; weights rounded before their product with V: w sum p |v|; fp16 weights of less than 2^-14 are off by 2^-25 each,
    where the largest is at least 1: 2^-25 n max |v|; the scores' fp32 sums of d products, each step off by at most 2^-23 of the sum of
    sizes, change a weight by d 2^-23 S, S = scale max sum |q k|, in numerator and denominator; exponentials 2^-21 each; sums over n
    rows 2^-23 n; the merge and the division 2^-20."""
    ref, ref_lse, size, spread, seen = orc.paged_attn_ref(q.cpu(), cache.cpu(), table.cpu(), lengths.cpu(), scale, causal,
                                                          None if sink is None else sink.cpu())
    w = HALF_STEP[q.dtype]
    n = seen.double().unsqueeze(-1)
    soft = q.shape[-1] * 2.0 ** -23 * spread + 2.0 ** -21 + n * 2.0 ** -23 + 2.0 ** -20        # of a weight, and of the denominator
    tiny = 2.0 ** -25 * n * float(size.max()) * 4 if q.dtype == torch.float16 else 0 * n       # (4: the largest |v| against the mean |v|)
    bound = w * ref.abs() + (w + 2 * soft).unsqueeze(-1) * size * (1 + w) + tiny.unsqueeze(-1) + 1e-30
    d = (out.cpu().double() - ref).abs()
    assert torch.isfinite(out).all(), "not finite"
    assert bool((d <= bound).all()), f"output off by {float((d / bound).max())} of its bound"
    nothing = ref_lse == -1e30
    assert torch.equal(lse.cpu() == -1e30, nothing), "rows that see nothing"
    inf = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse.cpu()), inf)
    fine = ~nothing & ~inf
    d = (lse.cpu().double() - ref_lse).abs()[fine]
    lse_bound = (2 * soft * 1.45 + 2.0 ** -22 * ref_lse.abs())[fine]
    assert bool((d <= lse_bound).all()), f"LSE off by {float((d / lse_bound).max())} of its bound"


def rotary_table(positions, seed=None):
    inv = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    a = torch.arange(positions, dtype=torch.float64).unsqueeze(1) * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def rows_of(cache, kind):
    """(latent bytes, scales, rotated values) of every row, [pages * page, ...]."""
    pages, page = cache.shape[:2]
    if kind in ("bf16", "fp16"):
        c = cache.reshape(pages * page, 576)
        return c[:, :512], c[:, :0], c[:, 512:]
    c = cache.contiguous()
    if kind == "v32":
        c = c.view(pages * page, 656)
        return c[:, :512], c[:, 512:528], c[:, 528:].contiguous().view(torch.bfloat16)
    flat = c.view(pages, page * 584)
    data, footer = flat[:, :page * 576].reshape(-1, 576), flat[:, page * 576:].reshape(-1, 8)
    return data[:, :448], footer, data[:, 448:].contiguous().view(torch.bfloat16)


__all__ = [n for n in dir() if not n.startswith("_")]
