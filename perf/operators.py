"""What a decode step does around the sparse attention: the rows it adds to the caches, and attention over a whole context.

    append   latent rows of new tokens into a paged cache, the positional part rotated on the way, the queries' too
    index    the indexer's keys of new tokens into its cache, and its queries: rotated, then e4m3 with a scale
    attend   attention of the newest tokens of every request over all of its rows, through a block table

Plain forms (`own` false) and the framework's calls (`own` true) take the same inputs.  Caches: rows of 576 bf16 or fp16 values;
656 bytes (512 e4m3 | 4 fp32 scales | 64 bf16); 584 bytes (448 e4m3 | 64 bf16, scales as exponents behind a page's rows).
"""
import math

import torch

own = False

DEVICE = "cuda"
LATENT = {"bf16": 512, "fp16": 512, "v32": 512, "model1": 448}      # values of a row before its 64 rotated ones
ROW_BYTES = {"bf16": 1152, "fp16": 1152, "v32": 656, "model1": 584}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "v32": torch.bfloat16, "model1": torch.bfloat16}
NEVER = -1e30                                                       # LSE of a row that sees nothing


def listed():
    return [
        # One request's next token: its whole latency is what counts.
        dict(name="append_one_token", kind="append", cache="v32", tokens=1, heads=128, page=64, interleaved=True, prompt=False),
        # A running batch, padded, over 16-bit rows; heads split over two GPUs.
        dict(name="append_batch", kind="append", cache="bf16", tokens=129, heads=64, page=64, interleaved=True, prompt=False),
        # A prompt's chunk into the 584-byte layout, halves rotated against each other.
        dict(name="append_chunk_model1", kind="append", cache="model1", tokens=2047, heads=64, page=64, interleaved=False, prompt=True),
        # The largest chunk, all heads on one GPU.
        dict(name="append_chunk_v32", kind="append", cache="v32", tokens=8192, heads=128, page=64, interleaved=True, prompt=True),
        # A decode batch's keys and queries of the indexer.
        dict(name="index_batch", kind="index", tokens=16, heads=64, interleaved=False, offset=0, prompt=False),
        # A prompt's chunk of them.
        dict(name="index_chunk", kind="index", tokens=4096, heads=64, interleaved=True, offset=64, prompt=True),
        # One request in the middle of a conversation, heads split over eight GPUs.
        dict(name="attend_short", kind="attend", cache="bf16", requests=1, s_q=1, heads=16, context=1000, page=64, sink=False),
        # One request with a very long context on one GPU.
        dict(name="attend_long", kind="attend", cache="bf16", requests=1, s_q=1, heads=128, context=131072, page=64, sink=False),
        # The serving batch, contexts of very different lengths.
        dict(name="attend_batch", kind="attend", cache="bf16", requests=64, s_q=1, heads=128, context=8192, page=64, sink=False),
        # Two tokens per request (one of them speculative), few heads, small pages.
        dict(name="attend_two_tokens", kind="attend", cache="fp16", requests=48, s_q=2, heads=16, context=4096, page=16, sink=False),
        # The cache that the sparse attention reads, with sinks.
        dict(name="attend_v32", kind="attend", cache="v32", requests=64, s_q=1, heads=64, context=8192, page=64, sink=True),
        # The same for the other packed layout, a small batch.
        dict(name="attend_model1", kind="attend", cache="model1", requests=13, s_q=1, heads=128, context=16384, page=64, sink=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "index", "attend", "attend", "attend"])
    if kind == "append":
        return dict(kind=kind, cache=rng.choice(["bf16", "fp16", "v32", "v32", "model1"]), tokens=_log_int(rng, 1, 8192),
                    heads=rng.choice([8, 16, 40, 64, 128]), page=rng.choice([16, 32, 64, 64]), interleaved=rng.random() < 0.7,
                    prompt=rng.random() < 0.5)
    if kind == "index":
        return dict(kind=kind, tokens=_log_int(rng, 1, 4096), heads=rng.choice([32, 64, 64]), interleaved=rng.random() < 0.5,
                    offset=rng.choice([0, 64]), prompt=rng.random() < 0.5)
    requests = _log_int(rng, 1, 96)
    context = _log_int(rng, 32, min(131072, 524288 // requests))
    return dict(kind=kind, cache=rng.choice(["bf16", "bf16", "fp16", "v32", "v32", "model1"]), requests=requests,
                s_q=rng.choice([1, 1, 1, 2, 3]), heads=rng.choice([8, 16, 24, 32, 64, 64, 128]), context=context,
                page=rng.choice([16, 64, 64, 64, 128]), sink=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _table(positions):
    """cos and sin of 32 angles per position (base 10000), computed in 64 bits: [positions, cos 32 | sin 32] fp32."""
    inv = 10000.0 ** (-torch.arange(32, device=DEVICE, dtype=torch.float64) / 32)
    a = torch.arange(positions, device=DEVICE, dtype=torch.float64).unsqueeze(1) * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _views(cache, kind):
    """The parts of a cache as the values they stand for (views of its memory)."""
    if kind in ("bf16", "fp16"):
        return (cache,)
    if kind == "v32":
        return cache[..., :512].view(torch.float8_e4m3fn), cache[..., 512:528].view(torch.float32), cache[..., 528:].view(torch.bfloat16)
    pages, page = cache.shape[:2]
    flat = cache.view(pages, page * 584)
    data, footer = flat[:, :page * 576].view(pages, page, 576), flat[:, page * 576:].view(pages, page, 8)
    return data[..., :448].view(torch.float8_e4m3fn), footer[..., :7].view(torch.float8_e8m0fnu), data[..., 448:].view(torch.bfloat16)


def _pool(g, kind, pages, page):
    """A cache with rows in it: unit noise around a mean per channel, as a trained projection leaves them."""
    lat = LATENT[kind]
    if kind in ("bf16", "fp16"):
        cache = torch.empty((pages, page, 1, 576), dtype=DTYPE[kind], device=DEVICE)
        offset = 0.5 * _randn(g, 576)
        for p in range(0, pages, 2048):
            n = min(2048, pages - p)
            cache[p:p + n] = (_randn(g, n, page, 1, 576) + offset).to(cache.dtype)
        return cache
    cache = torch.zeros((pages, page, 1, ROW_BYTES[kind]), dtype=torch.uint8, device=DEVICE)
    nope, scales, rope = _views(cache, kind)
    offset = 0.5 * _randn(g, lat)
    for p in range(0, pages, 2048):
        n = min(2048, pages - p)
        shape = (n, page, 1) if kind == "v32" else (n, page)
        nope.view(torch.uint8)[p:p + n] = ((_randn(g, *shape, lat) + offset) * 80).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        rope[p:p + n] = _randn(g, *shape, 64).to(torch.bfloat16)
        e = torch.randint(119, 122, shape + (scales.shape[-1],), device=DEVICE, generator=g)     # 2^-8 to 2^-6
        if kind == "v32":
            scales[p:p + n] = (e - 127).float().exp2()
        else:
            scales.view(torch.uint8)[p:p + n] = e.to(torch.uint8)
    return cache


def _slots(g, tokens, capacity, page, prompt):
    """Distinct rows of the cache: a prompt's run through shuffled pages, or one row of each request; a batch is padded (-1)."""
    if prompt:
        pages = torch.randperm(capacity // page, device=DEVICE, generator=g)
        at = torch.arange(tokens, device=DEVICE) + page // 2
        return pages[at // page] * page + at % page
    slots = torch.randperm(capacity, device=DEVICE, generator=g)[:tokens]
    if tokens >= 8:
        slots[-(tokens // 8):] = -1
    return slots


def _lengths(case):
    """Rows of each request: spread evenly between an eighth of the context and all of it."""
    n, c = case["requests"], case["context"]
    return [c] if n == 1 else [max(c // 8 + (c - c // 8) * i // (n - 1), 1) for i in range(n)]


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind in ("append", "index"):
        t, h = case["tokens"], case["heads"]
        capacity = -(-max(2 * t, 4096) // 64) * 64
        s["table"] = _table(16384)
        first = int(torch.randint(0, 8192, (1,), generator=g, device=DEVICE))
        s["positions"] = first + torch.arange(t, device=DEVICE) if case["prompt"] else torch.randint(0, 16384, (t,), device=DEVICE, generator=g)
    if kind == "append":
        s["slots"] = _slots(g, t, capacity, case["page"], case["prompt"])
        dt, lat = DTYPE[case["cache"]], LATENT[case["cache"]]
        s["cache"] = _pool(g, case["cache"], capacity // case["page"], case["page"])
        s["views"] = _views(s["cache"], case["cache"])
        down = (_randn(g, t, lat + 64) * (0.2 + 3 * torch.rand((t, 1), device=DEVICE, generator=g))).to(dt)    # the down projection's output
        s["kv_c"], s["k_pe"] = down[:, :lat], down[:, lat:]
        s["q_pe"] = _randn(g, t, h, 192).to(dt)[..., 128:]                           # the last 64 of a head's 192 query values
        s["q"] = _randn(g, t, h, lat + 64).to(dt)                                    # the absorbed query; its last 64 are written
        s["q_out"] = s["q"][..., lat:]
    elif kind == "index":
        s["slots"] = _slots(g, t, capacity, 64, case["prompt"])
        s["k"] = (2 * _randn(g, t, 128)).to(torch.bfloat16)
        s["q"] = (2 * _randn(g, t, h, 128)).to(torch.bfloat16)
        s["weights"] = 0.1 * _randn(g, t, h)
        s["ki"] = (100 * _randn(g, capacity, 128)).clamp(-448, 448).to(torch.float8_e4m3fn)
        s["k_scale"] = 0.01 + 0.01 * torch.rand(capacity, device=DEVICE, generator=g)
    else:
        page, n = case["page"], case["requests"]
        lengths = torch.tensor(_lengths(case), device=DEVICE, dtype=torch.int32)
        s["lengths"] = lengths[torch.randperm(n, device=DEVICE, generator=g)]
        owned = (s["lengths"] + page - 1) // page
        pages = int(owned.sum()) + 1
        s["cache"] = _pool(g, case["cache"], pages, page)
        order = torch.randperm(pages, device=DEVICE, generator=g).to(torch.int32)
        at = torch.arange(-(-case["context"] // page), device=DEVICE)
        mine = (owned.cumsum(0) - owned).unsqueeze(1) + at
        s["block_table"] = torch.where(at < owned.unsqueeze(1), order[mine.clamp(max=pages - 1)], -1).to(torch.int32)
        d = LATENT[case["cache"]] + 64
        s["q"] = (0.5 * _randn(g, n, case["s_q"], case["heads"], d)).to(DTYPE[case["cache"]])
        s["sink"] = _randn(g, case["heads"]) if case["sink"] else None
        s["scale"] = d ** -0.5
    return s


# ------------------------------------------------------------------ plain forms
def _rotated(x, table, positions, interleaved):
    """x [T, ..., 64] in 32 bits, each pair turned by its angle at the token's position."""
    cs = table[positions].view(x.shape[0], *([1] * (x.dim() - 2)), 64)
    c, s, x = cs[..., :32], cs[..., 32:], x.float()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :32], x[..., 32:])
    u, v = a * c - b * s, b * c + a * s
    return torch.stack([u, v], dim=-1).flatten(-2) if interleaved else torch.cat([u, v], dim=-1)


def _quantised(x, group):
    """(e4m3 values, power-of-two scales): one scale, rounded up, per `group` values of the last dimension."""
    x = x.float().unflatten(-1, (-1, group))
    most = x.abs().amax(dim=-1).clamp(min=1e-4)
    scale = (most / torch.full_like(most, 448)).clamp(min=1e-4)       # by a tensor: a number's reciprocal would miss powers of two
    mantissa, exponent = torch.frexp(scale)
    scale = torch.ldexp(torch.ones_like(scale), torch.where(mantissa == 0.5, exponent - 1, exponent))
    return (x / scale.unsqueeze(-1)).clamp(-448, 448).flatten(-2).to(torch.float8_e4m3fn), scale


def _plain_append(s):
    case = s["case"]
    kind, page, table, positions, pairs = case["cache"], case["page"], s["table"], s["positions"], case["interleaved"]
    k_pe = _rotated(s["k_pe"], table, positions, pairs).to(DTYPE[kind])
    s["q_out"].copy_(_rotated(s["q_pe"], table, positions, pairs))
    keep = s["slots"] >= 0
    row = s["slots"][keep]
    at = (row // page, row % page)
    if kind in ("bf16", "fp16"):
        s["cache"][at[0], at[1], 0] = torch.cat([s["kv_c"], k_pe], dim=1)[keep]
    elif kind == "v32":
        values, scale = _quantised(s["kv_c"], 128)
        packed = torch.cat([values.view(torch.uint8), scale.view(torch.uint8), k_pe.view(torch.uint8)], dim=1)
        s["cache"][at[0], at[1], 0] = packed[keep]
    else:
        values, scale = _quantised(s["kv_c"], 64)
        pages = s["cache"].shape[0]
        flat = s["cache"].view(pages, page * 584)
        data, footer = flat[:, :page * 576].view(pages, page, 576), flat[:, page * 576:].view(pages, page, 8)
        data[at] = torch.cat([values.view(torch.uint8), k_pe.view(torch.uint8)], dim=1)[keep]
        exponent = (scale.view(torch.int32) >> 23).to(torch.uint8)
        footer[at] = torch.cat([exponent, torch.zeros_like(exponent[:, :1])], dim=1)[keep]
    return s["views"], s["q"]


def _plain_index_rows(x, table, positions, interleaved, offset):
    rotated = _rotated(x[..., offset:offset + 64], table, positions, interleaved)
    x = torch.cat([rotated, x[..., 64:].float()] if offset == 0 else [x[..., :64].float(), rotated], dim=-1)
    most = x.abs().amax(dim=-1).clamp(min=1e-4)
    scale = most / torch.full_like(most, 448)
    return (x / scale.unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _plain_index(s):
    case = s["case"]
    how = (s["table"], s["positions"], case["interleaved"], case["offset"])
    k, k_scale = _plain_index_rows(s["k"], *how)
    keep = s["slots"] >= 0
    row = s["slots"][keep]
    s["ki"].view(torch.uint8)[row] = k.view(torch.uint8)[keep]
    s["k_scale"][row] = k_scale[keep]
    q, q_scale = _plain_index_rows(s["q"], *how)
    return s["ki"], s["k_scale"], q, s["weights"] * q_scale


def _plain_attend(s):
    case = s["case"]
    kind, page, n, s_q, h = case["cache"], case["page"], case["requests"], case["s_q"], case["heads"]
    pos = torch.arange(case["context"], device=DEVICE)
    at = (s["block_table"].clamp(min=0)[:, pos // page].long(), (pos % page).expand(n, -1))
    if kind in ("bf16", "fp16"):
        k = s["cache"][at[0], at[1], 0].float()
        v = k[..., :512]
    elif kind == "v32":
        rows = s["cache"][at[0], at[1], 0]
        lat = rows[..., :512].view(torch.float8_e4m3fn).float().unflatten(-1, (4, 128)) * rows[..., 512:528].contiguous().view(torch.float32).unsqueeze(-1)
        k = torch.cat([lat.flatten(-2), rows[..., 528:].contiguous().view(torch.bfloat16).float()], dim=-1)
        v = k[..., :512]
    else:
        pages = s["cache"].shape[0]
        flat = s["cache"].view(pages, page * 584)
        rows = flat[:, :page * 576].view(pages, page, 576)[at]
        scale = (flat[:, page * 576:].view(pages, page, 8)[at][..., :7].float() - 127).exp2()
        lat = rows[..., :448].view(torch.float8_e4m3fn).float().unflatten(-1, (7, 64)) * scale.unsqueeze(-1)
        k = v = torch.cat([lat.flatten(-2), rows[..., 448:].contiguous().view(torch.bfloat16).float()], dim=-1)
    scores = torch.matmul(s["q"].float().view(n, s_q * h, -1), k.transpose(1, 2)) * s["scale"]
    last = s["lengths"].unsqueeze(1) - s_q + 1 + torch.arange(s_q, device=DEVICE)               # rows that a token sees
    seen = (pos < last.unsqueeze(-1)).unsqueeze(2).expand(n, s_q, h, -1).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    p = (scores - most.masked_fill(most == -math.inf, 0)).exp()
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v).view(n, s_q, h, 512)
    total, most = total.view(n, s_q, h), most.view(n, s_q, h)
    if s["sink"] is not None:
        total = total + (s["sink"] - most).exp()
    out = torch.where(total.unsqueeze(-1) > 0, out / total.unsqueeze(-1), 0).to(s["q"].dtype)
    return out, torch.where(total > 0, total.log2() + most * math.log2(math.e), NEVER)


def run(s):
    case = s["case"]
    if own:
        from sparse_mla_sm120_b200 import paged
        if case["kind"] == "append":
            paged.append_kv_cache(s["kv_c"], s["k_pe"], s["cache"], s["slots"], s["positions"], s["table"],
                                  interleaved=case["interleaved"], q_pe=s["q_pe"], q_out=s["q_out"])
            return s["views"], s["q"]
        if case["kind"] == "index":
            q, w = paged.append_indexer_keys(s["k"], s["ki"], s["k_scale"], s["slots"], s["positions"], s["table"],
                                             interleaved=case["interleaved"], rope_offset=case["offset"], q=s["q"], weights=s["weights"])
            return s["ki"], s["k_scale"], q, w
        return paged.paged_mla_decode_fwd(s["q"], s["cache"], s["block_table"], s["lengths"], s["scale"], causal=True, attn_sink=s["sink"])
    if case["kind"] == "append":
        return _plain_append(s)
    return _plain_index(s) if case["kind"] == "index" else _plain_attend(s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "append":
        t, kept = case["tokens"], case["tokens"] - (0 if case["prompt"] or case["tokens"] < 8 else case["tokens"] // 8)
        return {"bytes": kept * (2 * LATENT[case["cache"]] + 128 + ROW_BYTES[case["cache"]]) + t * (256 + 16 + case["heads"] * 256), "flops": 0}
    if kind == "index":
        t, kept = case["tokens"], case["tokens"] - (0 if case["prompt"] or case["tokens"] < 8 else case["tokens"] // 8)
        return {"bytes": kept * (256 + 132) + t * (256 + 16 + case["heads"] * (256 + 128 + 8)), "flops": 0}
    rows, r, d = sum(_lengths(case)), case["s_q"] * case["heads"], LATENT[case["cache"]] + 64
    io = case["requests"] * (r * (2 * d + 2 * 512 + 4) + 4) + sum(-(-n // case["page"]) for n in _lengths(case)) * 4
    return {"bytes": rows * ROW_BYTES[case["cache"]] + io, "flops": 2 * r * rows * (d + 512)}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _turned(x, table, positions, interleaved):
    x, out = x.double(), torch.empty(x.shape, dtype=torch.float64, device=x.device)
    shape = (-1,) + (1,) * (x.dim() - 2)
    for i in range(32):
        c, s = (table[positions, i + j].double().view(shape) for j in (0, 32))
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 32)
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def _to_e4m3(x):
    """The nearest e4m3 value (ties to even) of 64-bit numbers of at most 448, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_append(s):
    case = s["case"]
    kind, lat = case["cache"], LATENT[case["cache"]]
    parts = [v.double() for v in s["views"]]
    k_pe = _turned(s["k_pe"], s["table"], s["positions"], case["interleaved"])
    q = s["q"].double()
    q[..., lat:] = _turned(s["q_pe"], s["table"], s["positions"], case["interleaved"])
    kept = torch.nonzero(s["slots"] >= 0).squeeze(1)
    row = s["slots"][kept]
    x = s["kv_c"].double()[kept]
    p, o = row // case["page"], row % case["page"]
    if kind in ("bf16", "fp16"):
        parts[0][p, o, 0, :512], parts[0][p, o, 0, 512:] = x, k_pe[kept]
        return tuple(parts), q
    group = 128 if kind == "v32" else 64
    at = (p, o, 0) if kind == "v32" else (p, o)
    values, scales = torch.empty_like(x), x.new_empty((x.shape[0], lat // group))
    for i in range(lat // group):
        part = x[:, i * group:(i + 1) * group]
        most = part.abs().max(dim=1).values.clamp(min=1e-4)
        power = torch.exp2(torch.floor(torch.log2(torch.maximum(most / 448, most.new_tensor(1e-4)))))      # one of these two: the
        scales[:, i] = torch.where(torch.maximum(most, most.new_tensor(448e-4)) <= 448 * power, power, 2 * power)    # products are exact
        values[:, i * group:(i + 1) * group] = _to_e4m3(part / scales[:, i:i + 1])
    parts[0][at], parts[1][at], parts[2][at] = values, scales, k_pe[kept]
    return tuple(parts), q


def _exact_index(s):
    case = s["case"]

    def rows(x):
        o = case["offset"]
        y = x.double()
        y[..., o:o + 64] = _turned(x[..., o:o + 64], s["table"], s["positions"], case["interleaved"])
        scale = y.abs().max(dim=-1).values.clamp(min=1e-4) / 448
        return _to_e4m3(y / scale.unsqueeze(-1)), scale
    ki, k_scale = s["ki"].double(), s["k_scale"].double()
    kept = torch.nonzero(s["slots"] >= 0).squeeze(1)
    k, ks = rows(s["k"])
    ki[s["slots"][kept]], k_scale[s["slots"][kept]] = k[kept], ks[kept]
    q, qs = rows(s["q"])
    return ki, k_scale, q, s["weights"].double() * qs


def _exact_attend(s):
    case = s["case"]
    page, s_q, h = case["page"], case["s_q"], case["heads"]
    views = _views(s["cache"], case["cache"])
    out = torch.zeros((case["requests"], s_q, h, 512), dtype=torch.float64, device=DEVICE)
    lse = torch.full((case["requests"], s_q, h), NEVER, dtype=torch.float64, device=DEVICE)
    for r, n in enumerate(s["lengths"].tolist()):
        pages = s["block_table"][r, :-(-n // page)].long()
        parts = [v.view(torch.uint8)[pages].view(v.dtype).double().reshape(pages.numel() * page, -1)[:n] for v in views]
        if len(parts) == 1:
            k = parts[0]
        else:
            k = torch.cat([parts[0] * parts[1].repeat_interleave(parts[0].shape[1] // parts[1].shape[1], dim=1), parts[2]], dim=1)
        for i in range(s_q):
            m = n - s_q + 1 + i
            if m <= 0:
                continue
            scores = s["q"][r, i].double() @ k[:m].T * s["scale"]
            lse_e = torch.logsumexp(scores, dim=1)
            if s["sink"] is not None:
                lse_e = torch.logaddexp(lse_e, s["sink"].double())
            out[r, i] = torch.exp(scores - lse_e.unsqueeze(1)) @ k[:m, :512]
            lse[r, i] = lse_e / math.log(2.0)
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "index": _exact_index, "attend": _exact_attend}[case["kind"]](s)
