"""What a decoding step does to and with whole caches: new tokens' rows go in, and attention over all of a request's rows.

``append_kv_cache`` writes latent rows (their positional part rotated on the way, the queries' too), ``append_indexer_keys`` what the
indexer reads, and ``paged_mla_decode_fwd`` attends over everything that a block table names: for layers without an indexer, and for
contexts that are not longer than the lists of those with one.  The reference's caches are written by the serving engine, and its
attention takes index lists only (flash_mla_sm120/interface.py:39-58)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._lib import native


def append_kv_cache(kv_c: torch.Tensor, k_pe: torch.Tensor, kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
                    positions: Optional[torch.Tensor] = None, cos_sin: Optional[torch.Tensor] = None, interleaved: bool = True,
                    q_pe: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Row ``slot_mapping[t]`` of ``kv_cache`` takes token t: ``kv_c`` [T, 512] (448 for the 584-byte layout) and ``k_pe`` [T, 64]
    turned by the token's angles.  Both may be slices of one projection's output (rows any multiple of 8 values apart).

    ``kv_cache``: 656-byte rows, 584-byte pages, or [num_blocks, block, 1, 576] bf16 / fp16, whose type kv_c, k_pe and the queries
    have (bf16 for the byte layouts); pages may be padded, and start on 16 bytes (584-byte pages on 8: those of an odd number of rows can be
    written without padding, but not read by paged_mla_decode_fwd).  Slots (int32 or int64) number rows through the pages: page s // block, row
    s % block.  One outside the cache, -1 say, leaves the cache as it is.  Slots must differ: of two tokens with one slot the row
    gets pieces of either.
    ``positions`` [T] (int32 or int64) are rows of ``cos_sin`` [positions, 64] fp32, 32 cosines and 32 sines; without both nothing is
    rotated.  ``interleaved``: values 2i and 2i + 1 turn by angle i, else values i and i + 32.  A token whose position lies outside
    the table leaves the cache and a given q_out as they are; an allocated q_out has zeros for it.
    ``q_pe`` [T, H, 64], the same tokens' queries, any distances between tokens and heads -> ``q_out`` (allocated if not given; a
    slice of the query [T, H, 576], or q_pe itself; no two vectors in one place), which is returned."""
    return native().append_kv(kv_c, k_pe, kv_cache, slot_mapping, positions, cos_sin, interleaved, q_pe, q_out)


def append_indexer_keys(k: torch.Tensor, ki: torch.Tensor, k_scale: torch.Tensor, slot_mapping: torch.Tensor,
                        positions: Optional[torch.Tensor] = None, cos_sin: Optional[torch.Tensor] = None, interleaved: bool = False,
                        rope_offset: int = 0, q: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                        ) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
    """What ``indexer.fp8_mqa_logits`` reads: ``k`` [T, 128] bf16, values [rope_offset, rope_offset + 64) turned by the token's angles
    (rope_offset 0 or 64), goes to rows ``slot_mapping`` of ``ki`` [s_k, 128] e4m3 and ``k_scale`` [s_k] fp32: scale = max(|k|, 1e-4) / 448,
    rounded once, from fp32.  Slots, positions, cos_sin and interleaved as in append_kv_cache.

    With ``q`` [T, H, 128] bf16 the same tokens' queries too; returns (qi [T, H, 128] e4m3, weights [T, H] fp32 times each query's scale,
    or the scales where no weights are given), zeros both for a token whose position lies outside the table."""
    return native().append_index(k, ki, k_scale, slot_mapping, positions, cos_sin, interleaved, rope_offset, q, weights)


def paged_mla_decode_fwd(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, cache_seqlens: torch.Tensor, sm_scale: float,
                         d_v: int = 512, causal: bool = False, attn_sink: Optional[torch.Tensor] = None,
                         out: Optional[torch.Tensor] = None, num_sm_parts: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of the newest tokens over all rows of their request: attention split over the rows -> merge.

    ``q`` [B, s_q, H, 576] or [B, H, 576] (512 wide over 584-byte pages), bf16 (fp16 over fp16 rows), H up to 128; ``kv_cache``
    [num_blocks, block, 1, 576] bf16 / fp16, or the 656- and 584-byte layouts, pages on 16 bytes (584-byte pages of an odd number of rows
    therefore padded); ``block_table`` [B, pages] int32 (rows any distance apart);
    ``cache_seqlens`` [B] int32 rows of each request, the new tokens' own among them (0: none; more than the table has pages for: all of
    those).  ``causal``: query i of s_q sees rows [0, cache_seqlens - s_q + 1 + i).  Rows in pages that the cache does not have (-1, say)
    count as no entry.  ``num_sm_parts``: partitions that all rows are cut into (default: one per SM and 64 query rows).
    Returns (out [..., H, 512] in q's type, lse [..., H] fp32, base 2 with the sink in it); 0 and -1e30 where a query sees nothing (with a
    sink above -inf: 0 and the sink).  What a query does not see has no part in its output, NaN and infinities included, in rows or in other
    queries.  (An infinity in a row that a query does see and scores at minus infinity: 0 times infinity is no number; but in the newest
    s_q - 1 rows under a causal mask, which other queries must not see, it may count as nothing.)
    Exact numerics: products of 16-bit values (the byte layouts' are exact in bf16 where their scales are
    powers of two, as append_kv_cache and pack_kv_cache write them, else rounded to it), fp32 sums and softmax; weights are rounded to 16
    bits for their product with V."""
    return native().paged_decode(q, kv_cache, block_table, cache_seqlens, sm_scale, d_v, causal, attn_sink, out, num_sm_parts)
