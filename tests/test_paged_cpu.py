"""What paged.py refuses, before any device work, and its oracle against the oracles that were there."""
import ctypes

import pytest
import torch

import paged_cases as P
from oracle import sparse_mla_oracle as orc
from sparse_mla_sm120_b200 import _lib, interface, paged


def _append(**kw):
    a = dict(kv_c=torch.zeros(3, 512, dtype=torch.bfloat16), k_pe=torch.zeros(3, 64, dtype=torch.bfloat16),
             kv_cache=torch.zeros(4, 64, 1, 656, dtype=torch.uint8), slot_mapping=torch.zeros(3, dtype=torch.int64))
    a.update(kw)
    return lambda: paged.append_kv_cache(**a)


ROT = dict(positions=torch.zeros(3, dtype=torch.int64), cos_sin=torch.zeros(8, 64))


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(kv_c=torch.zeros(3, 448, dtype=torch.bfloat16)), "kv_c must be"),
    (dict(kv_c=torch.zeros(3, 512)), "kv_c must be"),
    (dict(kv_c=torch.zeros(3, 512, dtype=torch.float16)), "kv_c must be"),
    (dict(kv_c=torch.zeros(512, 3, dtype=torch.bfloat16).T), "contiguous"),
    (dict(k_pe=torch.zeros(2, 64, dtype=torch.bfloat16)), "k_pe must be"),
    (dict(kv_cache=torch.zeros(4, 64, 1, 657, dtype=torch.uint8)), "rows must be"),
    (dict(kv_cache=torch.zeros(4, 64, 1, 576)), "byte tensor"),
    (dict(kv_cache=torch.zeros(4, 64, 2, 576, dtype=torch.bfloat16)), "16-bit rows"),
    (dict(kv_cache=torch.zeros(64, 576, dtype=torch.bfloat16)), "16-bit rows"),
    (dict(kv_cache=torch.zeros(4, 64, 1, 584, dtype=torch.uint8)), "kv_c must be"),
    (dict(kv_cache=torch.zeros(4, 64, 1, 576, dtype=torch.float16)), "kv_c must be"),
    (dict(slot_mapping=torch.zeros(2, dtype=torch.int64)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(3)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(6, dtype=torch.int32)[::2]), "slot_mapping"),
    (dict(positions=ROT["positions"]), "go together"),
    (dict(cos_sin=ROT["cos_sin"]), "go together"),
    (dict(ROT, cos_sin=torch.zeros(8, 32)), "cos_sin"),
    (dict(ROT, cos_sin=torch.zeros(8, 64, dtype=torch.float64)), "cos_sin"),
    (dict(ROT, positions=torch.zeros(4, dtype=torch.int64)), "positions"),
    (dict(q_pe=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "q_pe needs"),
    (dict(ROT, q_pe=torch.zeros(3, 8, 32, dtype=torch.bfloat16)), "q_pe must be"),
    (dict(ROT, q_pe=torch.zeros(3, 8, 64, dtype=torch.bfloat16), q_out=torch.zeros(3, 7, 64, dtype=torch.bfloat16)), "q_out must be"),
    (dict(ROT, q_out=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "without q_pe"),
])
def test_append_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _append(**kw)()


def test_append_takes_tensors_only():
    with pytest.raises(TypeError):
        _append(slot_mapping=[0, 1, 2])()
    with pytest.raises(TypeError):
        _append(kv_c=None)()


def _index(**kw):
    a = dict(k=torch.zeros(3, 128, dtype=torch.bfloat16), ki=torch.zeros(9, 128, dtype=torch.float8_e4m3fn), k_scale=torch.zeros(9),
             slot_mapping=torch.zeros(3, dtype=torch.int32))
    a.update(kw)
    return lambda: paged.append_indexer_keys(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(k=torch.zeros(3, 64, dtype=torch.bfloat16)), "k must be"),
    (dict(k=torch.zeros(3, 128)), "k must be"),
    (dict(ki=torch.zeros(9, 128)), "ki must be"),
    (dict(k_scale=torch.zeros(8)), "k_scale must be"),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), "slot_mapping"),
    (dict(positions=ROT["positions"]), "go together"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(2, 4, 128, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16), weights=torch.zeros(3, 5)), "weights must be"),
    (dict(weights=torch.zeros(3, 5)), "without q"),
])
def test_index_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _index(**kw)()


def _attend(**kw):
    a = dict(q=torch.zeros(2, 8, 576, dtype=torch.bfloat16), kv_cache=torch.zeros(4, 64, 1, 576, dtype=torch.bfloat16),
             block_table=torch.zeros(2, 3, dtype=torch.int32), cache_seqlens=torch.zeros(2, dtype=torch.int32), sm_scale=1.0)
    a.update(kw)
    return lambda: paged.paged_mla_decode_fwd(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros(2, 8, 512, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(2, 8, 576, dtype=torch.float16)), "q must be"),
    (dict(q=torch.zeros(2, 576, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(2, 576, 8, dtype=torch.bfloat16).transpose(1, 2)), "contiguous"),
    (dict(kv_cache=torch.zeros(4, 64, 1, 584, dtype=torch.uint8)), "q must be"),
    (dict(kv_cache=torch.zeros(64, 656, dtype=torch.uint8)), "num_blocks"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).T), "block_table"),
    (dict(cache_seqlens=torch.zeros(2, dtype=torch.int64)), "cache_seqlens"),
    (dict(cache_seqlens=torch.zeros(3, dtype=torch.int32)), "cache_seqlens"),
    (dict(attn_sink=torch.zeros(7)), "attn_sink"),
    (dict(attn_sink=torch.zeros(8, dtype=torch.bfloat16)), "attn_sink"),
    (dict(d_v=256), "d_v"),
    (dict(out=torch.zeros(2, 8, 576, dtype=torch.bfloat16)), "out must be"),
    (dict(out=torch.zeros(2, 8, 512)), "out must be"),
])
def test_attention_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _attend(**kw)()


def test_entry_points_check_before_they_launch():
    lib, fake = _lib.load(), 4096

    def decode(layout=2, pages=4, page=64, stride=64 * 1152, table=fake, batch=1, s_q=1, heads=16, parts=3, scratch=1 << 30, q=fake, cache=fake):
        return lib.smla_paged_decode(q, cache, layout, pages, page, stride, table, 4, 4, fake, fake, fake, batch, s_q, heads, 1.0, 0, None, parts, fake,
                                     scratch, None, None)
    assert decode(layout=4) == -2 and decode(page=0) == -2 and decode(stride=64 * 1152 - 16) == -2 and decode(heads=129) == -2
    assert decode(heads=0) == -2 and decode(batch=-1) == -2 and decode(parts=-1) == -2 and decode(parts=1 << 20) == -2
    assert decode(table=None) == -1 and decode(q=fake + 8) == -3 and decode(stride=64 * 1152 + 8) == -3 and decode(cache=fake + 8) == -3
    assert decode(layout=1, page=63, stride=63 * 584) == -3      # pages of 584-byte rows that do not start on 16 bytes
    assert decode(scratch=1000) == -5 and b"scratch" in lib.smla_last_error()
    assert decode(batch=0) == 0 and decode(s_q=0) == 0
    need = lib.smla_paged_scratch_bytes(5, 2, 16, 4, 64, 3)
    assert need == 6 * 32 * 513 * 4 + 5 * 8 and lib.smla_paged_scratch_bytes(5, 2, 16, 4, 64, 1) == 40
    assert lib.smla_paged_scratch_bytes(5, 2, 129, 4, 64, 3) == 0

    def append(layout=0, stride=64 * 656, slots=fake, kv_c=fake, pos=None, cs=None, q=None, q_out=None, step=576, n=1, heads=0):
        return lib.smla_append_kv(kv_c, step, fake, 576, fake, layout, 4, 64, stride, slots, 1, pos, 1, cs, 8, 1, q, 64, 64, q_out, 64, 64, n, heads, None)
    assert append(layout=7) == -2 and append(stride=64) == -2 and append(slots=None) == -1 and append(kv_c=fake + 2) == -3 and append(step=577) == -3
    assert append(pos=fake) == -1 and append(cs=fake) == -1 and append(q=fake) == -1 and append(q=fake, q_out=fake) == -1 and append(n=-1) == -2
    assert append(n=0) == 0 and append(pos=fake, cs=fake + 4) == -3

    def index(offset=0, q=None, qi=None, w=None, k=fake, n=1, cap=8):
        return lib.smla_append_index(k, 128, fake, fake, cap, fake, 0, None, 0, None, 0, 1, offset, q, None, qi, w, n, 4, None)
    assert index(offset=32) == -2 and index(q=fake) == -1 and index(k=None) == -1 and index(k=fake + 8) == -3 and index(n=0) == 0 and index(cap=-1) == -2


def test_flashmla_surface_without_indices():
    meta, _ = interface.get_mla_metadata()
    q = torch.zeros(2, 1, 8, 576, dtype=torch.bfloat16)
    kv = torch.zeros(4, 64, 1, 576, dtype=torch.bfloat16)
    table, n = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="block_table"):
        interface.flash_mla_with_kvcache(q, kv, table, None, 512, meta)
    with pytest.raises(ValueError, match="does not go with"):
        interface.flash_mla_with_kvcache(q, kv, table, n, 512, meta, is_fp8_kvcache=True)
    with pytest.raises(ValueError, match="go with indices"):
        interface.flash_mla_with_kvcache(q, kv, table, n, 512, meta, topk_length=n)
    with pytest.raises(ValueError, match="d_v"):
        interface.flash_mla_with_kvcache(q, kv, table, n, 256, meta)
    with pytest.raises(ValueError, match="CUDA"):
        interface.flash_mla_with_kvcache(q, kv, table, n, 512, meta)
    assert not meta.have_initialized


@pytest.mark.parametrize("kind", ["v32", "model1"])
def test_oracle_agrees_with_the_sparse_one(kind):
    """All rows of a request as an index list, through the oracle that is pinned to the reference's own code."""
    cache = P.make_cache(kind, 5, 16, 3)
    deq = (orc.dequantize_kv_v32 if kind == "v32" else orc.dequantize_kv_model1)(cache)
    assert torch.equal(orc.cache_values(cache), deq[:, :, 0].double())
    lengths = torch.tensor([33, 7])
    table = P.table_of(lengths.tolist(), 16, 5, 4)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 1, 4, P.LATENT[kind] + 64, generator=g).to(torch.bfloat16)
    out, lse, *_ = orc.paged_attn_ref(q, cache, table, lengths, 0.05, True)
    for b, n in enumerate(lengths.tolist()):
        pos = torch.arange(n)
        rows = (table[b].long()[pos // 16] * 16 + pos % 16).to(torch.int32)
        ref, ref_lse = orc.ref_sparse_attn(q[b:b + 1], deq, rows.view(1, 1, -1), 0.05)
        assert float((out[b:b + 1] - ref.double()).abs().max()) <= 2.0 ** -8 * float(ref.abs().max()) + 1e-5
        assert float((lse[b] * orc.LN2 - ref_lse[0].double()).abs().max()) < 1e-5


def test_oracle_rotation_keeps_lengths():
    x = torch.randn(5, 3, 64, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    cs = P.rotary_table(100)
    pos = torch.tensor([0, 1, 17, 98, 99])
    for inter in (True, False):
        y = orc.rotate_ref(x, cs, pos, inter)
        assert torch.equal(y[0], x[0])
        assert float((y.square().sum(-1) - x.square().sum(-1)).abs().max()) < 1e-4
