"""Refusals of the serving entry points (rxq4_qk_norm_rope,
rxq4_attention_paged_f16, rxq4_sample_f32), on the CPU: every bad argument is
found before the device is looked at, so nothing is launched."""
from __future__ import annotations

import ctypes

import pytest
import torch

import rxq4
from rxq4 import capi

P = 1 << 20  # an aligned address that is never read


def _cache(**over):
    a = dict(k=P, v=P, k_scales=None, v_scales=None, page_table=P, page_stride=0, table_stride=4, n_pages=8,
             page_size=16, n_kv_heads=2, head_dim=64, kv_int8=0)
    return capi.PagedKVStruct(**(a | over))


def _batch(**over):
    a = dict(q_starts=P, seq_lens=P, n_seqs=2, n_tokens=5, max_new=4, max_len=60)
    return capi.SeqBatchStruct(**(a | over))


def _attend(cache=None, batch=None, **over):
    a = dict(out=P, q=P, n_heads=8, scale=0.125) | over
    ref = lambda x: None if x is False else ctypes.byref(x)  # noqa: E731
    return rxq4.load().rxq4_attention_paged_f16(a["out"], a["q"], a["n_heads"], a["scale"],
                                                ref(_batch() if batch is None else batch),
                                                ref(_cache() if cache is None else cache), None)


def _rope(cache=None, batch=None, **over):
    a = dict(q_out=P, q=2 * P, k=3 * P, v=4 * P, x_dtype=1, q_stride=512, kv_stride=128, n_heads=8, q_weight=P,
             k_weight=P, eps=1e-6, inv_freq=P, n_rot=64, interleaved=0) | over
    return rxq4.load().rxq4_qk_norm_rope(*a.values(), ctypes.byref(_batch() if batch is None else batch),
                                         ctypes.byref(_cache() if cache is None else cache), None)


def _sample(**over):
    a = dict(ids=P, logits=P, row_stride=100, n_rows=3, n_vocab=100, temperature=None, top_k=None, top_p=None,
             min_p=None, u=P) | over
    return rxq4.load().rxq4_sample_f32(*a.values(), None)


def refused(status, word):
    assert status == rxq4.INVALID_ARGUMENT
    assert word in capi.last_error(), capi.last_error()


BAD_CACHE = [(dict(k=None), "null"), (dict(v=P + 8), "aligned"), (dict(n_kv_heads=3), "multiple"),
             (dict(n_kv_heads=0), "multiple"), (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"),
             (dict(head_dim=264), "head_dim"), (dict(kv_int8=1, head_dim=72), "head_dim"),
             (dict(page_size=0), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=2048), "page_size"),
             (dict(n_pages=-1), "n_pages"), (dict(n_pages=1 << 27), "n_pages"), (dict(page_stride=2040), "page_stride"),
             (dict(page_stride=2052), "page_stride"), (dict(page_stride=-2048), "page_stride"),
             (dict(page_table=None), "page_table"), (dict(table_stride=-1), "table_stride")]
BAD_BATCH = [(dict(n_seqs=-1), "n_seqs"), (dict(n_tokens=-1), "n_tokens"), (dict(max_new=-1), "max_new"),
             (dict(max_len=-1), "max_len"), (dict(q_starts=None), "null"), (dict(seq_lens=None), "null"),
             (dict(n_seqs=65537), "n_seqs"), (dict(n_tokens=(1 << 20) + 1), "n_tokens"),
             (dict(max_len=(1 << 24) + 1), "max_len")]


@pytest.mark.parametrize("call", [_attend, _rope])
@pytest.mark.parametrize("over,word", BAD_CACHE)
def test_bad_caches(call, over, word):
    refused(call(cache=_cache(**over)), word)


@pytest.mark.parametrize("call", [_attend, _rope])
@pytest.mark.parametrize("over,word", BAD_BATCH)
def test_bad_batches(call, over, word):
    refused(call(batch=_batch(**over)), word)


@pytest.mark.parametrize("over,word", [(dict(out=None), "null"), (dict(q=P + 2), "aligned"), (dict(n_heads=0), "n_heads"),
                                       (dict(n_heads=7), "multiple"), (dict(n_heads=2048), "n_heads"),
                                       (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale")])
def test_bad_attention(over, word):
    refused(_attend(**over), word)


def test_null_descriptors():
    refused(_attend(batch=False), "null batch")
    refused(_attend(cache=False), "null cache")


@pytest.mark.parametrize("over,word", [
    (dict(x_dtype=3), "x_dtype"), (dict(q_stride=504), "q_stride"), (dict(kv_stride=120), "kv_stride"),
    (dict(q_stride=516), "q_stride"), (dict(n_rot=63), "n_rot"), (dict(n_rot=66), "n_rot"), (dict(n_rot=-2), "n_rot"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(inv_freq=None), "inv_freq"), (dict(q=None), "null"),
    (dict(q_out=None), "null"), (dict(k=3 * P + 2), "aligned"), (dict(v=None), "null"),
    (dict(q=P, q_stride=520), "overlaps"), (dict(q=P, x_dtype=2), "overlaps"), (dict(q=P - 64), "overlaps"),
    (dict(q=P + 64), "overlaps")])
def test_bad_rope(over, word):
    refused(_rope(**over), word)


@pytest.mark.parametrize("missing", ["k_scales", "v_scales"])
def test_rope_int8_needs_scales(missing):
    refused(_rope(cache=_cache(**({"kv_int8": 1, "k_scales": P, "v_scales": P} | {missing: None}))), "scale")


@pytest.mark.parametrize("over,word", [(dict(n_rows=-1), "n_rows"), (dict(n_vocab=0), "n_vocab"),
                                       (dict(n_vocab=(1 << 22) + 1, row_stride=1 << 23), "n_vocab"),
                                       (dict(row_stride=99), "row_stride"), (dict(ids=None), "null"),
                                       (dict(logits=None), "null"), (dict(u=None), "null")])
def test_bad_sample(over, word):
    refused(_sample(**over), word)


def test_nothing_to_do_is_success():
    assert _attend(batch=_batch(n_seqs=0, q_starts=None, seq_lens=None)) == rxq4.SUCCESS
    assert _attend(batch=_batch(n_tokens=0), q=None) == rxq4.SUCCESS
    assert _rope(batch=_batch(n_tokens=0), q=None) == rxq4.SUCCESS
    assert _sample(n_rows=0, logits=None) == rxq4.SUCCESS


def test_python_binding_refuses():
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    table = torch.zeros((2, 2), dtype=torch.int32)
    with pytest.raises(ValueError):
        capi.PagedKV(k, k.float(), table)
    with pytest.raises(ValueError):
        capi.PagedKV(k, k, table.long())
    with pytest.raises(ValueError):
        capi.PagedKV(k.transpose(1, 2), k.transpose(1, 2), table)
    with pytest.raises(ValueError):
        capi.PagedKV(k.char(), k.char(), table, torch.zeros((4, 16, 3)))
    starts, lens = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        capi.SeqBatch(starts[:2], lens, 3, 3, 3)
    with pytest.raises(ValueError):
        capi.SeqBatch(starts.long(), lens, 3, 3, 3)
    cache, batch = capi.PagedKV(k, k, table), capi.SeqBatch(starts, lens, 3, 3, 3)
    q = torch.zeros((3, 8, 64), dtype=torch.float16)
    with pytest.raises(ValueError):  # one sequence more than the table has rows
        capi.attention_paged_f16(q, q, capi.SeqBatch(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32),
                                                     3, 3, 3), cache, 1.0)
    with pytest.raises(ValueError):  # rows
        capi.attention_paged_f16(q[:2], q[:2], batch, cache, 1.0)
    with pytest.raises(ValueError):  # not on the GPU
        capi.attention_paged_f16(q, q, batch, cache, 1.0)
    kv = torch.zeros((3, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError):  # k and v rows differently far apart
        capi.qk_norm_rope(q, q.clone(), kv, torch.zeros((3, 4, 64), dtype=torch.float16)[:, :2], batch, cache, None)
    logits, u = torch.zeros((3, 100)), torch.zeros(3)
    with pytest.raises(ValueError):
        capi.sample_f32(torch.zeros(3, dtype=torch.int64), logits, u)
    with pytest.raises(ValueError):
        capi.sample_f32(torch.zeros(3, dtype=torch.int32), logits, u[:2])
    with pytest.raises(ValueError):
        capi.sample_f32(torch.zeros(3, dtype=torch.int32), logits.t().contiguous().t(), u)


@pytest.mark.parametrize("n_seqs", [1, 2])
def test_an_empty_page_table_is_a_table(n_seqs):
    """A table without entries, whose tensor has no address, is no contiguous cache: the
    descriptor names a table of width 0, and no position is in it."""
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    cache = capi.PagedKV(k, k, torch.zeros((n_seqs, 0), dtype=torch.int32))
    assert cache.struct.page_table and cache.struct.table_stride == 0
    assert cache.n_seqs == n_seqs


def test_pages_that_share_memory_are_refused():
    """An expanded page (stride 0, which the C side takes for dense) and pages that
    overlap; one page may have any stride."""
    page = torch.zeros((1, 16, 2, 64), dtype=torch.float16)
    table = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(ValueError):
        capi.PagedKV(page.expand(4, -1, -1, -1), page.expand(4, -1, -1, -1), table)
    half = torch.zeros(4096, dtype=torch.float16).as_strided((3, 16, 2, 64), (1024, 128, 64, 1))
    with pytest.raises(ValueError):
        capi.PagedKV(half, half, table)
    apart = torch.zeros((3, 2, 16, 2, 64), dtype=torch.float16)
    assert capi.PagedKV(apart[:, 0], apart[:, 1], table).struct.page_stride == 4096
    assert capi.PagedKV(page, page, table).struct.page_stride == 2048


@pytest.mark.parametrize("over", [dict(q_out=3 * P), dict(q_out=4 * P), dict(q_out=3 * P - 16),
                                  dict(q_out=4 * P + 1264), dict(q_out=4 * P + 2544, x_dtype=0),
                                  dict(q_out=3 * P + 8192, kv_stride=4096)])
def test_rope_output_over_keys_or_values(over):
    """5 rows of 128 elements: 1280 bytes of fp16, 2560 of fp32."""
    refused(_rope(**over), "overlaps")


@pytest.mark.parametrize("out,q", [(P, P + 16), (P + 16, P), (P, P + 5104), (P + 5104, P)])
def test_attention_output_partly_over_the_queries(out, q):
    """5 rows of 8 heads of 64: 5120 bytes."""
    refused(_attend(out=out, q=q), "overlaps")


def test_more_rows_than_the_limit():
    """2^20 rows, as for the other operators; the launches count them in 32 bits."""
    refused(_sample(n_rows=(1 << 20) + 1), "n_rows")
