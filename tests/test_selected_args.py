"""Refusals of the entry points for long and multimodal contexts
(rxq4_qk_norm_rope_axes, rxq4_kv_bounds, rxq4_select_pages,
rxq4_attention_selected_f16), on the CPU: every bad argument is found before the device
is looked at, so nothing is launched."""
from __future__ import annotations

import ctypes

import pytest
import torch

import rxq4
from rxq4 import capi
from tests.test_serving_args import BAD_BATCH, BAD_CACHE, P, _batch, _cache, refused


def _refs(batch, cache):
    return ctypes.byref(_batch() if batch is None else batch), ctypes.byref(_cache() if cache is None else cache)


def _axes(cache=None, batch=None, **over):
    a = dict(q_out=P, q=2 * P, k=3 * P, v=4 * P, x_dtype=1, q_stride=512, kv_stride=128, n_heads=8, q_weight=P,
             k_weight=P, eps=1e-6, inv_freq=P, n_rot=64, interleaved=0, positions=5 * P, position_stride=5, n_axes=3,
             axis_of=6 * P) | over
    return rxq4.load().rxq4_qk_norm_rope_axes(*a.values(), *_refs(batch, cache), None)


def _bounds(cache=None, batch=None, **over):
    a = dict(bounds=2 * P, scales=3 * P) | over
    return rxq4.load().rxq4_kv_bounds(*a.values(), *_refs(batch, cache), None)


def _select(cache=None, batch=None, **over):
    a = dict(pages=2 * P, n_select=4, n_first=1, n_last=1, q=3 * P, n_heads=8, bounds=4 * P, scales=5 * P) | over
    return rxq4.load().rxq4_select_pages(*a.values(), *_refs(batch, cache), None)


def _attend(cache=None, batch=None, **over):
    a = dict(out=P, q=P, n_heads=8, scale=0.125, pages=2 * P, n_select=4) | over
    return rxq4.load().rxq4_attention_selected_f16(*a.values(), *_refs(batch, cache), None)


CALLS = [_axes, _bounds, _select, _attend]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("over,word", BAD_CACHE)
def test_bad_caches(call, over, word):
    if call is _bounds and over == dict(n_kv_heads=3):
        pytest.skip("no query heads that 3 would have to divide")
    refused(call(cache=_cache(**over)), word)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("over,word", BAD_BATCH)
def test_bad_batches(call, over, word):
    refused(call(batch=_batch(**over)), word)


def test_null_descriptors():
    lib = rxq4.load()
    b, c = _refs(None, None)
    refused(lib.rxq4_kv_bounds(P, P, None, c, None), "null batch")
    refused(lib.rxq4_kv_bounds(P, P, b, None, None), "null cache")
    refused(lib.rxq4_select_pages(P, 1, 0, 0, P, 8, P, P, None, c, None), "null batch")
    refused(lib.rxq4_select_pages(P, 1, 0, 0, P, 8, P, P, b, None, None), "null cache")
    refused(lib.rxq4_attention_selected_f16(P, P, 8, 1.0, P, 1, None, c, None), "null batch")
    refused(lib.rxq4_attention_selected_f16(P, P, 8, 1.0, P, 1, b, None, None), "null cache")


@pytest.mark.parametrize("over,word", [
    (dict(n_axes=0), "n_axes"), (dict(n_axes=-1), "n_axes"), (dict(n_axes=17), "n_axes"),
    (dict(position_stride=4), "position_stride"), (dict(position_stride=-5), "position_stride"),
    (dict(position_stride=(1 << 32) + 1), "position_stride"), (dict(positions=None), "positions"),
    (dict(positions=5 * P + 2), "positions"), (dict(axis_of=6 * P + 1), "axis_of"), (dict(x_dtype=3), "x_dtype"),
    (dict(q_stride=504), "q_stride"), (dict(n_rot=63), "n_rot"), (dict(eps=-1.0), "eps"), (dict(inv_freq=None), "inv_freq"),
    (dict(q_out=None), "null"), (dict(q=P + 64), "overlaps"), (dict(positions=P + 4 * 1024), "positions"),
    (dict(positions=P - 56), "positions"), (dict(axis_of=P + 16), "axis_of"), (dict(axis_of=P - 124), "axis_of")])
def test_bad_axes(over, word):
    refused(_axes(**over), word)


@pytest.mark.parametrize("missing", ["k_scales", "v_scales"])
def test_axes_int8_needs_scales(missing):
    refused(_axes(cache=_cache(**({"kv_int8": 1, "k_scales": P, "v_scales": P} | {missing: None}))), "scale")


# the cache of _cache: 8 pages of 16 positions, 2 heads of 64: 32768 bytes of keys from P, 2048 of bounds, 64 of scales
@pytest.mark.parametrize("over,word", [
    (dict(bounds=None), "null"), (dict(scales=None), "null"), (dict(bounds=2 * P + 8), "aligned"),
    (dict(scales=3 * P + 2), "aligned"), (dict(scales=2 * P + 2044), "overlap"), (dict(scales=2 * P - 60), "overlap"),
    (dict(bounds=P + 32752), "overlap"), (dict(bounds=P - 2032), "overlap"), (dict(scales=P + 32764), "overlap")])
def test_bad_bounds(over, word):
    refused(_bounds(**over), word)


# 5 tokens: 160 bytes of lists, 5120 of queries
@pytest.mark.parametrize("over,word", [
    (dict(n_select=0), "n_select"), (dict(n_select=-3), "n_select"), (dict(n_select=4097), "n_select"),
    (dict(n_first=-1), "n_first"), (dict(n_last=-1), "n_last"), (dict(n_first=3, n_last=2), "fit"),
    (dict(n_first=2 ** 31 - 1, n_last=2 ** 31 - 1), "fit"), (dict(n_heads=0), "n_heads"), (dict(n_heads=7), "multiple"),
    (dict(pages=None), "null"), (dict(pages=2 * P + 2), "aligned"), (dict(q=None), "null"), (dict(q=3 * P + 8), "aligned"),
    (dict(bounds=None), "null"), (dict(bounds=4 * P + 8), "aligned"), (dict(scales=None), "null"),
    (dict(scales=5 * P + 1), "aligned"), (dict(pages=3 * P + 5116), "overlaps"), (dict(pages=3 * P - 156), "overlaps"),
    (dict(pages=4 * P + 2044), "overlaps"), (dict(pages=5 * P - 156), "overlaps")])
def test_bad_select(over, word):
    refused(_select(**over), word)


@pytest.mark.parametrize("over,word", [
    (dict(out=None), "null"), (dict(q=P + 2), "aligned"), (dict(n_heads=0), "n_heads"), (dict(n_heads=7), "multiple"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(q=P + 64), "overlaps"),
    (dict(n_select=0), "n_select"), (dict(n_select=4097), "n_select"), (dict(pages=None), "null"),
    (dict(pages=2 * P + 1), "aligned"), (dict(pages=P + 5116), "overlaps"), (dict(pages=P - 156), "overlaps")])
def test_bad_attention(over, word):
    refused(_attend(**over), word)


def test_nothing_to_do_is_success():
    none = _batch(n_seqs=0, q_starts=None, seq_lens=None)
    assert _axes(batch=none, positions=None) == rxq4.SUCCESS
    assert _axes(batch=_batch(n_tokens=0), q=None, positions=None) == rxq4.SUCCESS
    for over in (dict(n_seqs=0, q_starts=None, seq_lens=None), dict(n_tokens=0), dict(max_new=0)):
        assert _bounds(batch=_batch(**over), bounds=None) == rxq4.SUCCESS
        assert _select(batch=_batch(**over), pages=None, q=None) == rxq4.SUCCESS
        assert _attend(batch=_batch(**over), out=None, q=None, pages=None) == rxq4.SUCCESS
    assert _bounds(cache=_cache(n_pages=0, k=None, v=None), bounds=None) == rxq4.SUCCESS


def _on_cpu():
    k, v = (torch.zeros((4, 8, 2, 64), dtype=torch.float16) for _ in range(2))
    cache = capi.PagedKV(k, v, torch.zeros((2, 2), dtype=torch.int32))
    batch = capi.SeqBatch(torch.tensor([0, 1, 3], dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32), 3, 2, 16)
    return cache, batch


def test_binding_refuses_shapes_and_types():
    cache, batch = _on_cpu()
    f16, i32 = torch.float16, torch.int32
    q = torch.zeros((3, 4, 64), dtype=f16)
    kv = torch.zeros((3, 2, 64), dtype=f16)
    freq, at, axis = torch.zeros(32), torch.zeros((3, 3), dtype=i32), torch.zeros(32, dtype=i32)
    for bad in (dict(positions=at.long()), dict(positions=at[:, :2]), dict(positions=at.t()), dict(axis_of=axis[:31]),
                dict(axis_of=axis.long()), dict(q=q.double()), dict(q=q[:2])):
        a = dict(q=q, positions=at, axis_of=axis) | bad
        with pytest.raises((ValueError, KeyError)):
            capi.qk_norm_rope_axes(torch.zeros_like(q), a["q"], kv, kv, batch, cache, freq, a["positions"], a["axis_of"])
    bounds, scales, pages = torch.zeros((4, 2, 8, 2, 8), dtype=torch.int8), torch.zeros((4, 2)), torch.zeros((3, 2, 4), dtype=i32)
    for bad in (dict(bounds=bounds.short()), dict(bounds=bounds[:3]), dict(bounds=bounds.transpose(0, 1)), dict(scales=scales[:3]),
                dict(scales=scales.half()), dict(scales=torch.zeros((2, 4)).t())):
        a = dict(bounds=bounds, scales=scales) | bad
        with pytest.raises(ValueError):
            capi.kv_bounds(a["bounds"], a["scales"], batch, cache)
        with pytest.raises(ValueError):
            capi.select_pages(pages, q, a["bounds"], a["scales"], batch, cache)
    for bad in (dict(q=q.float()), dict(q=q[:2]), dict(q=q[..., :32]), dict(q=q.transpose(0, 1)), dict(pages=pages.long()),
                dict(pages=pages[:2]), dict(pages=pages[:, :1]), dict(pages=pages[..., 0]), dict(pages=pages.transpose(0, 2))):
        a = dict(q=q, pages=pages) | bad
        with pytest.raises(ValueError):
            capi.select_pages(a["pages"], a["q"], bounds, scales, batch, cache)
        with pytest.raises(ValueError):
            capi.attention_selected_f16(torch.zeros_like(a["q"]), a["q"], a["pages"], batch, cache, 0.1)
    with pytest.raises(ValueError):
        capi.attention_selected_f16(torch.zeros((3, 4, 32), dtype=f16), q, pages, batch, cache, 0.1)


def test_binding_refuses_tensors_off_the_gpu():
    cache, batch = _on_cpu()
    q, pages = torch.zeros((3, 4, 64), dtype=torch.float16), torch.zeros((3, 2, 4), dtype=torch.int32)
    bounds, scales = torch.zeros((4, 2, 8, 2, 8), dtype=torch.int8), torch.zeros((4, 2))
    for call in (lambda: capi.kv_bounds(bounds, scales, batch, cache),
                 lambda: capi.select_pages(pages, q, bounds, scales, batch, cache),
                 lambda: capi.attention_selected_f16(torch.zeros_like(q), q, pages, batch, cache, 0.1)):
        with pytest.raises(ValueError, match="current GPU"):
            call()
