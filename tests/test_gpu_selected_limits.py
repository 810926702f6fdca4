"""The choice of pages (rxq4_select_pages) at the ends of its ranges: the most rows, launches
of the most workgroups."""
from __future__ import annotations

import pytest
import torch

import rxq4
from rxq4 import capi

pytestmark = pytest.mark.gpu
ROWS, KV, HD = 1 << 20, 8, 8


def _call(rows, max_new, width=4):
    """`rows` new tokens of one sequence in `width` pages of 1024, lists of the first and the last."""
    k = torch.zeros((width, 1024, KV, HD), dtype=torch.float16, device="cuda")
    cache = capi.PagedKV(k, torch.zeros_like(k), torch.arange(width, dtype=torch.int32, device="cuda")[None])
    batch = capi.SeqBatch(torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                          torch.tensor([rows], dtype=torch.int32, device="cuda"), rows, max_new, rows)
    q = torch.ones((rows, KV, HD), dtype=torch.float16, device="cuda")
    bounds = torch.ones((width, KV, HD // 8, 2, 8), dtype=torch.int8, device="cuda")
    pages = torch.full((rows, KV, 2), -7, dtype=torch.int32, device="cuda")
    capi.select_pages(pages, q, bounds, torch.ones((width, KV), device="cuda"), batch, cache, 1, 1)
    torch.cuda.synchronize()
    return pages


def test_the_most_rows_in_tiles():
    """2^20 tokens and 8 KV heads, sixteen tokens a workgroup."""
    pages = _call(ROWS, ROWS)
    last = (torch.arange(ROWS, device="cuda") // 1024).clamp(max=3)
    assert (pages[..., 0] == 0).all()
    assert (pages[..., 1] == torch.where(last > 0, last, -1)[:, None]).all()


def test_more_workgroups_than_a_launch_may_have():
    """A token a workgroup (the sequences have one new token each, by the batch's limit)."""
    with pytest.raises(rxq4.RxQ4Error):
        _call(ROWS, 1)
    pages = _call(ROWS - 8, 1)  # 2^23 - 64 workgroups
    assert pages[0].tolist() == [[0, -1]] * KV
    assert (pages[1:] == -7).all()
