"""The choice of pages (rxq4_select_pages) at the ends of its ranges: the most rows, launches
of the most workgroups."""
from __future__ import annotations

import pytest
import torch

import rxq4
from rxq4 import capi

pytestmark = pytest.mark.gpu
ROWS, HD = 1 << 20, 8


def _call(rows, max_new, KV=8, width=4):
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


def test_the_most_rows_with_one_new_token():
    """A token a workgroup would be more than a launch may have."""
    pages = _call(ROWS, 1)
    assert pages[0].tolist() == [[0, -1]] * 8
    assert (pages[1:] == -7).all()


def test_more_workgroups_than_a_launch_may_have():
    """Sixteen tokens a workgroup and KV head, 1024 of them."""
    rows = 1 << 17
    with pytest.raises(rxq4.RxQ4Error):
        _call(rows, rows, KV=1024)
    rows -= 256  # 2^23 - 8192 workgroups
    pages = _call(rows, rows, KV=1024)
    last = (torch.arange(rows, device="cuda") // 1024).clamp(max=3)
    assert (pages[..., 0] == 0).all()
    assert (pages[..., 1] == torch.where(last > 0, last, -1)[:, None]).all()
