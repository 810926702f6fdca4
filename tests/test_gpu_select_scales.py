"""The choice of pages (rxq4_select_pages) where scales of bounds are no scales: negative,
NaN and infinite ones, as arrays that were never written hold them.  The first and the last
pages are chosen all the same; others of a negative or NaN scale are not; an infinite one
makes scores infinite, and 0 of 0."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import selected_reference as sel
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def expected(p, both, scale, n_select, n_first, n_last):
    out = np.full((p.rows, p.kv, n_select), -7, np.int32)
    one = np.ones_like(scale)
    for i, (n, m) in enumerate(zip(p.new, p.lens)):
        for t in range(n):
            row, v = int(p.starts[i]) + t, sel.visible(p, m - n + t)
            out[row] = -1
            page = p.table[i, :v].numpy()
            there = (page >= 0) & (page < p.pages)
            safe = np.where(there, page, 0)
            y = sel.scores(p.q[row].numpy(), both[safe], one[safe])
            j = np.arange(v)
            always = ((j < n_first) | (j >= v - n_last)) & there
            for h in range(p.kv):
                x = scale[safe, h]
                with np.errstate(all="ignore"):
                    s = np.where((y[h] == 0) & np.isinf(x), np.float32(0), y[h] * x)
                    mine = there & ~always & (x >= 0)
                best = j[mine][np.lexsort((j[mine], -s[mine]))]
                order = np.concatenate((j[always], best))[:n_select]
                out[row, h, :len(order)] = np.sort(order)
    return out


def spoil(scale, both, rng):
    kind = rng.integers(0, 12, scale.shape)
    for i, x in enumerate((np.nan, -np.nan, -1.0, -1e-45, -np.inf, np.inf, -0.0)):
        scale[kind == i] = x
    both[rng.random(scale.shape[0]) < 0.15] = 0  # sums of 0


# heads, page, new, lens, (n_select, n_first, n_last): a token a workgroup, tiles (one and
# several parts), the choice in a launch of its own, groups of up to 40
CASES = [
    ((16, 2, 128), 16, [1, 1, 1], [1, 300, 1001], (12, 1, 2)),
    ((8, 2, 64), 4, [30], [400], (20, 3, 4)),
    ((8, 8, 64), 4, [40, 9], [400, 30], (200, 2, 2)),
    ((16, 1, 256), 8, [9], [900], (7, 3, 4)),
    ((40, 2, 64), 4, [40], [500], (30, 1, 1)),
    ((4, 2, 64), 1, [40], [3000], (100, 5, 9)),
    ((4, 1, 64), 1, [1], [3000], (64, 7, 9)),
    ((24, 1, 80), 1, [1, 2], [9000, 700], (300, 2, 2)),
    ((32, 16, 64), 4, [60], [400], (20, 3, 4)),
    ((16, 16, 64), 1, [170], [2100], (100, 5, 9)),
    ((320, 16, 64), 4, [50], [300], (30, 1, 1)),
    ((4, 2, 96), 1, [1], [14000], (4096, 5, 9)),
]


@pytest.mark.parametrize("heads,page,new,lens,how", CASES)
def test_first_and_last_pages_whatever_their_scales(heads, page, new, lens, how):
    print(f"select {heads} page={page} new={new} lens={lens} {how}", flush=True)
    holes = [(0, 0)] if len(new) > 1 else [(0, (lens[0] - 1) // page)] if lens[0] % 3 == 0 else []
    p = ref.Paged(91, *heads, page, new, lens, holes=holes, pad=3, lead=2)
    both, scale = sel.random_bounds(92, p.pages, p.kv, p.hd)
    spoil(scale, both, np.random.default_rng(93))
    cache, batch = p.device(capi)
    got = torch.full((p.rows, p.kv, how[0]), -7, dtype=torch.int32, device="cuda")
    capi.select_pages(got, p.q.cuda(), torch.from_numpy(both).cuda(), torch.from_numpy(scale).cuda(), batch, cache, *how[1:])
    got, want = got.cpu().numpy(), expected(p, both, scale, *how)
    assert np.array_equal(got, want), [(tuple(x), got[tuple(x)], want[tuple(x)]) for x in np.argwhere(got != want)[:5]]


@pytest.mark.parametrize("new,length", [([1], 400), ([40], 400), ([1], 3000)])
def test_arrays_never_written_leave_the_first_and_last_pages(new, length):
    p = ref.Paged(94, 8, 2, 64, 4, new, [length])
    cache, batch = p.device(capi)
    bounds = torch.zeros((p.pages, 2, 8, 2, 8), dtype=torch.int8, device="cuda")
    scales = torch.full((p.pages, 2), float("nan"), device="cuda")
    got = torch.empty((p.rows, 2, 6), dtype=torch.int32, device="cuda")
    capi.select_pages(got, p.q.cuda(), bounds, scales, batch, cache, 2, 3)
    for t in range(new[0]):
        v = sel.visible(p, length - new[0] + t)
        assert got[t].tolist() == [[0, 1, v - 3, v - 2, v - 1, -1]] * 2


@pytest.mark.parametrize("heads,new,length", [((4, 2, 64), [1], 400), ((4, 2, 64), [1], 1500), ((32, 16, 64), [90], 1500),
                                              ((16, 16, 64), [190], 2500)])
@pytest.mark.parametrize("low,high", [(-np.inf, np.inf), (-1e38, 3.3e38), (-1e38, np.inf), (-np.inf, 3.3e38), (-1e-38, np.inf)])
def test_scores_at_both_ends_of_their_range(heads, new, length, low, high):
    """Many of the largest there are beside some of the smallest: the borders of their keys'
    range lie at the ends of 32 bits."""
    p = ref.Paged(95, *heads, 1, new, [length])
    p.q[:] = 1.0
    rng = np.random.default_rng(96)
    kind = rng.integers(0, 6, (p.pages, p.kv))
    sign = np.where(kind <= 1, -1, 1).astype(np.int8)  # sums of 64 or -64
    both = np.broadcast_to(sign[:, :, None, None, None], (p.pages, p.kv, 8, 2, 8)).copy()
    scale = rng.random(kind.shape).astype(np.float32) + 1
    scale[kind == 0], scale[kind == 5] = -low / 64, high / 64
    cache, batch = p.device(capi)
    for n in (9, 40, 200):
        got = torch.full((p.rows, p.kv, n), -7, dtype=torch.int32, device="cuda")
        capi.select_pages(got, p.q.cuda(), torch.from_numpy(both).cuda(), torch.from_numpy(scale).cuda(), batch, cache, 1, 2)
        assert np.array_equal(got.cpu().numpy(), expected(p, both, scale, n, 1, 2)), n
