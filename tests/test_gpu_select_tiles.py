"""The choice of pages (rxq4_select_pages) where several tokens share a workgroup: batches
with enough of them, of every group of heads, around the size where one starts to be
taken, against the definition (selected_reference).  Lists have to be equal."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import selected_reference as sel
from tests import serving_reference as ref
from tests.test_gpu_selected import check_select, run_select

pytestmark = pytest.mark.gpu

# heads, page, new, lens, (n_select, n_first, n_last)
TILES = [
    ((32, 8, 128), 16, [100, 3], [1100, 40], (16, 0, 1)),
    ((16, 16, 64), 4, [60, 20, 33], [300, 20, 40], (10, 2, 2)),  # groups of 1: sixteen tokens a tile
    ((32, 16, 64), 8, [50, 3], [600, 90], (10, 2, 2)),           # of 2: eight
    ((48, 16, 96), 8, [50], [700], (30, 0, 0)),
    ((80, 16, 200), 16, [50], [900], (7, 3, 4)),                 # the forced fill the list
    ((56, 8, 128), 32, [100], [1500], (12, 1, 2)),               # of 7: two
    ((256, 16, 64), 4, [50], [300], (9, 1, 1)),                  # of 16: one or two
    ((320, 16, 64), 4, [50], [300], (9, 1, 1)),                  # of 20: two passes
    ((32, 16, 256), 16, [50], [900], (7, 1, 1)),
    ((48, 16, 8), 2, [50], [190], (11, 1, 1)),
    ((32, 32, 16), 1, [50], [400], (1, 0, 1)),
    ((64, 64, 80), 1, [33], [300], (300, 1, 1)),                 # more than there are
    ((64, 64, 80), 1, [33], [300], (297, 1, 1)),                 # the border at the last pages
    ((32, 16, 72), 128, [200], [1000], (3, 1, 1)),
    ((32, 16, 64), 1, [100], [2100], (100, 1, 1)),                # several parts
    ((16, 16, 64), 1, [170], [2100], (100, 1, 1)),
    ((64, 8, 128), 1, [245], [4000], (64, 1, 63)),           # the last pages always
    ((16, 16, 256), 1, [165], [1500], (512, 1, 1)),              # the longest lists of a tile, its most LDS
    ((64, 16, 256), 1, [100], [1500], (512, 1, 1)),
    ((64, 8, 200), 1, [180], [1500], (511, 1, 1)),
    ((16, 4, 64), 1, [490], [9000], (200, 5, 5)),
]


@pytest.mark.parametrize("heads,page,new,lens,how", TILES)
def test_tiles(heads, page, new, lens, how):
    print(f"select {heads} page={page} new={new} lens={lens} {how}", flush=True)
    p = ref.Paged(171, *heads, page, new, lens, pad=3, lead=2)
    both, scale = sel.random_bounds(172, p.pages, p.kv, p.hd)
    check_select(p, run_select(p, both, scale, *how), both, scale, *how)


@pytest.mark.parametrize("heads,new", [((32, 8, 64), 56), ((16, 16, 64), 42), ((48, 4, 64), 112), ((32, 8, 256), 42)])
def test_both_sides_of_the_border(heads, new):
    """A token less takes a token a workgroup on a card of 256 CUs; the lists are the same."""
    p = ref.Paged(173, *heads, 8, [new], [1000])
    both, scale = sel.random_bounds(174, p.pages, p.kv, p.hd)
    want = sel.select(p, both, scale, 12, 1, 2)
    cache, _ = p.device(capi)
    for n in (new - 1, new):
        batch = capi.SeqBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                              torch.tensor([1000 - new + n], dtype=torch.int32, device="cuda"), n, n, 1000)
        got = torch.full((n, p.kv, 12), -7, dtype=torch.int32, device="cuda")
        capi.select_pages(got, p.q[:n].contiguous().cuda(), torch.from_numpy(both).cuda(), torch.from_numpy(scale).cuda(),
                          batch, cache, 1, 2)
        assert np.array_equal(got.cpu().numpy(), want[:n]), n


@pytest.mark.parametrize("seqs,new", [(60, 2), (40, 3), (33, 9)])
def test_drafts_of_many_sequences(seqs, new):
    rng = np.random.default_rng(seqs)
    lens = [new + int(x) for x in rng.integers(0, 900, seqs)]
    p = ref.Paged(175, 32, 8, 64, 8, [new] * seqs, lens, pad=2, lead=3)
    both, scale = sel.random_bounds(176, p.pages, p.kv, p.hd)
    check_select(p, run_select(p, both, scale, 12, 1, 2), both, scale, 12, 1, 2)


@pytest.mark.parametrize("group,kv,new", [(1, 16, 100), (2, 16, 50), (4, 16, 50), (8, 8, 100), (16, 8, 100), (24, 8, 100)])
def test_ties_in_tiles(group, kv, new):
    p = ref.Paged(177, kv * group, kv, 64, 4, [new], [700])
    both, scale = sel.random_bounds(178, 6, kv, 64)
    pick = np.random.default_rng(179).integers(0, 6, p.pages)
    both, scale = both[pick], scale[pick]
    p.q[::3] = 0
    for how in ((20, 1, 1), (100, 2, 3), (1, 0, 0)):
        check_select(p, run_select(p, both, scale, *how), both, scale, *how)


def test_crowded_scores_in_tiles():
    p = ref.Paged(180, 8, 4, 64, 1, [480], [1500])
    both, scale = sel.random_bounds(181, p.pages, 4, 64)
    scale *= 1 + 1e-3 * np.random.default_rng(182).random(scale.shape).astype(np.float32)
    scale[p.table[0, 5], :], scale[p.table[0, 11], :] = 1e4, 1e3
    for n in (100, 300, 500):
        check_select(p, run_select(p, both, scale, n, 1, 1), both, scale, n, 1, 1)


@pytest.mark.parametrize("kind", ["rising", "falling", "alike", "few"])
def test_parts_of_tiles_whose_scores_rise_fall_or_tie(kind):
    p = ref.Paged(183, 16, 8, 64, 1, [245], [4000], holes=[(0, j) for j in range(4000) if kind == "few" and j % 97])
    both, scale = sel.random_bounds(184, 1, 8, 64)
    both = np.repeat(both, p.pages, 0)
    rank = np.empty(p.pages)
    rank[p.table[0].numpy().clip(0, p.pages - 1)] = np.arange(4000)
    slope = {"rising": 1 + rank / 100, "falling": 100 - rank / 100, "alike": 0 * rank + 1, "few": 1 + (rank * 7919 % 1000)}[kind]
    scale = (scale * slope[:, None]).astype(np.float32)
    for how in ((40, 1, 1), (256, 2, 3)):
        check_select(p, run_select(p, both, scale, *how), both, scale, *how)


def test_holes_padding_and_limits_in_tiles():
    new, lens = [60, 1, 45], [1260, 1201, 1245]
    holes = [(0, 0), (0, 1), (0, 7), (0, 1259 // 16), (2, 5)]
    p = ref.Paged(185, 64, 16, 64, 16, new, lens, holes=holes, pad=2, lead=1)
    both, scale = sel.random_bounds(186, p.pages, 16, 64)
    for how in ((12, 2, 3), (73, 1, 1)):
        for limits in ({}, {"max_len": 900}, {"max_new": 5}, {"max_len": 1 << 20}):
            check_select(p, run_select(p, both, scale, *how, **limits), both, scale, *how, **limits)


def test_tiles_that_see_nothing():
    p = ref.Paged(187, 32, 16, 64, 16, [60, 20, 1], [20, 40, 0], holes=[(1, 0), (1, 1), (1, 2)])
    both, scale = sel.random_bounds(188, p.pages, 16, 64)
    got = run_select(p, both, scale, 5, 1, 1)
    check_select(p, got, both, scale, 5, 1, 1)
    assert (got[:40] == -1).all() and (got[60:] == -1).all()


@pytest.mark.parametrize("starts", [[0, 50, 30], [-4, 20, 90], [0, 100000, 100001], [70, 20, 10], [2 ** 31 - 1] * 3, [-2 ** 31] * 3])
@pytest.mark.parametrize("lens", [[64, 64], [2 ** 31 - 1, -2 ** 31]])
def test_starts_and_lengths_outside_their_limits_in_tiles(starts, lens):
    p = ref.Paged(189, 32, 16, 64, 16, [40, 24], [64, 64])
    cache, batch = p.device(capi)
    batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
    batch.tensors[1].copy_(torch.tensor(lens, dtype=torch.int32))
    both, scale = (torch.from_numpy(a).cuda() for a in sel.random_bounds(190, p.pages, 16, 64))
    lists = torch.full((p.rows + 20, 16, 3), -9, dtype=torch.int32, device="cuda")
    capi.select_pages(lists[10:-10], p.q.cuda(), both, scale, batch, cache)
    assert (lists[:10] == -9).all() and (lists[-10:] == -9).all()
    assert ((lists >= -1) & (lists < 4) | (lists == -9)).all()


def test_tiles_replayed_and_on_another_stream():
    p = ref.Paged(191, 32, 8, 128, 16, [90, 20], [1500, 700])
    both, scale = sel.random_bounds(192, p.pages, p.kv, p.hd)
    want = sel.select(p, both, scale, 20, 1, 2)
    cache, batch = p.device(capi)
    q, b, s = p.q.cuda(), torch.from_numpy(both).cuda(), torch.from_numpy(scale).cuda()
    out = torch.full((p.rows, 8, 20), -7, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        capi.select_pages(out, q, b, s, batch, cache, 1, 2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            capi.select_pages(out, q, b, s, batch, cache, 1, 2)
        for _ in range(3):
            out.fill_(-7)
            graph.replay()
            stream.synchronize()
            assert np.array_equal(out.cpu().numpy(), want)
