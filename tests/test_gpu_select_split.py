"""The choice of pages (rxq4_select_pages) in two launches, scores through the stream's
workspace: groups of more than 8 and of more than 16 heads, which pass over the scores
several times, after calls that left others there."""
from __future__ import annotations

import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import selected_reference as sel
from tests import serving_reference as ref
from tests.test_gpu_selected import check_select, run_select

pytestmark = pytest.mark.gpu

# heads, page, new, lens, (n_select, n_first, n_last)
SPLIT = [
    ((40, 1, 64), 1, [1], [3000], (64, 1, 1)),
    ((16, 1, 128), 1, [1, 2], [9000, 700], (33, 2, 2)),
    ((20, 1, 256), 1, [1], [2000], (9, 1, 1)),
    ((9, 1, 80), 1, [1, 1, 1], [2000, 5, 700], (100, 0, 0)),
    ((64, 2, 96), 4, [1, 3], [4000, 2500], (40, 1, 2)),
    ((33, 1, 8), 1, [2], [12000], (600, 3, 3)),
]


def stale(heads):
    """Scores above those of any other call, at every place."""
    p = ref.Paged(201, *heads, 1, [1, 1], [14000, 14000])
    both, scale = sel.random_bounds(202, p.pages, p.kv, p.hd)
    run_select(p, both, scale * 1e20, 8, 1, 1)


@pytest.mark.parametrize("heads,page,new,lens,how", SPLIT)
def test_large_groups_after_other_calls(heads, page, new, lens, how):
    print(f"select {heads} page={page} new={new} lens={lens} {how}", flush=True)
    p = ref.Paged(203, *heads, page, new, lens, pad=3, lead=2, holes=[(0, 7)])
    both, scale = sel.random_bounds(204, p.pages, p.kv, p.hd)
    want = sel.select(p, both, scale, *how)
    for _ in range(2):
        stale(heads)
        check_select(p, run_select(p, both, scale, *how), both, scale, *how)
    assert (want[p.starts[0]] >= 0).any()


def test_replayed_among_other_calls_of_the_stream():
    heads, how = (40, 1, 64), (64, 1, 1)
    p = ref.Paged(205, *heads, 1, [1], [3000])
    both, scale = sel.random_bounds(206, p.pages, 1, 64)
    want = torch.from_numpy(sel.select(p, both, scale, *how))
    cache, batch = p.device(capi)
    q, b, s = p.q.cuda(), torch.from_numpy(both).cuda(), torch.from_numpy(scale).cuda()
    out = torch.empty((1, 1, 64), dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        capi.select_pages(out, q, b, s, batch, cache, 1, 1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            capi.select_pages(out, q, b, s, batch, cache, 1, 1)
        for _ in range(3):
            stale(heads)
            out.fill_(-7)
            graph.replay()
            stream.synchronize()
            assert torch.equal(out.cpu(), want)
