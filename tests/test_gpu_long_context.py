"""The operators for long and multimodal contexts together, as a decoder's step runs
them: projections from the library's quantised products, rotation on three axes and the
cache's store, bounds of the pages, the choice of pages, attention over them, the next
token's input from the attention's output."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import selected_reference as sel
from tests import serving_reference as ref
from tests.test_gpu_qk_rope import freqs
from tests.test_gpu_rope_axes import check as check_append
from tests.test_gpu_selected import check_attend, check_select

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, HD, ROOM = 512, 8, 2, 64, 400
SCALE = HD ** -0.5


class Step:
    """A layer over a batch, into buffers of its own; the bounds are the cache's."""

    def __init__(self, p, batch, cache, bounds, scales, n_select):
        rows = p.rows
        half = lambda *shape: torch.zeros(shape, dtype=torch.float16, device="cuda")  # noqa: E731
        self.p, self.batch, self.cache, self.bounds, self.scales = p, batch, cache, bounds, scales
        self.x, self.qkv = half(rows, HIDDEN), half(rows, HEADS + 2 * KV, HD)
        self.q, self.out = half(rows, HEADS, HD), half(rows, HEADS, HD)
        self.lists = torch.zeros((rows, KV, n_select), dtype=torch.int32, device="cuda")
        self.positions = torch.zeros((3, rows), dtype=torch.int32, device="cuda")
        self.axis_of = (torch.arange(HD // 2) % 3).int()
        self.inv_freq = freqs(HD)
        self.on_device = self.inv_freq.cuda(), self.axis_of.cuda()

    def run(self, w_qkv, stream):
        capi.gemm_noalloc(self.qkv, w_qkv, self.x, (HEADS + 2 * KV) * HD, len(self.x), HIDDEN, stream)
        q, k, v = self.qkv[:, :HEADS], self.qkv[:, HEADS:HEADS + KV], self.qkv[:, HEADS + KV:]
        inv_freq, axis_of = self.on_device
        capi.qk_norm_rope_axes(self.q, q, k, v, self.batch, self.cache, inv_freq, self.positions, axis_of, stream=stream)
        capi.kv_bounds(self.bounds, self.scales, self.batch, self.cache, stream)
        capi.select_pages(self.lists, self.q, self.bounds, self.scales, self.batch, self.cache, 1, 2, stream)
        capi.attention_selected_f16(self.out, self.q, self.lists, self.batch, self.cache, SCALE, stream)

    def check(self, both, scales):
        """Each operator of the last run from what it was given; p, both and scales hold
        the cache and its bounds as they were before, and are brought up to now."""
        p, how = self.p, (self.lists.shape[2], 1, 2)
        f = self.qkv.cpu()
        x = f[:, :HEADS], f[:, HEADS:HEADS + KV], f[:, HEADS + KV:]
        check_append(p, x, self.q, self.cache, self.inv_freq, self.positions.cpu(), self.axis_of, None, None, 1e-6, False)
        k, v, _, ks, vs = self.cache.tensors
        p.both = torch.stack([k.cpu(), v.cpu()])
        p.ks, p.vs = (None, None) if ks is None else (ks.cpu(), vs.cpu())
        p.q = self.q.cpu()
        for page, held in sel.touched(p, max_len=ROOM):
            both[page], scales[page] = sel.bounds(p, page, held)
        assert np.array_equal(self.bounds.cpu().numpy(), both) and np.array_equal(self.scales.cpu().numpy(), scales)
        check_select(p, self.lists, both, scales, *how, max_len=ROOM)
        check_attend(p, self.out, self.lists.cpu().numpy(), SCALE)


@pytest.mark.parametrize("page,int8,prompts", [(16, False, [150, 1, 70]), (8, True, [90, 33, 2]), (32, True, [200, 5, 64]),
                                               (4, False, [40, 17, 120])])
def test_prompts_then_decoding_eager_and_replayed(page, int8, prompts):
    """Three prompts of image patches and text prefilled together, then eight tokens
    each: every step against the definitions, then the same eight again as replays of one
    captured step, eager work on another stream between them, which has to leave the same
    lists, outputs and cache."""
    print(f"long context page={page} int8={int8} {prompts}", flush=True)
    g = torch.Generator().manual_seed(141)
    w_qkv = capi.quantize((torch.randn(((HEADS + 2 * KV) * HD, HIDDEN), generator=g) * 0.05).cuda())
    p = ref.Paged(142, HEADS, KV, HD, page, prompts, [ROOM] * 3, int8)
    p.lens, p.seq_lens = list(prompts), torch.tensor(prompts, dtype=torch.int32)
    cache, batch = p.device(capi, max_len=ROOM)
    bounds = torch.zeros((p.pages, KV, HD // 8, 2, 8), dtype=torch.int8, device="cuda")
    scales = torch.zeros((p.pages, KV), device="cuda")
    both, by = bounds.cpu().numpy().copy(), scales.cpu().numpy().copy()
    s = torch.cuda.Stream()

    first = Step(p, batch, cache, bounds, scales, 6)
    first.x.copy_(torch.randn(first.x.shape, generator=g))
    i = torch.cat([torch.arange(n) for n in prompts])
    first.positions.copy_(torch.stack([i // 12, i // 4 % 3, i % 4]).int())
    torch.cuda.synchronize()
    first.run(w_qkv, s)
    torch.cuda.synchronize()
    first.check(both, by)

    d = ref.Paged(142, HEADS, KV, HD, page, [1] * 3, [ROOM] * 3, int8)
    d.table, d.pages, d.both, d.ks, d.vs = p.table, p.pages, p.both, p.ks, p.vs
    d.starts, d.rows = torch.tensor([0, 1, 2, 3], dtype=torch.int32), 3
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    batch = capi.SeqBatch(d.starts.cuda(), lens, 3, 1, ROOM)
    step = Step(d, batch, cache, bounds, scales, 6)
    begin = [t.clone() for t in (*[c for c in cache.tensors if c is not None], bounds, scales)]
    start = first.out.view(-1, HIDDEN)[torch.tensor(np.cumsum(prompts) - 1).cuda()].clone()
    text = torch.tensor([n // 12 + 5 for n in prompts], dtype=torch.int32)  # text goes on behind the image's last row

    def after(n):
        step.x.copy_(start if n == 0 else step.out.view(3, HIDDEN) * 3)
        lens.copy_(torch.tensor([m + n + 1 for m in prompts], dtype=torch.int32))
        step.positions.copy_((text + n).expand(3, 3))
        torch.cuda.synchronize()

    seen = []
    for n in range(8):
        after(n)
        step.run(w_qkv, s)
        torch.cuda.synchronize()
        d.lens = [m + n + 1 for m in prompts]
        d.seq_lens = torch.tensor(d.lens, dtype=torch.int32)
        step.check(both, by)
        seen.append((step.lists.clone(), step.out.clone()))
    end = [t.clone() for t in (*[c for c in cache.tensors if c is not None], bounds, scales)]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step.run(w_qkv, s)
    torch.cuda.synchronize()
    for t, was in zip((*[c for c in cache.tensors if c is not None], bounds, scales), begin):
        t.copy_(was)
    other = torch.empty_like(first.out)
    for n in range(8):
        after(n)
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step.lists, seen[n][0]) and torch.equal(step.out, seen[n][1])
        capi.attention_paged_f16(other, first.q, first.batch, cache, SCALE)
    for t, was in zip((*[c for c in cache.tensors if c is not None], bounds, scales), end):
        assert torch.equal(t.view(torch.int8), was.view(torch.int8))
    capi.release_workspace(s)


def test_a_loaded_prefix_gets_its_bounds_from_a_batch_of_all_its_tokens():
    """Keys that came with their pages: a batch whose new tokens are all of them, no
    arrays behind its rows."""
    p = ref.Paged(143, HEADS, KV, HD, 16, [300, 77], [300, 77])
    cache, batch = p.device(capi)
    bounds = torch.zeros((p.pages, KV, HD // 8, 2, 8), dtype=torch.int8, device="cuda")
    scales = torch.zeros((p.pages, KV), device="cuda")
    capi.kv_bounds(bounds, scales, batch, cache)
    for page, held in sel.touched(p):
        b, s = sel.bounds(p, page, held)
        assert np.array_equal(bounds[page].cpu().numpy(), b) and np.array_equal(scales[page].cpu().numpy(), s)
    assert len(sel.touched(p)) == 19 + 5
