"""The serving operators together, as a decoder's step runs them: token rows and
projections from the library's quantised products, head norms, rotation and the
cache's store, attention over the pages, the next token drawn on the device."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import serving_reference as ref
from tests.test_gpu_paged import check as check_attention
from tests.test_gpu_qk_rope import check as check_append, freqs

pytestmark = pytest.mark.gpu
HIDDEN, VOCAB, HEADS, KV, HD, ROOM = 512, 1000, 8, 2, 64, 200
SCALE = HD ** -0.5


class Step:
    """A layer and the head over a batch, into buffers of its own."""

    def __init__(self, rows, batch, cache, weights, last, seed):
        self.rows, self.batch, self.cache, self.weights, self.last = rows, batch, cache, weights, last
        n = last.numel()
        half = lambda *shape: torch.zeros(shape, dtype=torch.float16, device="cuda")  # noqa: E731
        self.x, self.qkv = half(rows, HIDDEN), half(rows, HEADS + 2 * KV, HD)
        self.q, self.out, self.top = half(rows, HEADS, HD), half(rows, HEADS, HD), half(n, HIDDEN)
        self.logits = torch.zeros((n, VOCAB), device="cuda")
        g = torch.Generator().manual_seed(seed)
        self.inv_freq = freqs(HD)
        self.norms = [1 + 0.2 * torch.randn(HD, generator=g) for _ in range(2)]
        self.on_device = [t.cuda() for t in (self.inv_freq, *self.norms)]
        self.temperature = torch.tensor([0.0, 0.8, 1.3], device="cuda")[:n].contiguous()
        self.top_k = torch.tensor([0, 40, 0], dtype=torch.int32, device="cuda")[:n].contiguous()
        self.top_p = torch.tensor([1.0, 0.9, 0.95], device="cuda")[:n].contiguous()

    def run(self, tokens, u, ids, stream):
        embed, w_qkv, w_head = self.weights
        capi.embed_rows_f16(self.x, embed, VOCAB, tokens, HIDDEN, stream)
        capi.gemm_noalloc(self.qkv, w_qkv, self.x, (HEADS + 2 * KV) * HD, self.rows, HIDDEN, stream)
        q, k, v = self.qkv[:, :HEADS], self.qkv[:, HEADS:HEADS + KV], self.qkv[:, HEADS + KV:]
        inv_freq, qw, kw = self.on_device
        capi.qk_norm_rope(self.q, q, k, v, self.batch, self.cache, inv_freq, qw, kw, 1e-6, False, stream)
        capi.attention_paged_f16(self.out, self.q, self.batch, self.cache, SCALE, stream)
        with torch.cuda.stream(stream):
            torch.index_select(self.out.view(self.rows, HIDDEN), 0, self.last, out=self.top)
        capi.gemm_noalloc(self.logits, w_head, self.top, VOCAB, len(self.top), HIDDEN, stream)
        capi.sample_f32(ids, self.logits, u, self.temperature, self.top_k, self.top_p, stream=stream)

    def check(self, p, u, ids):
        """Each operator of the last run against 64 bits, from what it was given; p
        holds the cache as it was before."""
        f = self.qkv.cpu()
        x = f[:, :HEADS], f[:, HEADS:HEADS + KV], f[:, HEADS + KV:]
        check_append(p, x, self.q, self.cache, self.inv_freq, *self.norms, 1e-6, False)
        k, v, _, ks, vs = self.cache.tensors
        p.both = torch.stack([k.cpu(), v.cpu()])
        p.ks, p.vs = (None, None) if ks is None else (ks.cpu(), vs.cpu())
        p.q = self.q.cpu()
        check_attention(p, self.out, SCALE)
        settings = [t.tolist() for t in (self.temperature, self.top_k, self.top_p)]
        logits = self.logits.cpu().numpy()
        assert np.isfinite(logits).all()
        assert ids.tolist() == [ref.sample(l, x, *s) for l, x, *s in zip(logits, u.cpu().numpy(), *settings)]


@pytest.mark.parametrize("page,int8", [(16, False), (8, True), (64, True), (4, False)])
def test_prompts_then_decoding_eager_and_replayed(page, int8):
    """Three prompts prefilled together, then twelve tokens each: every step against
    64 bits, then the same twelve again as replays of one captured step, which has to
    give the same tokens and the same cache."""
    print(f"serving page={page} int8={int8}", flush=True)
    g = torch.Generator().manual_seed(41)
    weights = [capi.quantize((torch.randn((rows, HIDDEN), generator=g) * scale).cuda())
               for rows, scale in ((VOCAB, 1.0), ((HEADS + 2 * KV) * HD, 0.05), (VOCAB, 0.3))]
    prompts, steps = [40, 1, 133], 12
    p = ref.Paged(43, HEADS, KV, HD, page, prompts, [ROOM] * 3, int8)
    p.lens, p.seq_lens = list(prompts), torch.tensor(prompts, dtype=torch.int32)
    cache, batch = p.device(capi, max_len=ROOM)
    s = torch.cuda.Stream()
    us = torch.rand((steps + 1, 3), generator=g).cuda()
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")

    tokens = torch.randint(0, VOCAB, (sum(prompts),), generator=g).int().cuda()
    last = (p.starts[1:] - 1).cuda()
    torch.cuda.synchronize()
    prefill = Step(sum(prompts), batch, cache, weights, last, 47)
    prefill.run(tokens, us[0], ids, s)
    torch.cuda.synchronize()
    prefill.check(p, us[0], ids)

    p.new, p.rows, p.starts = [1] * 3, 3, torch.arange(4, dtype=torch.int32)
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    decoding = capi.SeqBatch(p.starts.cuda(), lens, 3, 1, ROOM)
    step = Step(3, decoding, cache, weights, torch.arange(3, device="cuda"), 47)
    before = [None if t is None else t.clone() for t in cache.tensors], ids.clone()
    u = torch.zeros(3, device="cuda")
    torch.cuda.synchronize()

    def one():
        with torch.cuda.stream(s):
            lens.add_(1)
        step.run(ids, u, ids, s)

    said = []
    for i in range(steps):
        u.copy_(us[1 + i])
        torch.cuda.synchronize()
        one()
        torch.cuda.synchronize()
        p.lens = [n + 1 + i for n in prompts]
        step.check(p, u, ids)
        said.append(ids.tolist())
    after = [None if t is None else t.clone() for t in cache.tensors]

    def back():
        for t, b in zip(cache.tensors, before[0]):
            if t is not None:
                t.copy_(b)
        ids.copy_(before[1])
        lens.copy_(torch.tensor(prompts, dtype=torch.int32))
        torch.cuda.synchronize()

    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        one()
    back()
    again = []
    for i in range(steps):
        u.copy_(us[1 + i])
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        again.append(ids.tolist())
    assert again == said
    for t, b in zip(cache.tensors, after):
        assert t is None or torch.equal(t, b)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_a_table_without_entries(new, int8):
    """No position has a slot: nothing is stored, and every token sees nothing."""
    p = ref.Paged(51, HEADS, KV, HD, 16, [new], [new], int8)
    p.table = p.table[:, :0]
    cache, batch = p.device(capi)
    before = [None if t is None else t.clone() for t in cache.tensors]
    g = torch.Generator().manual_seed(52)
    x = [torch.randn((new, n, HD), generator=g).half().cuda() for n in (HEADS, KV, KV)]
    q, out = (torch.full((new, HEADS, HD), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    capi.qk_norm_rope(q, *x, batch, cache, freqs(HD).cuda())
    capi.attention_paged_f16(out, q, batch, cache, SCALE)
    assert not out.any() and not (q == 7.0).any()
    for t, b in zip(cache.tensors, before):
        assert t is None or torch.equal(t, b)
