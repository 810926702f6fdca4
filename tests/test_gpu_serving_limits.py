"""The serving operators at the ends of what they accept: positions, sequences, rows
and heads (rxq4.h's RXQ4_MAX_*), and first calls inside a capture."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import serving_reference as ref
from tests.test_gpu_paged import attend, check
from tests.test_gpu_qk_rope import check as check_append, freqs, inputs, run

pytestmark = pytest.mark.gpu
POSITIONS, SEQS, ROWS, HEADS = 1 << 24, 65536, 1 << 20, 1024


@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("page,int8,table", [(1024, False, True), (1, False, True), (16, False, False), (1024, True, True)])
def test_all_positions(new, page, int8, table):
    """2^24 positions of one head, the last `new` of them the tokens': the sums of 64
    chunks of 2^18.  A token's output is a mean of values that all weigh the same but
    one: scores are 0, and 10 at position 12345678."""
    print(f"positions page={page} int8={int8} table={table} new={new}", flush=True)
    n, hd, at, scale = POSITIONS, 16 if int8 else 8, 12345678, 0.5
    pages = n // page
    g = torch.Generator(device="cuda").manual_seed(61)
    k = torch.zeros((pages, page, 1, hd), dtype=torch.int8 if int8 else torch.float16, device="cuda")
    v = torch.randint(-127, 128, k.shape, generator=g, device="cuda").to(k.dtype)
    place = torch.arange(n, device="cuda").view(pages, page)  # which position is at a slot
    order = None
    if table:
        order = torch.randperm(pages, generator=g, device="cuda").int()
        place[order.long()] = place.clone()
    k[place == at] = 4
    scales = (torch.ones((pages, page, 1), device="cuda"),) * 2 if int8 else (None, None)
    q = torch.zeros((new, 1, hd), dtype=torch.float16, device="cuda")
    q[..., :5] = 1.0  # scores 4 * 5 * 0.5
    cache = capi.PagedKV(k, v, None if order is None else order[None], *scales)
    batch = capi.SeqBatch(*(torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, new], [n])), new, new, n)
    out = torch.empty_like(q)
    capi.attention_paged_f16(out, q, batch, cache, scale)
    # the values of positions [0, n), then each token's sums
    values = v.view(n, hd) if order is None else v[order.long()].view(n, hd)
    e10 = float(np.exp(10.0))
    total, size = (torch.zeros(hd, dtype=torch.float64, device="cuda") for _ in range(2))
    for part in values[:n - new].split(1 << 20):
        total += part.double().sum(0)
        size += part.double().abs().sum(0)
    total += (e10 - 1) * values[at].double()
    size += (e10 - 1) * values[at].double().abs()
    weight = n - new + e10 - 1
    for t in range(new):
        total, size, weight = total + values[n - new + t].double(), size + values[n - new + t].double().abs(), weight + 1
        want = total / weight
        # weights off by (hd + 12) u S, S = 10.  Of the 64 chunks 63 have equal weights, whose sums
        # are of whole numbers below 2^24: exact; the other, at most 1 / 32 of the weight, sums 2^14
        # terms a lane.  64 chunks are joined
        rel = 2 * ((hd + 12) * ref.U * 10 + (2 ** 14 // 32 + 128) * ref.U + 2.0 ** -21)
        bound = rel * size / weight + ref.H16 * want.abs() + ref.TINY16
        assert ((out[t, 0].double() - want).abs() <= bound).all(), ((out[t, 0].double() - want).abs() / bound).max()


@pytest.mark.parametrize("int8", [False, True])
def test_all_sequences(int8):
    """65536 of them, every 7th empty: a token that sees one position gets its value."""
    n, hd = SEQS, 16
    new = np.where(np.arange(n) % 7 == 3, 0, 1)
    lens = torch.from_numpy(new.astype(np.int32))
    starts = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    rows = int(starts[-1])
    g = torch.Generator().manual_seed(62)
    x = torch.randn((rows, 1, hd), generator=g)
    table = torch.randperm(n, generator=g).int()[:, None]
    k = torch.zeros((n, 4, 1, hd), dtype=torch.int8 if int8 else torch.float16, device="cuda")
    v = torch.zeros_like(k)
    scales = [torch.zeros((n, 4, 1), device="cuda") if int8 else None for _ in range(2)]
    cache = capi.PagedKV(k, v, table.cuda(), *scales)
    batch = capi.SeqBatch(starts.cuda(), lens.cuda(), rows, 1, 1)
    q, out = (torch.empty((rows, 1, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    xs = x.cuda()
    capi.qk_norm_rope(q, xs, xs, xs, batch, cache, freqs(hd).cuda())
    assert torch.equal(q, xs.half())  # position 0
    capi.attention_paged_f16(out, q, batch, cache, 0.25)
    stored = v[table[:, 0].long().cuda()[torch.from_numpy(new).cuda() == 1], 0].float()
    if int8:
        stored = stored * scales[1][table[:, 0].long().cuda()[torch.from_numpy(new).cuda() == 1], 0, :, None]
        assert (stored - xs).abs().max() <= xs.abs().max() / 254 * (1 + 2.0 ** -14)
    else:
        assert torch.equal(stored, xs.half().float())
    assert ((out.float() - stored).abs() <= 2.0 ** -10 * stored.abs() + ref.TINY16).all()


def test_all_rows_of_one_sequence():
    """2^20 tokens stored and rotated at once, and their attention over the first 64
    positions' values (max_len): means, sums of 64 in fp32 (64 u of the largest and the
    division, 2^-17 of it)."""
    n, hd = ROWS, 8
    g = torch.Generator().manual_seed(63)
    x = torch.randn((n, 1, hd), generator=g).half().cuda()
    k = torch.zeros((n // 1024, 1024, 1, hd), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    cache = capi.PagedKV(k, v, torch.arange(n // 1024, dtype=torch.int32, device="cuda")[None])
    one = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, n], [n])]
    q = torch.empty_like(x)
    capi.qk_norm_rope(q, x, x, x, capi.SeqBatch(*one, n, n, n), cache, freqs(hd).cuda())
    assert torch.equal(v.view(n, 1, hd), x)
    at = torch.tensor([0, 1, 65537, n - 1])
    want, bound = ref.rope(x[at.cuda()].cpu().double().numpy(), None, 0.0, at.numpy(), freqs(hd).numpy(), False)
    off = np.abs(q[at.cuda()].cpu().double().numpy() - want)
    assert (off <= bound + ref.H16 * np.abs(want) + ref.TINY16).all()
    out = torch.full_like(q, 7.0)
    zero = torch.zeros_like(q)
    capi.attention_paged_f16(out, zero, capi.SeqBatch(*one, n, n, 64), cache, 0.5)
    mean = x[:64, 0].double().cumsum(0) / torch.arange(1, 65, device="cuda", dtype=torch.float64)[:, None]
    mean = mean[torch.arange(n, device="cuda").clamp(max=63)]
    size = x[:64, 0].double().abs().max()
    assert ((out[:, 0].double() - mean).abs() <= 2.0 ** -11 * mean.abs() + 2.0 ** -17 * size + ref.TINY16).all()


@pytest.mark.parametrize("kv", [1, 1024, 512])
@pytest.mark.parametrize("int8", [False, True])
def test_all_heads(kv, int8):
    p = ref.Paged(64, HEADS, kv, 16, 8, [1, 2, 20], [70, 9, 33], int8)
    check(p, attend(p, 0.25), 0.25)
    args = (freqs(16), None, None, 1e-6, True)
    x = inputs(p, torch.float16, True)
    got, cache = run(p, x, *args)
    check_append(p, x, got, cache, *args)


def test_all_rows_of_logits():
    n = ROWS
    r = np.random.default_rng(65)
    l = r.standard_normal((n, 3)).astype(np.float32)
    u = r.random(n).astype(np.float32)
    ids = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    capi.sample_f32(ids, torch.from_numpy(l).cuda(), torch.from_numpy(u).cuda())
    order = np.argsort(-l, axis=1, kind="stable")
    w = np.take_along_axis(np.exp(l.astype(np.float64) - l.max(1, keepdims=True)), order, 1)
    c = w.cumsum(1)
    x = u.astype(np.float64) * c[:, 2]
    far = np.abs(c - x[:, None]).min(1) > 2.0 ** -40
    want = np.take_along_axis(order, np.minimum((c <= x[:, None]).sum(1), 2)[:, None], 1)[:, 0]
    assert far.sum() > n - 10
    assert (ids.cpu().numpy() == want)[far].all()


@pytest.mark.parametrize("new,lens,hd,page,int8", [([1, 1], [3000, 5], 256, 8, True), ([40, 1], [2000, 9], 200, 4, True),
                                                   ([70], [2500], 96, 2, False)])
def test_first_calls_inside_a_capture(new, lens, hd, page, int8):
    """A stream without a workspace, kernels that no other test launches this way."""
    hd = hd - hd % 16 if int8 else hd
    p = ref.Paged(66, 4, 2, hd, page, new, lens, int8)
    cache, batch = p.device(capi)
    q, out = p.q.cuda(), torch.full((p.rows, 4, hd), 7.0, dtype=torch.float16, device="cuda")
    logits = torch.from_numpy(np.random.default_rng(67).standard_normal((2, 5003)).astype(np.float32)).cuda()
    u, ids = torch.tensor([0.25, 0.75], device="cuda"), torch.full((2,), -7, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.attention_paged_f16(out, q, batch, cache, 0.0625, stream=s)
        capi.sample_f32(ids, logits, u, stream=s)
    for _ in range(3):
        out.fill_(7.0)
        ids.fill_(-7)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        check(p, out, 0.0625)
        assert ids.tolist() == [ref.sample(a, x) for a, x in zip(logits.cpu().numpy(), u.cpu().numpy())]
    del graph
    capi.release_workspace(s)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [256, 300])
def test_many_decoding_with_one_long_and_a_capacity(n, int8):
    """Chunks from the lengths and, past 256 sequences, from max_len and the table,
    both far above the lengths."""
    lens = [50 + i % 90 for i in range(n)]
    lens[n // 3] = 13000
    p = ref.Paged(68, 4, 1, 64, 16, [1] * n, lens, int8)
    p.table = torch.cat([p.table, torch.full((n, 8192 - p.table.shape[1]), -1, dtype=torch.int32)], 1)
    check(p, attend(p, 0.125, max_len=131072), 0.125)


@pytest.mark.parametrize("pad", [0, 600, 4000])
@pytest.mark.parametrize("decodes", [0, 520])
def test_a_short_chunk_after_a_long_context_among_many_rows(pad, decodes):
    """Split, and whole where decoding or padding rows are many."""
    p = ref.Paged(69, 16, 2, 64, 16, [16] + [1] * decodes, [5000] + [20] * decodes, pad=pad)
    check(p, attend(p, 0.125), 0.125)
