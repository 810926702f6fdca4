"""GPU attention over a paged cache (rxq4_attention_paged_f16) against its
definition in 64 bits (serving_reference.attend, which derives the bounds)."""
from __future__ import annotations

import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def attend(p, scale, cache=None, batch=None, out=None, **limits):
    if cache is None:
        cache, batch = p.device(capi, **limits)
    out = torch.full((p.rows, p.heads, p.hd), 7.0, dtype=torch.float16, device="cuda") if out is None else out
    capi.attention_paged_f16(out, p.q.cuda(), batch, cache, scale)
    return out


def check(p, got, scale):
    want, bound = ref.attend(p, scale)
    got = got.cpu().double()
    mine = ~torch.isnan(want)
    assert ((got - want).abs() <= bound)[mine].all(), ((got - want).abs() / bound)[mine].max()
    assert (got[~mine] == 7.0).all()  # rows of no sequence
    norm = want[mine].norm()
    assert (got - want)[mine].norm() <= ref.H16 * norm + 1e-9


# heads, KV heads, head_dim, page size, int8, new tokens, lengths
CASES = [
    # decoding: one position, page borders, long, several
    ((16, 2, 128), 16, False, [1], [1]),
    ((16, 2, 128), 16, False, [1, 1, 1, 1, 1], [16, 17, 64, 65, 1000]),
    ((32, 8, 128), 64, False, [1, 1, 1], [5000, 63, 129]),
    ((32, 8, 128), 16, True, [1, 1, 1, 1], [3000, 1, 200, 257]),
    ((28, 4, 128), 32, False, [1, 1], [2000, 999]),
    ((8, 8, 64), 1, False, [1, 1], [130, 70]),
    ((8, 2, 64), 4, True, [1, 1], [130, 1100]),
    ((8, 4, 80), 8, False, [1, 1, 1], [333, 64, 1]),
    ((8, 4, 80), 8, True, [1, 1], [333, 650]),
    ((6, 2, 96), 128, False, [1, 1], [700, 127]),
    ((4, 1, 256), 16, False, [1, 1], [2100, 3]),
    ((4, 4, 256), 256, True, [1, 1], [600, 256]),
    ((3, 1, 8), 2, False, [1, 2], [9, 200]),
    ((2, 2, 16), 16, True, [1, 3], [40, 70]),
    ((5, 1, 200), 16, False, [1, 7], [90, 300]),
    ((32, 1, 128), 16, False, [1, 1], [1800, 40]),    # a group of 32
    ((40, 1, 64), 32, False, [1, 2], [500, 90]),      # and of 40
    # drafts
    ((28, 4, 128), 32, False, [5, 3, 6, 1], [1500, 64, 300, 77]),
    ((8, 8, 128), 16, False, [2, 16, 17], [18, 1000, 17]),
    ((16, 2, 128), 1024, True, [4, 4], [3000, 5]),
    # chunks
    ((16, 2, 128), 16, False, [64], [64]),
    ((16, 2, 128), 16, False, [100], [1100]),
    ((32, 8, 128), 64, False, [130, 33, 257], [130, 700, 300]),
    ((32, 8, 128), 32, True, [130, 65], [400, 65]),
    ((8, 8, 64), 8, False, [70, 200], [75, 500]),
    ((8, 4, 80), 1, False, [90], [150]),
    ((8, 4, 80), 16, True, [90, 44], [150, 300]),
    ((12, 2, 96), 4, False, [77], [300]),
    ((4, 1, 256), 16, False, [90, 30], [350, 30]),
    ((4, 2, 256), 64, True, [70], [200]),
    ((6, 6, 48), 2, False, [80], [81]),
    # mixed: chunks, drafts, decoding, a sequence without new tokens
    ((8, 4, 80), 8, True, [150, 1, 1, 0, 3, 60], [300, 500, 1, 90, 10, 2000]),
    ((16, 2, 128), 16, False, [1, 200, 1, 0, 40, 1, 2], [900, 200, 3000, 0, 41, 64, 2]),
    ((32, 8, 128), 64, False, [1] * 70 + [40], [1 + 13 * i for i in range(70)] + [333]),
]


@pytest.mark.parametrize("heads,page,int8,new,lens", CASES)
def test_against_64_bits(heads, page, int8, new, lens):
    print(f"paged attention {heads} page={page} int8={int8} new={new} lens={lens}", flush=True)
    p = ref.Paged(11, *heads, page, new, lens, int8)
    scale = heads[2] ** -0.5
    check(p, attend(p, scale), scale)


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [700, 40, 1]), ([33, 1], [300, 100])])
@pytest.mark.parametrize("int8", [False, True])
def test_pages_apart_padding_and_larger_limits(new, lens, int8):
    """K and V pages alternating in one allocation, rows of no sequence around the
    batch, limits far above what the batch holds."""
    p = ref.Paged(12, 16, 2, 128, 16, new, lens, int8, pad=5, lead=2, apart=True)
    check(p, attend(p, 0.09, max_new=200, max_len=100000), 0.09)


def test_int8_without_scales():
    p = ref.Paged(13, 8, 2, 64, 16, [1, 40], [300, 90], True, scales=False)
    check(p, attend(p, 0.0005), 0.0005)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
@pytest.mark.parametrize("new", [1, 30])
def test_scales(scale, new):
    p = ref.Paged(14, 8, 2, 64, 16, [new], [400])
    check(p, attend(p, scale), scale)


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [90, 70]])
@pytest.mark.parametrize("int8", [False, True])
def test_holes_are_not_seen(new, int8):
    """Pages freed at a sequence's start, in it, and under the new tokens."""
    lens = [n + 400 for n in new]
    last = [(n - 1) // 16 for n in lens]
    p = ref.Paged(15, 16, 4, 64, 16, new, lens, int8, holes=[(0, 0), (0, 1), (0, 7), (1, last[1]), (1, 5)])
    check(p, attend(p, 0.125), 0.125)


def test_nothing_to_see_gives_zeros():
    """Every page a hole; more new tokens than positions; length 0."""
    p = ref.Paged(16, 8, 2, 64, 16, [1, 40, 5, 1, 30], [40, 20, 2, 0, 64], holes=[(0, 0), (0, 1), (0, 2)] +
                  [(4, j) for j in range(4)])
    got = attend(p, 0.125)
    check(p, got, 0.125)
    assert not got[:1].any() and not got[1:21].any() and not got[-30:].any()


def test_table_shorter_than_a_sequence():
    """Positions past the table are not seen."""
    p = ref.Paged(17, 8, 2, 64, 16, [1, 20], [64, 64])
    p.seq_lens = p.seq_lens + 10
    p.lens = [n + 10 for n in p.lens]
    check(p, attend(p, 0.125), 0.125)


def test_limits_bound_what_is_computed():
    """New tokens past max_new are left alone; positions past max_len not seen."""
    p = ref.Paged(18, 8, 2, 64, 16, [40], [300])
    got = attend(p, 0.125, max_new=24)
    want, bound = ref.attend(p, 0.125)
    assert ((got.cpu().double() - want).abs() <= bound)[:24].all()
    assert (got[24:] == 7.0).all()
    got = attend(p, 0.125, max_len=256)
    p.table = p.table[:, :16]  # 256 positions
    check(p, got, 0.125)


@pytest.mark.parametrize("starts", [[0, 5, 3], [-4, 2, 9], [0, 100000, 100001], [7, 2, 1], [2 ** 31 - 1] * 3])
def test_starts_outside_the_rows_write_nothing_outside(starts):
    p = ref.Paged(19, 8, 2, 64, 16, [4, 5], [64, 64])
    cache, batch = p.device(capi)
    batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
    big = torch.full((p.rows + 20, 8, 64), 7.0, dtype=torch.float16, device="cuda")
    capi.attention_paged_f16(big[10:-10], p.q.cuda(), batch, cache, 0.125)
    assert (big[:10] == 7.0).all() and (big[-10:] == 7.0).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("new,length", [(1, 100), (3, 100), (20, 150), (100, 333)])
@pytest.mark.parametrize("hd", [64, 80, 128])
def test_infinities_and_nan_in_places_not_seen(bad, new, length, hd):
    """V (and K) of the later new tokens, of slots past the end, of other pages: no
    earlier token's row changes; the tokens that see them get them."""
    p = ref.Paged(20, 8, 2, hd, 16, [new], [length], spare=3)
    clean = attend(p, 0.125).cpu()
    slots = p.slots(0, length)
    rest = torch.ones(p.pages * 16, dtype=torch.bool)
    rest[slots] = False
    k, v = p.both[0].view(-1, 2, hd), p.both[1].view(-1, 2, hd)
    k[rest], v[rest] = bad, bad
    assert torch.equal(attend(p, 0.125).cpu(), clean)
    at = length - (new + 1) // 2  # a position of the new ones
    if new > 1:
        v[slots[at], 0, 5] = bad
        got = attend(p, 0.125).cpu()
        first = at - (length - new)  # the first token that sees it
        assert torch.equal(got[:first], clean[:first])
        hit = got[first:, :4, 5].float()
        assert torch.isnan(hit).all() if bad != bad else (hit == bad).all()
        got[first:, :4, 5] = clean[first:, :4, 5]
        assert torch.isfinite(got).all()


def test_infinite_int8_scales_in_places_not_seen():
    p = ref.Paged(21, 8, 2, 64, 16, [50], [120], True)
    clean = attend(p, 0.125).cpu()
    slots = p.slots(0, 120)
    p.vs.view(-1, 2)[slots[100], 1] = float("nan")
    p.ks.view(-1, 2)[slots[119], 0] = float("nan")
    got = attend(p, 0.125).cpu()
    assert torch.equal(got[:30], clean[:30])
    assert torch.isnan(got[30:, 4:]).all() and torch.isfinite(got[:49, :4]).all()
    assert torch.isnan(got[49, :4]).all()


def test_a_row_does_not_depend_on_its_batch():
    """The same sequence alone and among others (within the bounds, not bit for
    bit: the split of its positions follows the batch)."""
    p = ref.Paged(22, 16, 2, 128, 16, [1, 1, 150, 1], [600, 3000, 400, 40])
    check(p, attend(p, 0.09), 0.09)
    q = ref.Paged(22, 16, 2, 128, 16, [1], [600])
    check(q, attend(q, 0.09), 0.09)


def test_results_repeat_bit_for_bit():
    p = ref.Paged(23, 32, 8, 128, 16, [1, 70, 1, 3], [4000, 900, 3, 2000])
    cache, batch = p.device(capi)
    first = attend(p, 0.09, cache, batch).clone()
    for _ in range(4):
        assert torch.equal(attend(p, 0.09, cache, batch), first)


def test_large_pool_offsets():
    """A pool of more than 4 GiB a tensor, the pages at its far end: byte offsets
    past 32 bits."""
    kv, hd, page = 8, 256, 1024
    n = 2 ** 32 // (page * kv * hd * 2) + 8  # pages
    k = torch.zeros((n, page, kv, hd), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    p = ref.Paged(24, 16, kv, hd, page, [1, 60], [1500, 2000], spare=0)
    far = p.pages
    k[n - far:] = p.k.cuda()
    v[n - far:] = p.v.cuda()
    cache = capi.PagedKV(k, v, torch.where(p.table >= 0, p.table + (n - far), -1).int().cuda())
    batch = capi.SeqBatch(p.starts.cuda(), p.seq_lens.cuda(), p.rows, 60, 2000)
    check(p, attend(p, 0.0625, cache, batch), 0.0625)


def test_contiguous_cache_as_one_sequence():
    """page_table None: the contiguous cache of the other attention entry points,
    and their results."""
    kv, hd, H, S = 2, 128, 16, 512
    g = torch.Generator().manual_seed(25)
    k, v = (torch.randn((S, kv, hd), generator=g).half().cuda() for _ in range(2))
    q = torch.randn((1, H, hd), generator=g).half().cuda()
    want = torch.empty_like(q)
    capi.attention_decode_f16(want, q, k, v, H, kv, hd, 500, 0.09)
    cache = capi.PagedKV(k.view(-1, 16, kv, hd), v.view(-1, 16, kv, hd))
    lens = torch.tensor([500], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    got = torch.empty_like(q)
    capi.attention_paged_f16(got, q, capi.SeqBatch(starts, lens, 1, 1, 500), cache, 0.09)
    assert (got.double() - want.double()).abs().max() <= 2 * ref.H16 * want.abs().max().item()


def test_two_streams_at_once():
    a = ref.Paged(26, 32, 8, 128, 16, [1, 1], [5000, 3000])
    b = ref.Paged(27, 32, 8, 128, 16, [40], [6000])
    ca, cb = a.device(capi), b.device(capi)
    qa, qb = a.q.cuda(), b.q.cuda()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    oa, ob = torch.empty_like(qa), torch.empty_like(qb)
    torch.cuda.synchronize()
    for _ in range(10):
        capi.attention_paged_f16(oa, qa, ca[1], ca[0], 0.09, stream=sa)
        capi.attention_paged_f16(ob, qb, cb[1], cb[0], 0.09, stream=sb)
    torch.cuda.synchronize()
    check(a, oa, 0.09)
    check(b, ob, 0.09)
    for s in (sa, sb):
        capi.release_workspace(s)


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [900, 30, 2500]), ([40, 1, 3], [700, 300, 64])])
def test_captured_and_replayed_with_other_lengths(new, lens):
    """A captured launch follows seq_lens and the table as they are at its replay."""
    p = ref.Paged(28, 16, 2, 128, 16, new, lens)
    cache, batch = p.device(capi, max_len=4000)
    q = p.q.cuda()
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    capi.attention_paged_f16(out, q, batch, cache, 0.09, stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.attention_paged_f16(out, q, batch, cache, 0.09, stream=s)
    for step in range(4):
        now = [max(n, m - 17 * step) for n, m in zip(new, lens)]
        p.lens, p.seq_lens = now, torch.tensor(now, dtype=torch.int32)
        batch.tensors[1].copy_(p.seq_lens)
        out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        check(p, out, 0.09)
        eager = attend(p, 0.09, cache, batch)
        assert torch.equal(eager, out)


@pytest.mark.parametrize("n,heads,page,int8", [(64, (8, 2, 64), 16, False), (65, (8, 2, 64), 4, True),
                                               (256, (4, 2, 64), 16, True), (257, (4, 2, 64), 16, False),
                                               (700, (4, 1, 64), 1, False)])
def test_many_sequences_decoding(n, heads, page, int8):
    """A lane's one sequence, several, and more than a workgroup counts; some of no
    new tokens, some of no positions."""
    new = [0 if i % 13 == 5 else 1 + i % 3 for i in range(n)]
    lens = [0 if i % 31 == 7 else 1 + (i * 97) % 400 + (1500 if i % 50 == 0 else 0) for i in range(n)]
    p = ref.Paged(35, *heads, page, new, lens, int8)
    check(p, attend(p, 0.125), 0.125)


@pytest.mark.parametrize("n", [65, 1024, 1030])
def test_many_sequences_of_chunks(n):
    """Blocks found among more sequences than lanes, and among more than are cut."""
    new = [0 if i % 13 == 5 else 1 + i % 29 for i in range(n)]
    lens = [m + (i * 37) % 90 for i, m in enumerate(new)]
    lens[3] += 1500
    p = ref.Paged(36, 2, 1, 16, 16, new, lens)
    check(p, attend(p, 0.25), 0.25)


@pytest.mark.parametrize("new,int8", [([1, 1, 1], False), ([1, 1, 1], True), ([1, 40, 2], False), ([90, 30, 20], True)])
def test_limits_of_a_whole_context(new, int8):
    """max_len and the table at a capacity far above the lengths, as for a captured
    step: the chunks follow the lengths."""
    p = ref.Paged(37, 16, 2, 128, 16, new, [9000] * 3, int8)
    for lens in ([9000, 900, 90], [130, 129, 95], [200, 8000, 3000]):
        p.lens, p.seq_lens = lens, torch.tensor(lens, dtype=torch.int32)
        check(p, attend(p, 0.09, max_len=9000), 0.09)


@pytest.mark.parametrize("hd", [64, 80, 96, 128, 200, 256])
@pytest.mark.parametrize("new,length", [(1, 700), (40, 700)])
def test_pages_of_sixteen_or_more_with_holes(hd, new, length):
    """The page of a wave's 16 rows from the lane that looked it up: every head
    width, pages that end inside a tile, holes between them, K and V apart."""
    p = ref.Paged(38, 4, 2, hd, 16, [new], [length], holes=[(0, 1), (0, 2), (0, 9), (0, 42)], apart=True)
    check(p, attend(p, 0.125), 0.125)
    p = ref.Paged(39, 4, 2, hd - hd % 16, 32, [new], [length], True, holes=[(0, 3), (0, 20)])
    check(p, attend(p, 0.0625), 0.0625)


@pytest.mark.parametrize("n", [300, 1000])
def test_chunks_among_many_decoding(n):
    """Split blocks of a few sequences among many that decode."""
    new, lens = [1] * n, [1 + (i * 53) % 60 for i in range(n)]
    for i, m in ((7, 40), (n // 2, 100), (n - 1, 33)):
        new[i], lens[i] = m, 2000 + i
    p = ref.Paged(40, 4, 2, 64, 16, new, lens)
    check(p, attend(p, 0.125), 0.125)


@pytest.mark.parametrize("n", [1, 20, 100, 126, 127])
def test_blocks_up_to_one_a_cu(n):
    """As many blocks as nearly fill the CUs, of very different lengths: the chunks'
    length where few divisions fit."""
    new = [17] * n
    lens = [17 + (i * i * 13) % 700 + (6000 if i == n // 2 else 0) for i in range(n)]
    p = ref.Paged(41, 2, 2, 16, 16, new, lens)
    check(p, attend(p, 0.25), 0.25)


@pytest.mark.parametrize("n", [1, 33])
def test_lengths_outside_the_limits(n):
    """seq_lens past max_len and below zero, to the type's ends: the cache as far as it
    goes, and nothing."""
    p = ref.Paged(42, 4, 2, 64, 16, [n] * 4, [64] * 4)
    p.seq_lens = torch.tensor([2 ** 31 - 1, -5, -2 ** 31, 64], dtype=torch.int32)
    got = attend(p, 0.125, max_len=64)
    assert not got[n:3 * n].any()
    p.lens = [64 + n, -5, -64, 64]  # past the table: every position is seen by every row
    check(p, got, 0.125)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("new,length,page", [(1, 100, 16), (1, 3000, 8), (3, 100, 8), (20, 150, 16), (100, 333, 8)])
@pytest.mark.parametrize("hd", [64, 80, 128])
def test_int8_scales_that_are_not_finite_in_places_seen(bad, new, length, page, hd):
    """A V scale of a seen position: the rows that see it get that times its bytes, NaN
    where a byte is 0, whichever kernel takes them; no other row or head changes."""
    p = ref.Paged(43, 8, 2, hd, page, [new], [length], True)
    clean = attend(p, 0.0625).cpu()
    at = length - (new + 1) // 2
    slot = int(p.slots(0, length)[at])
    p.v.view(-1, 2, hd)[slot, 1, 7] = 0
    p.vs.view(-1, 2)[slot, 1] = bad
    got = attend(p, 0.0625).cpu()
    first = at - (length - new)  # the first token that sees it
    want = p.v.view(-1, 2, hd)[slot, 1].float() * bad
    for head in range(4, 8):
        assert torch.equal(got[:first, head], clean[:first, head])
        assert torch.equal(torch.nan_to_num(got[first:, head].float(), 3.0, 2.0, 1.0),
                           torch.nan_to_num(want, 3.0, 2.0, 1.0).expand(new - first, hd))
    assert torch.equal(got[:, :4], clean[:, :4])


@pytest.mark.parametrize("new,length", [(1, 100), (1, 3000), (3, 2000), (20, 150), (20, 3000), (100, 333)])
@pytest.mark.parametrize("gap", [30.0, 900.0])
def test_infinities_seen_with_little_weight(new, length, gap):
    """Infinite V at positions whose weights are e^-gap of the largest's, with e^-900 below
    fp32's range: any weight times them is infinite, however the positions are split
    over waves and chunks, of which one alone holds the position that weighs."""
    p = ref.Paged(44, 4, 1, 64, 16, [new], [length])
    p.q[:] = 0.0
    p.q[..., 0] = 1.0
    slots = p.slots(0, length)
    k, v = p.k.view(-1, 64), p.v.view(-1, 64)
    k[slots, 0] = 0.0
    k[slots[length - new], 0] = gap
    for at in (1, 40, 77):
        v[slots[at], at % 64] = float("inf") if at % 2 else float("-inf")
    got = attend(p, 1.0).cpu()
    assert (got[..., 1] == float("inf")).all() and (got[..., 40] == float("-inf")).all()
    assert (got[..., 13] == float("inf")).all()
    got[..., [1, 13, 40]] = 0.0
    assert torch.isfinite(got).all()


def test_a_batch_too_large_for_one_kernel_writes_nothing():
    """A mixed batch whose chunk fits its launch and whose decoding sequences do not."""
    n, kv = 16500, 512
    q = torch.zeros((n + 199, kv, 8), dtype=torch.float16, device="cuda")
    k = torch.zeros((1, 1024, kv, 8), dtype=torch.float16, device="cuda")
    starts = torch.arange(n + 1, dtype=torch.int32)
    starts[1:] += 199
    lens = torch.ones(n, dtype=torch.int32)
    lens[0] = 200
    cache = capi.PagedKV(k, k, torch.zeros((n, 1), dtype=torch.int32, device="cuda"))
    batch = capi.SeqBatch(starts.cuda(), lens.cuda(), n + 199, 200, 200)
    out = torch.full_like(q, 7.0)
    with pytest.raises(rxq4.RxQ4Error):
        capi.attention_paged_f16(out, q, batch, cache, 1.0)
    assert (out == 7.0).all()


@pytest.mark.parametrize("new,lens", [([1, 1, 1], [700, 40, 1]), ([1, 3], [5000, 2000]), ([33, 70], [300, 3000]),
                                      ([1, 150, 1, 2], [900, 400, 1, 3000]), ([300], [300])])
@pytest.mark.parametrize("int8", [False, True])
def test_in_place(new, lens, int8):
    """out is q: whole rows and split ones, both kernels, alone and together."""
    p = ref.Paged(45, 16, 2, 128, 16, new, lens, int8)
    cache, batch = p.device(capi)
    want = attend(p, 0.09, cache, batch)
    q = p.q.cuda()
    capi.attention_paged_f16(q, q, batch, cache, 0.09)
    assert torch.equal(q, want)
