"""GPU bounds of pages (rxq4_kv_bounds), choice of pages (rxq4_select_pages) and
attention over chosen pages (rxq4_attention_selected_f16) against their definitions
(selected_reference): bytes and lists have to be equal, outputs within the bounds that
are derived there."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import rxq4  # noqa: F401
from rxq4 import capi
from tests import selected_reference as sel
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- bounds
def run_bounds(p, cache=None, batch=None, **limits):
    if cache is None:
        cache, batch = p.device(capi, **limits)
    bounds = torch.full((p.pages, p.kv, p.hd // 8, 2, 8), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((p.pages, p.kv), 7.0, device="cuda")
    capi.kv_bounds(bounds, scales, batch, cache)
    return bounds, scales


def check_bounds(p, got, **limits):
    bounds, scales = (t.cpu().numpy() for t in got)
    left = np.ones(p.pages, bool)
    for page, held in sel.touched(p, **limits):
        left[page] = False
        b, s = sel.bounds(p, page, held)
        assert np.array_equal(scales[page], s), (page, scales[page], s)
        assert np.array_equal(bounds[page], b), page
    assert (bounds[left] == 99).all() and (scales[left] == 7.0).all()


# heads, page, int8, new, lens
BOUNDS = [
    ((16, 2, 128), 16, False, [1], [1001]),
    ((16, 2, 128), 16, False, [1], [1]),
    ((32, 8, 128), 16, True, [1] * 20, [1 + 9 * i for i in range(20)]),
    ((32, 8, 128), 64, False, [70, 1, 300], [70, 64, 1000]),
    ((8, 8, 64), 1, False, [5, 0, 9], [5, 9, 100]),
    ((8, 4, 80), 8, True, [40, 3], [64, 1000]),
    ((6, 2, 96), 32, False, [17], [40]),
    ((4, 1, 256), 16, False, [300], [320]),
    ((3, 1, 8), 2, False, [5], [9]),
    ((40, 40, 8), 4, False, [9], [30]),
    ((2, 2, 16), 1024, True, [1500], [1700]),
    ((5, 5, 200), 128, False, [7, 200], [300, 200]),
    ((7, 7, 72), 16, False, [33], [50]),
    ((2, 1, 64), 16, False, [3000, 1], [3001, 17]),  # several rows a workgroup
    ((2, 1, 64), 2, True, [2100, 5], [2500, 17]),
]


@pytest.mark.parametrize("heads,page,int8,new,lens", BOUNDS)
def test_bounds(heads, page, int8, new, lens):
    print(f"bounds {heads} page={page} int8={int8} new={new} lens={lens}", flush=True)
    p = ref.Paged(61, *heads, page, new, lens, int8, pad=3, lead=2)
    check_bounds(p, run_bounds(p))


@pytest.mark.parametrize("int8", [False, True])
def test_bounds_of_pages_apart_with_holes_and_limits(int8):
    p = ref.Paged(62, 8, 2, 64, 16, [60, 7, 9, 1], [100, 3, 9, 0], int8, holes=[(0, 3), (2, 0)], apart=True)
    check_bounds(p, run_bounds(p))
    check_bounds(p, run_bounds(p, max_new=24), max_new=24)
    check_bounds(p, run_bounds(p, max_len=70), max_len=70)
    check_bounds(p, run_bounds(p, max_new=500, max_len=1 << 24))


def test_bounds_of_keys_that_are_not_numbers():
    """NaN left out, a dim of nothing else 0, infinities as fp32's largest; zeros;
    fp16's smallest numbers."""
    p = ref.Paged(63, 4, 4, 64, 16, [48], [48])
    k = p.both[0].view(p.pages, 16, 4, 64)
    first, second, third = (int(p.table[0, j]) for j in range(3))
    k[first, 3, 0, 5], k[first, :, 1, 7], k[first, 2, 2, 9] = float("nan"), float("nan"), float("inf")
    k[first, 2, 3, 9], k[first, 4, 3, 9], k[first, 5, 3, 8] = float("-inf"), float("inf"), float("nan")
    k[second, :, 0], k[second, :, 1] = 0.0, float("nan")
    k[second, :, 2] = 6e-8
    k[second, :, 3] = -0.0
    k[third] *= 1e-4
    check_bounds(p, run_bounds(p))


def test_bounds_of_int8_scales_that_are_not_numbers():
    p = ref.Paged(64, 4, 4, 64, 16, [40], [48], True)
    page = int(p.table[0, 0])
    p.ks[page, 1, 0], p.ks[page, 2, 1], p.ks[page, 3, 2] = float("nan"), float("inf"), 0.0
    p.ks[page, :, 3] = 1e-44
    check_bounds(p, run_bounds(p))


def test_bounds_without_int8_scales():
    p = ref.Paged(65, 4, 2, 64, 16, [40], [48], True, scales=False)
    check_bounds(p, run_bounds(p))


@pytest.mark.parametrize("starts", [[0, 5, 3], [-4, 2, 9], [0, 100000, 100001], [7, 2, 1], [2 ** 31 - 1] * 3, [-2 ** 31] * 3])
@pytest.mark.parametrize("lens", [[64, 64], [2 ** 31 - 1, -2 ** 31]])
def test_starts_and_lengths_outside_their_limits_stay_inside(starts, lens):
    """No list, byte or row outside the arrays, whatever the device arrays hold."""
    p = ref.Paged(66, 8, 2, 64, 16, [4, 5], [64, 64])
    cache, batch = p.device(capi)
    batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
    batch.tensors[1].copy_(torch.tensor(lens, dtype=torch.int32))
    b = torch.full((p.pages + 2, 2, 8, 2, 8), 99, dtype=torch.int8, device="cuda")
    s = torch.full((p.pages + 2, 2), 7.0, device="cuda")
    capi.kv_bounds(b[1:-1], s[1:-1], batch, cache)
    assert (b[0] == 99).all() and (b[-1] == 99).all() and (s[0] == 7.0).all() and (s[-1] == 7.0).all()
    b.zero_(), s.zero_()
    q = p.q.cuda()
    lists = torch.full((p.rows + 20, 2, 3), -9, dtype=torch.int32, device="cuda")
    capi.select_pages(lists[10:-10], q, b[1:-1], s[1:-1], batch, cache)
    assert (lists[:10] == -9).all() and (lists[-10:] == -9).all()
    assert ((lists >= -1) & (lists < 4) | (lists == -9)).all()
    out = torch.full((p.rows + 20, 8, 64), 7.0, dtype=torch.float16, device="cuda")
    capi.attention_selected_f16(out[10:-10], q, lists[10:-10], batch, cache, 0.125)
    assert (out[:10] == 7.0).all() and (out[-10:] == 7.0).all()


# ---------------------------------------------------------------- the choice
def run_select(p, both, scale, n_select, n_first, n_last, cache=None, batch=None, stream=None, out=None, **limits):
    if cache is None:
        cache, batch = p.device(capi, **limits)
    if out is None:
        out = torch.full((p.rows, p.kv, n_select), -7, dtype=torch.int32, device="cuda")
    to = lambda a: a if isinstance(a, torch.Tensor) else torch.from_numpy(a).cuda()  # noqa: E731
    capi.select_pages(out, p.q.cuda(), to(both), to(scale), batch, cache, n_first, n_last, stream)
    return out


def check_select(p, got, both, scale, *how, **limits):
    want = sel.select(p, both, scale, *how, **limits)
    got = got.cpu().numpy()
    assert np.array_equal(got, want), [(tuple(x), got[tuple(x)], want[tuple(x)]) for x in np.argwhere(got != want)[:5]]


# heads, page, new, lens, (n_select, n_first, n_last)
SELECT = [
    ((16, 2, 128), 16, [1], [1], (4, 1, 1)),
    ((16, 2, 128), 16, [1], [1001], (16, 1, 2)),
    ((32, 8, 128), 16, [1] * 12, [1 + 97 * i for i in range(12)], (8, 1, 2)),
    ((28, 4, 128), 32, [70], [1500], (12, 1, 2)),             # groups of 7: two tokens a tile
    ((32, 8, 128), 16, [37], [1100], (16, 0, 1)),             # of 4: four
    ((16, 8, 64), 8, [50, 3], [600, 90], (10, 2, 2)),         # of 2: eight
    ((8, 8, 64), 4, [90, 20, 33], [300, 20, 40], (10, 2, 2)),  # of 1: sixteen
    ((6, 2, 96), 8, [40], [700], (30, 0, 0)),                 # of 3
    ((5, 1, 200), 16, [9], [900], (7, 3, 4)),                 # of 5; the forced fill the list
    ((40, 1, 64), 16, [3, 1], [500, 900], (9, 1, 1)),         # of 40: three blocks of heads
    ((20, 1, 256), 16, [5], [500], (9, 1, 1)),                # of 20
    ((3, 1, 8), 2, [5], [90], (11, 1, 1)),
    ((2, 2, 16), 1, [6], [400], (1, 0, 1)),
    ((4, 4, 80), 1, [4], [300], (300, 1, 1)),                 # more than there are
    ((4, 4, 80), 1, [4], [300], (297, 1, 1)),                 # the border at the last pages
    ((4, 2, 72), 128, [200], [1000], (3, 1, 1)),
    ((4, 1, 64), 1, [1], [3000], (64, 1, 1)),                 # one token, many pages: split
    ((2, 2, 64), 1, [1, 2], [15000, 9000], (33, 2, 2)),       # split; more keys than LDS holds
    ((2, 1, 64), 1, [1], [14000], (4096, 5, 9)),
    ((2, 2, 64), 1, [40], [2100], (100, 1, 1)),               # sixteen tokens, several parts
    ((4, 1, 128), 1, [12], [9000], (200, 1, 1)),
    ((64, 4, 64), 1, [20], [13000], (64, 1, 1)),              # of 16: two tokens a tile, several parts
    ((4, 4, 256), 1, [40], [1500], (512, 1, 1)),              # the longest lists of a tile, its most LDS
    ((8, 4, 256), 1, [40], [1500], (512, 1, 1)),
    ((16, 4, 200), 1, [40], [1500], (511, 1, 1)),
    ((32, 2, 256), 1, [9], [1500], (512, 1, 1)),
    ((4, 4, 256), 1, [40], [3000], (256, 1, 1)),              # several parts, pages of one token
    ((4, 4, 256), 1, [40], [3000], (257, 1, 1)),
    ((8, 2, 64), 1, [30], [9000], (70, 1, 69)),               # several parts; the last pages always
    ((8, 2, 64), 1, [30], [9000], (70, 69, 1)),
    ((2, 2, 64), 1, [50], [7000], (10, 0, 0)),
    ((16, 1, 64), 1, [20], [9000], (200, 5, 5)),
    ((8, 2, 64), 1, [12], [9000], (513, 1, 1)),               # longer ones: a token a workgroup
    ((4, 2, 256), 1, [300], [9000], (4096, 1, 1)),
]


@pytest.mark.parametrize("heads,page,new,lens,how", SELECT)
def test_select(heads, page, new, lens, how):
    print(f"select {heads} page={page} new={new} lens={lens} {how}", flush=True)
    p = ref.Paged(71, *heads, page, new, lens, pad=3, lead=2)
    both, scale = sel.random_bounds(72, p.pages, p.kv, p.hd)
    check_select(p, run_select(p, both, scale, *how), both, scale, *how)


@pytest.mark.parametrize("new", [[1], [9], [40]])
@pytest.mark.parametrize("group", [1, 2, 4, 8, 16, 24])
def test_ties_go_to_the_first_pages(new, group):
    """Pages of the same bounds, and queries of zeros, for which all pages are."""
    p = ref.Paged(73, 2 * group, 2, 64, 4, new, [700])
    both, scale = sel.random_bounds(74, 6, 2, 64)
    pick = np.random.default_rng(75).integers(0, 6, p.pages)
    both, scale = both[pick], scale[pick]
    p.q[::3] = 0
    for how in ((20, 1, 1), (41, 0, 0), (100, 2, 3), (1, 0, 0)):
        check_select(p, run_select(p, both, scale, *how), both, scale, *how)


def test_scores_at_their_ends():
    """Queries with NaN and infinities, scales of 0 and of fp32's ends, scores that
    overflow and that are 0 with either sign."""
    p = ref.Paged(76, 8, 2, 64, 4, [30], [400])
    both, scale = sel.random_bounds(77, p.pages, 2, 64)
    p.q[1, 0, 3], p.q[2, 1], p.q[3, 2, 9], p.q[4, 3, 9] = float("nan"), float("nan"), float("inf"), float("-inf")
    p.q[5], p.q[6], p.q[7] = 0.0, 6e-8, -65504.0
    rng = np.random.default_rng(78)
    scale[rng.random(scale.shape) < 0.3] = 0.0
    scale[rng.random(scale.shape) < 0.2] = 2.6e36
    scale[rng.random(scale.shape) < 0.2] = 1e-45
    both[rng.random(p.pages) < 0.1] = 0
    both[rng.random(p.pages) < 0.1] = -127
    for how in ((20, 1, 1), (70, 0, 0)):
        check_select(p, run_select(p, both, scale, *how), both, scale, *how)


@pytest.mark.parametrize("new,length", [([300], 1500), ([1], 1500), ([1] * 140, 1500), ([40], 6000)])
def test_scores_crowded_beside_a_few_far_ones(new, length):
    """Most scores in one of equal parts of their range, lists that end among them: one
    token a wave, a token a workgroup, the choice in a launch of its own."""
    p = ref.Paged(84, 4, 2, 64, 1, new, [length] * len(new))
    both, scale = sel.random_bounds(85, p.pages, 2, 64)
    scale *= 1 + 1e-3 * np.random.default_rng(86).random(scale.shape).astype(np.float32)
    for i in range(len(new)):
        scale[p.table[i, 5], :], scale[p.table[i, 11], :] = 1e4, 1e3
    for n in (100, 300, 500):
        check_select(p, run_select(p, both, scale, n, 1, 1), both, scale, n, 1, 1)


@pytest.mark.parametrize("kind", ["rising", "falling", "alike", "few"])
def test_parts_whose_scores_rise_fall_or_tie(kind):
    """Several parts of pages: every later one above the first's list, none, all the same,
    and candidates only here and there."""
    p = ref.Paged(87, 4, 2, 64, 1, [40], [6000], holes=[(0, j) for j in range(6000) if kind == "few" and j % 97])
    both, scale = sel.random_bounds(88, 1, 2, 64)
    both = np.repeat(both, p.pages, 0)
    rank = np.empty(p.pages)
    rank[p.table[0].numpy().clip(0, p.pages - 1)] = np.arange(6000)
    slope = {"rising": 1 + rank / 100, "falling": 100 - rank / 100, "alike": 0 * rank + 1, "few": 1 + (rank * 7919 % 1000)}[kind]
    scale = (scale * slope[:, None]).astype(np.float32)
    for how in ((40, 1, 1), (100, 0, 0), (256, 2, 3)):
        check_select(p, run_select(p, both, scale, *how), both, scale, *how)


@pytest.mark.parametrize("new,page", [([1, 1], 16), ([30, 1, 9], 16), ([1], 1)])
def test_select_with_holes_padding_and_limits(new, page):
    lens = [n + 1200 for n in new]
    holes = [(0, 0), (0, 1), (0, 7), (0, (lens[0] - 1) // page), (len(new) - 1, 5)]
    p = ref.Paged(79, 16, 4, 64, page, new, lens, holes=holes, pad=2, lead=1)
    both, scale = sel.random_bounds(80, p.pages, 4, 64)
    for how in ((12, 2, 3), (73, 1, 1)):
        check_select(p, run_select(p, both, scale, *how), both, scale, *how)
        check_select(p, run_select(p, both, scale, *how, max_len=900), both, scale, *how, max_len=900)
        check_select(p, run_select(p, both, scale, *how, max_new=5), both, scale, *how, max_new=5)
        check_select(p, run_select(p, both, scale, *how, max_len=1 << 20), both, scale, *how, max_len=1 << 20)


def test_select_where_nothing_is_seen():
    p = ref.Paged(81, 8, 2, 64, 16, [1, 40, 5, 1], [40, 20, 2, 0], holes=[(0, 0), (0, 1), (0, 2)])
    both, scale = sel.random_bounds(82, p.pages, 2, 64)
    got = run_select(p, both, scale, 5, 1, 1)
    check_select(p, got, both, scale, 5, 1, 1)
    assert (got[0] == -1).all() and (got[1:21] == -1).all() and (got[-1] == -1).all()


def test_score_bounds_every_key_of_the_page():
    """Up to the steps: |q - step z| <= step / 2 and |lo - scale byte| <= scale / 2
    in each dim, so the largest product is at most the score + sum_d (step |k_d| + scale
    |q_d| + step scale / 2) / 2."""
    p = ref.Paged(83, 8, 2, 64, 16, [80], [80], spare=0)
    bounds, scales = (t.cpu().numpy() for t in run_bounds(p))
    row = 79
    q = p.q[row].double().numpy()
    step = np.abs(q).max(-1) / 127
    s = sel.scores(p.q[row].numpy(), bounds[p.table[0].numpy()], scales[p.table[0].numpy()])
    for j in range(5):
        page = int(p.table[0, j])
        k = sel.page_keys(p, page).astype(np.float64)
        for h in range(2):
            heads = range(4 * h, 4 * h + 4)
            slack = max((step[e] * np.abs(k[:, h]) + scales[page, h] * np.abs(q[e]) + step[e] * scales[page, h] / 2).sum(-1).max() / 2
                        for e in heads)
            most = max((k[:, h] @ q[e]).max() for e in heads)
            assert most <= s[h, j] + slack + 1e-3


# ---------------------------------------------------------------- attention
def run_attend(p, lists, scale, cache=None, batch=None, stream=None, **limits):
    if cache is None:
        cache, batch = p.device(capi, **limits)
    out = torch.full((p.rows, p.heads, p.hd), 7.0, dtype=torch.float16, device="cuda")
    lists = lists if isinstance(lists, torch.Tensor) else torch.from_numpy(lists).cuda()
    capi.attention_selected_f16(out, p.q.cuda(), lists, batch, cache, scale, stream)
    return out


def check_attend(p, got, lists, scale):
    want, bound = sel.attend(p, lists, scale)
    got = got.cpu().double()
    mine = ~torch.isnan(want)
    assert ((got - want).abs() <= bound)[mine].all(), ((got - want).abs() / bound)[mine].max()
    assert (got[~mine] == 7.0).all()  # rows of no sequence


# heads, page, int8, new, lens, n_select
ATTEND = [
    ((16, 2, 128), 16, False, [1], [1], 4),
    ((16, 2, 128), 16, False, [1], [1001], 16),
    ((16, 2, 128), 16, False, [1, 1, 1], [16, 17, 2000], 100),
    ((32, 8, 128), 64, False, [1, 1, 1], [3000, 63, 129], 9),
    ((32, 8, 128), 16, True, [1, 1, 1], [1300, 1, 257], 40),
    ((28, 4, 128), 32, False, [5, 3], [900, 64], 7),
    ((8, 8, 64), 1, False, [1, 2], [130, 70], 50),
    ((8, 2, 64), 4, True, [1, 3], [130, 600], 33),
    ((8, 2, 64), 4, False, [9], [600], 70),
    ((8, 4, 80), 8, False, [1, 1, 1], [333, 64, 1], 20),
    ((8, 4, 80), 8, True, [1, 20], [333, 350], 18),
    ((6, 2, 96), 128, False, [1, 4], [700, 127], 3),
    ((6, 2, 96), 2, False, [3], [200], 64),
    ((4, 1, 256), 16, False, [1, 6], [900, 30], 20),
    ((4, 4, 256), 256, True, [1, 1], [600, 256], 2),
    ((4, 2, 256), 8, False, [3], [200], 12),
    ((4, 2, 256), 4, True, [3], [200], 40),
    ((3, 1, 8), 2, False, [1, 2], [9, 200], 30),
    ((2, 2, 16), 16, True, [1, 3], [40, 70], 3),
    ((5, 1, 200), 16, False, [1, 7], [90, 300], 12),
    ((32, 1, 128), 16, False, [1, 2], [600, 40], 30),   # a group of 32: two blocks of heads
    ((40, 1, 64), 32, False, [2], [500], 9),            # of 40: three
    ((17, 1, 64), 8, True, [2], [300], 30),
    ((16, 2, 128), 1024, True, [4, 4], [2500, 5], 2),
    ((16, 2, 128), 16, False, [60, 1, 0, 9], [400, 900, 1, 9], 10),
    ((32, 8, 128), 32, False, [130], [500], 4),
    ((8, 2, 64), 16, False, [1], [5000], 300),          # more than 32 steps of a wave
    ((4, 2, 64), 16, False, [700], [900], 260),         # the same in one chunk
]


@pytest.mark.parametrize("heads,page,int8,new,lens,n_select", ATTEND)
def test_attention(heads, page, int8, new, lens, n_select):
    print(f"selected {heads} page={page} int8={int8} new={new} lens={lens} n_select={n_select}", flush=True)
    p = ref.Paged(91, *heads, page, new, lens, int8, pad=3, lead=2)
    lists = sel.random_lists(p, n_select, 92)
    scale = heads[2] ** -0.5
    check_attend(p, run_attend(p, lists, scale), lists, scale)


# heads, page, int8, new, lens, n_select: several tokens' lists walked together (256 tiles or more)
TILES = [
    ((32, 32, 16), 16, False, [70, 1, 3], [300, 200, 3], 6),     # eight tokens a tile
    ((64, 32, 64), 16, True, [60, 9, 5], [400, 9, 64], 9),       # of 2 heads: eight
    ((48, 16, 80), 32, False, [90, 1, 1], [300, 40, 200], 5),    # of 3: five
    ((64, 16, 128), 16, False, [75, 20, 2], [600, 33, 90], 12),  # of 4: four
    ((80, 16, 64), 64, True, [60], [500], 4),                    # of 5: three
    ((112, 16, 128), 32, False, [40, 7], [500, 64], 7),          # of 7: two
    ((56, 8, 256), 16, False, [70, 4], [300, 4], 11),
    ((64, 8, 96), 128, False, [70], [700], 3),                   # of 8: two
    ((32, 32, 48), 8, False, [70, 2], [200, 30], 13),            # pages of fewer positions than an operand
    ((64, 32, 64), 4, True, [60, 9, 5], [300, 9, 64], 33),
    ((64, 16, 128), 8, False, [75, 20, 2], [400, 33, 90], 24),
    ((64, 16, 128), 1, True, [75, 2], [300, 33], 90),
    ((48, 16, 80), 8, True, [90], [300], 15),
    ((64, 16, 200), 2, False, [70], [120], 21),
    ((16, 8, 64), 16, False, [300], [320], 256),                 # lists of all that a tile holds
    ((32, 16, 16), 1, False, [140], [50000], 9),                 # more pages than are marked at a time
]


@pytest.mark.parametrize("order", ["ascending", "any"])
@pytest.mark.parametrize("heads,page,int8,new,lens,n_select", TILES)
def test_attention_of_tiles(heads, page, int8, new, lens, n_select, order):
    """Ascending lists are merged; lists with pages twice, in any order, with -1s
    between or places that are none are walked as they are."""
    print(f"tiles {heads} page={page} int8={int8} new={new} lens={lens} n_select={n_select} {order}", flush=True)
    p = ref.Paged(116, *heads, page, new, lens, int8, pad=3, lead=2, apart=page == 32)
    lists = sel.random_lists(p, n_select, 117, odd=order == "any")
    scale = heads[2] ** -0.5
    check_attend(p, run_attend(p, lists, scale), lists, scale)


def test_tiles_whose_lists_agree_differ_and_are_empty():
    """Neighbours with the same list, with none in common, with holes, and with nothing
    that is theirs to see."""
    p = ref.Paged(118, 64, 16, 64, 16, [80], [400], holes=[(0, 3), (0, 9)])
    lists = np.full((p.rows, 16, 8), -1, np.int32)
    for t in range(80):
        last = (320 + t) // 16
        lists[t, :, :4] = [0, 3, 7, last] if t < 30 else [t % 4, 4 + t % 4, 9, 10 + t % 4]
        if t % 11 == 5:
            lists[t] = -1
        if t % 11 == 6:
            lists[t] = [3, 9] + [-1] * 6
        if t % 11 == 7:
            lists[t] = [last + 1, last + 2] + [-1] * 6
    got = run_attend(p, lists, 0.125)
    check_attend(p, got, lists, 0.125)
    assert not got[5].any() and not got[6].any() and not got[7].any()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("page,int8", [(16, False), (8, False), (16, True), (4, True)])
def test_tiles_keep_what_one_token_looks_at_from_the_others(bad, page, int8):
    """Infinities and NaN in a page that only one token of the tile lists, and in the
    last positions, which the tokens before do not see."""
    p = ref.Paged(119, 64, 16, 64, page, [80], [400], int8)
    lists = np.full((p.rows, 16, 3), -1, np.int32)
    for t in range(80):
        lists[t, :, 0], lists[t, :, 1] = 0, (320 + t) // page
    lists[41, :] = [0, 2, (320 + 41) // page]
    clean = run_attend(p, lists, 0.125).cpu()
    check_attend(p, clean, lists, 0.125)
    slots = p.slots(0, 400)
    at = slots[2 * page + 1]
    if int8:
        p.vs.view(-1, 16)[at, 3], p.ks.view(-1, 16)[at, 5] = bad, bad
        p.vs.view(-1, 16)[slots[399], 3] = bad
    else:
        p.both[1].view(-1, 16, 64)[at, 3, 7], p.both[0].view(-1, 16, 64)[at, 5, 7] = bad, bad
        p.both[1].view(-1, 16, 64)[slots[399], 3, 7] = bad
    got = run_attend(p, lists, 0.125).cpu()
    rest = [t for t in range(79) if t != 41]
    assert torch.equal(got[rest], clean[rest])
    assert not torch.isfinite(got[41, 12:16]).all() and not torch.isfinite(got[79, 12:16]).all()
    keep = torch.ones(64, dtype=torch.bool)
    keep[12:16] = False
    assert torch.equal(got[79][keep], clean[79][keep])
    keep[20:24] = False
    assert torch.equal(got[41][keep], clean[41][keep])


# heads, page, int8, new, lens, n_select: 17 to 32 rows a tile, tiles for the whole chip
WIDE_TILES = [
    ((96, 32, 16), 16, False, [150, 7, 3], [300, 200, 3], 6),    # of 3 heads: eight tokens
    ((64, 16, 128), 16, False, [210, 20, 2], [600, 33, 90], 12), # of 4: eight
    ((80, 16, 64), 64, True, [240], [700], 4),                   # of 5: six
    ((112, 16, 128), 32, False, [110, 7], [500, 64], 7),         # of 7: four
    ((64, 8, 96), 128, False, [220], [700], 3),                  # of 8: four
    ((72, 8, 64), 16, True, [230], [400], 9),                    # of 9: three
    ((128, 8, 128), 16, True, [110, 3], [300, 3], 9),            # of 16: two
    ((32, 8, 128), 16, False, [415], [420], 256),                # lists of all that a tile holds
    ((64, 16, 128), 8, False, [210, 20, 2], [400, 33, 90], 24),  # pages of fewer positions than an operand
    ((64, 16, 128), 1, True, [220], [300], 90),
    ((48, 16, 80), 8, True, [220], [300], 15),
    ((56, 8, 96), 4, False, [220], [300], 30),
    ((64, 16, 64), 2, False, [370], [400], 21),
]


@pytest.mark.parametrize("order", ["ascending", "any"])
@pytest.mark.parametrize("heads,page,int8,new,lens,n_select", WIDE_TILES)
def test_attention_of_wide_tiles(heads, page, int8, new, lens, n_select, order):
    print(f"wide tiles {heads} page={page} int8={int8} new={new} lens={lens} n_select={n_select} {order}", flush=True)
    p = ref.Paged(129, *heads, page, new, lens, int8, pad=3, lead=2, apart=page == 32)
    lists = sel.random_lists(p, n_select, 130, odd=order == "any")
    scale = heads[2] ** -0.5
    check_attend(p, run_attend(p, lists, scale), lists, scale)


@pytest.mark.parametrize("page", [4, 16])
def test_wide_tiles_whose_lists_agree_differ_and_are_empty(page):
    p = ref.Paged(131, 64, 16, 64, page, [330], [700], holes=[(0, 3), (0, 9)])
    lists = np.full((p.rows, 16, 8), -1, np.int32)
    for t in range(330):
        last = (370 + t) // page
        lists[t, :, :4] = [0, 3, 7, last] if t < 130 else [t % 4, 4 + t % 4, 9, 10 + t % 4]
        if t % 11 == 5 or 200 <= t < 216:
            lists[t] = -1
        if t % 11 == 6:
            lists[t] = [3, 9] + [-1] * 6
        if t % 11 == 7:
            lists[t] = [last + 1, last + 2] + [-1] * 6
    got = run_attend(p, lists, 0.125)
    check_attend(p, got, lists, 0.125)
    assert not got[5].any() and not got[6].any() and not got[7].any() and not got[200:216].any()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("page,int8", [(16, False), (8, False), (16, True), (4, True)])
def test_wide_tiles_keep_what_one_token_looks_at_from_the_others(bad, page, int8):
    p = ref.Paged(132, 64, 16, 64, page, [330], [700], int8)
    lists = np.full((p.rows, 16, 3), -1, np.int32)
    for t in range(330):
        lists[t, :, 0], lists[t, :, 1] = 0, (370 + t) // page
    looks = [41, 46]  # of one tile's rows the first and the second half
    for t in looks:
        lists[t, :] = [0, 2, (370 + t) // page]
    clean = run_attend(p, lists, 0.125).cpu()
    check_attend(p, clean, lists, 0.125)
    slots = p.slots(0, 700)
    at = slots[2 * page + 1]
    if int8:
        p.vs.view(-1, 16)[at, 3], p.ks.view(-1, 16)[at, 5] = bad, bad
        p.vs.view(-1, 16)[slots[699], 3] = bad
    else:
        p.both[1].view(-1, 16, 64)[at, 3, 7], p.both[0].view(-1, 16, 64)[at, 5, 7] = bad, bad
        p.both[1].view(-1, 16, 64)[slots[699], 3, 7] = bad
    got = run_attend(p, lists, 0.125).cpu()
    rest = [t for t in range(329) if t not in looks]
    assert torch.equal(got[rest], clean[rest])
    keep = torch.ones(64, dtype=torch.bool)
    keep[12:16] = False
    assert torch.equal(got[329][keep], clean[329][keep])
    keep[20:24] = False
    for t in looks + [329]:
        assert not torch.isfinite(got[t, 12:16]).all()
        assert torch.equal(got[t][keep], clean[t][keep])


@pytest.mark.parametrize("starts", [[0, 5, 3], [-4, 2, 9], [0, 100000, 100001], [70, 2, 1], [2 ** 31 - 1] * 3, [-2 ** 31] * 3])
@pytest.mark.parametrize("lens", [[64, 64], [2 ** 31 - 1, -2 ** 31]])
@pytest.mark.parametrize("page", [4, 16])
def test_wide_tiles_with_starts_and_lengths_outside_their_limits_stay_inside(starts, lens, page):
    p = ref.Paged(133, 256, 64, 16, page, [36, 36], [64, 64])
    cache, batch = p.device(capi)
    batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
    batch.tensors[1].copy_(torch.tensor(lens, dtype=torch.int32))
    lists = torch.from_numpy(np.random.default_rng(134).integers(-2, 70 // page, (p.rows, 64, 6)).astype(np.int32)).cuda()
    out = torch.full((p.rows + 20, 256, 16), 7.0, dtype=torch.float16, device="cuda")
    capi.attention_selected_f16(out[10:-10], p.q.cuda(), lists, batch, cache, 0.25)
    assert (out[:10] == 7.0).all() and (out[-10:] == 7.0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("page,int8", [(16, False), (4, True)])
def test_wide_tiles_of_many_sequences_replayed_and_in_place(page, int8):
    new = [(i * 7) % 30 if i % 9 else 0 for i in range(28)]
    lens = [0 if i % 17 == 3 else 3 + (i * 29) % 220 for i in range(28)]
    p = ref.Paged(135, 64, 16, 64, page, new, lens, int8)
    cache, batch = p.device(capi, max_len=300)
    q = p.q.cuda()
    lists = sel.random_lists(p, 9, 136)
    ours, out = torch.from_numpy(lists).cuda(), torch.empty_like(q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.attention_selected_f16(out, q, ours, batch, cache, 0.125, stream=s)
    eager = run_attend(p, ours, 0.125, cache, batch)
    check_attend(p, eager, lists, 0.125)
    mine = (eager != 7.0).flatten(1).any(1)
    for _ in range(3):
        out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    capi.attention_selected_f16(q, q, ours, batch, cache, 0.125)
    assert torch.equal(q[mine], eager[mine])


def check_all(p, how, scale=0.125, seed=120, **limits):
    """The choice against bounds of its own, and attention over its lists."""
    both, by = sel.random_bounds(seed, p.pages, p.kv, p.hd)
    cache, batch = p.device(capi, **limits)
    got = run_select(p, both, by, *how, cache=cache, batch=batch)
    check_select(p, got, both, by, *how, **limits)
    out = run_attend(p, got, scale, cache, batch)
    want, bound = sel.attend(p, got.cpu().numpy(), scale)
    mine = ~torch.isnan(want)
    for i, n in enumerate(p.new):  # new tokens past max_new are left alone
        if limits.get("max_new") is not None and n > limits["max_new"]:
            first = int(p.starts[i])
            mine[first + limits["max_new"]:first + n] = False
    out = out.cpu().double()
    assert ((out - want).abs() <= bound)[mine].all()
    assert (out[~mine] == 7.0).all()


@pytest.mark.parametrize("heads", [(64, 64, 16), (32, 16, 32), (64, 16, 64), (80, 16, 16)])
@pytest.mark.parametrize("page", [4, 16])
def test_tiles_of_many_sequences(heads, page):
    """Sequences that begin and end inside a tile's rows, some without new tokens, some
    without positions, some with fewer positions than new tokens."""
    new = [(i * 7) % 10 if i % 9 else 0 for i in range(60)]
    lens = [0 if i % 17 == 3 else 3 + (i * 29) % 120 for i in range(60)]
    p = ref.Paged(121, *heads, page, new, lens, pad=3, lead=1)
    check_all(p, (5, 1, 1))


@pytest.mark.parametrize("page,int8", [(16, False), (8, True)])
def test_tiles_within_limits(page, int8):
    p = ref.Paged(122, 64, 16, 64, page, [70, 25, 40], [300, 25, 12], int8, pad=2, lead=1, holes=[(0, 1), (1, 0)])
    check_all(p, (6, 1, 2))
    check_all(p, (6, 1, 2), max_new=24)
    p = ref.Paged(123, 64, 16, 64, page, [70, 25], [300, 25], int8)
    both, by = sel.random_bounds(124, p.pages, p.kv, p.hd)
    for limits in (dict(max_len=250), dict(max_len=1 << 24)):
        check_select(p, run_select(p, both, by, 6, 1, 2, **limits), both, by, 6, 1, 2, **limits)


@pytest.mark.parametrize("starts", [[0, 5, 3], [-4, 2, 9], [0, 100000, 100001], [7, 2, 1], [2 ** 31 - 1] * 3, [-2 ** 31] * 3])
@pytest.mark.parametrize("lens", [[64, 64], [2 ** 31 - 1, -2 ** 31]])
@pytest.mark.parametrize("page", [4, 16])
def test_tiles_with_starts_and_lengths_outside_their_limits_stay_inside(starts, lens, page):
    p = ref.Paged(125, 64, 64, 16, page, [4, 5], [64, 64])
    cache, batch = p.device(capi)
    batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
    batch.tensors[1].copy_(torch.tensor(lens, dtype=torch.int32))
    lists = torch.from_numpy(np.random.default_rng(126).integers(-2, 70 // page, (p.rows, 64, 6)).astype(np.int32)).cuda()
    out = torch.full((p.rows + 20, 64, 16), 7.0, dtype=torch.float16, device="cuda")
    capi.attention_selected_f16(out[10:-10], p.q.cuda(), lists, batch, cache, 0.25)
    assert (out[:10] == 7.0).all() and (out[-10:] == 7.0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("page,int8", [(16, False), (4, True)])
def test_tiles_captured_replayed_and_in_place(page, int8):
    new, lens = [75, 20, 2], [500, 90, 64]
    p = ref.Paged(127, 64, 16, 64, page, new, lens, int8)
    cache, batch = p.device(capi, max_len=600)
    q, n = p.q.cuda(), 7
    out, lists = torch.empty_like(q), torch.zeros((p.rows, 16, n), dtype=torch.int32, device="cuda")
    both, by = sel.random_bounds(128, p.pages, p.kv, p.hd)
    bounds, scales = torch.from_numpy(both).cuda(), torch.from_numpy(by).cuda()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.select_pages(lists, q, bounds, scales, batch, cache, 1, 1, stream=s)
        capi.attention_selected_f16(out, q, lists, batch, cache, 0.125, stream=s)
    for step in range(3):
        p.lens = [max(k, m - 19 * step) for k, m in zip(new, lens)]
        p.seq_lens = torch.tensor(p.lens, dtype=torch.int32)
        batch.tensors[1].copy_(p.seq_lens)
        out.fill_(7.0), lists.fill_(-7)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        check_select(p, lists, both, by, n, 1, 1, max_len=600)
        check_attend(p, out, lists.cpu().numpy(), 0.125)
        eager, again = torch.empty_like(out), torch.zeros_like(lists)
        capi.select_pages(again, q, bounds, scales, batch, cache, 1, 1)
        capi.attention_selected_f16(eager, q, again, batch, cache, 0.125)
        assert torch.equal(again, lists) and torch.equal(eager, out)
    capi.attention_selected_f16(q, q, lists, batch, cache, 0.125)
    assert torch.equal(q, out)


@pytest.mark.parametrize("int8,page", [(False, 16), (True, 16), (False, 4), (True, 8)])
def test_all_pages_listed_is_the_paged_attention(int8, page):
    """Within what two roundings of the same sums differ by: each is within its bound."""
    p = ref.Paged(93, 16, 4, 64, page, [1, 30], [300, 200], int8)
    n = -(-300 // page)
    lists = np.broadcast_to(np.arange(n, dtype=np.int32), (p.rows, 4, n)).copy()
    got = run_attend(p, lists, 0.125).cpu().double()
    cache, batch = p.device(capi)
    full = torch.empty((p.rows, 16, 64), dtype=torch.float16, device="cuda")
    capi.attention_paged_f16(full, p.q.cuda(), batch, cache, 0.125)
    want, bound = ref.attend(p, 0.125)
    assert ((got - want).abs() <= bound).all() and ((full.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [8, 16, 64])
def test_attention_with_holes_apart_and_larger_limits(int8, page):
    p = ref.Paged(94, 16, 2, 128, page, [1, 20, 1], [700, 400, 40], int8, holes=[(0, 0), (0, 2), (1, 1), (1, (399) // page)],
                  apart=True, pad=1)
    lists = sel.random_lists(p, 11, 95)
    check_attend(p, run_attend(p, lists, 0.09), lists, 0.09)
    check_attend(p, run_attend(p, lists, 0.09, max_new=500, max_len=700), lists, 0.09)


def test_attention_limits_bound_what_is_computed():
    p = ref.Paged(96, 8, 2, 64, 16, [40], [300])
    lists = sel.random_lists(p, 6, 97)
    got = run_attend(p, lists, 0.125, max_new=24)
    want, bound = sel.attend(p, lists, 0.125)
    assert ((got.cpu().double() - want).abs() <= bound)[:24].all()
    assert (got[24:] == 7.0).all()
    got = run_attend(p, lists, 0.125, max_len=250)
    p.table = torch.where(torch.arange(p.table.shape[1])[None] < 16, p.table, -1)
    seen = ref.Paged(96, 8, 2, 64, 16, [40], [300])
    for t in range(40):  # positions from 250 on are not seen: as a token at 249 at most
        if 260 + t >= 250:
            seen_row = sel.attend(_at(seen, t, 250), lists[t:t + 1], 0.125)
            assert ((got[t].cpu().double() - seen_row[0][0]).abs() <= seen_row[1][0]).all()


def _at(p, row, length):
    """One token of p's as the last of `length` positions."""
    one = ref.Paged(96, p.heads, p.kv, p.hd, p.page, [1], [length], spare=0)
    one.table, one.both, one.pages = p.table, p.both, p.pages
    one.q = p.q[row:row + 1]
    return one


def test_attention_to_nothing_gives_zeros():
    """Empty lists, holes alone, pages behind the token, tokens without a position."""
    p = ref.Paged(98, 8, 2, 64, 16, [1, 1, 1, 5, 1], [40, 40, 40, 2, 0], holes=[(1, 0), (1, 1), (1, 2)])
    lists = np.full((p.rows, 2, 3), -1, np.int32)
    lists[1] = [0, 1, 2]
    lists[2] = [3, 4, 2 ** 31 - 1]
    lists[3:] = [0, 1, 0]
    got = run_attend(p, lists, 0.125)
    check_attend(p, got, lists, 0.125)
    assert not got[:3].any() and not got[3:6].any() and not got[-1].any()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("hd,page,new", [(64, 16, 1), (80, 8, 3), (128, 16, 9), (128, 4, 1), (256, 16, 1)])
def test_infinities_and_nan_where_no_token_looks(bad, hd, page, new):
    """In positions behind a token, in pages that are not listed, in slots of no
    sequence; then one in a listed place, which its tokens get."""
    p = ref.Paged(99, 8, 2, hd, page, [new], [200], spare=3)
    n = 6
    lists = np.full((p.rows, 2, n), -1, np.int32)
    last = (200 - new) // page  # the page of the first new token
    for t in range(new):
        for h in range(2):
            lists[t, h] = [0, 1 + h, 3, -1, last, (200 - new + t) // page if (200 - new + t) // page != last else -1]
    clean = run_attend(p, lists, 0.125).cpu()
    check_attend(p, clean, lists, 0.125)
    k, v = p.both[0].view(-1, 2, hd), p.both[1].view(-1, 2, hd)
    slots = p.slots(0, 200)
    rest = torch.ones(p.pages * page, dtype=torch.bool)
    rest[slots] = False
    k[rest], v[rest] = bad, bad
    for j in (2, 4, 5):  # listed for neither, or for the other KV head
        at = slots[j * page:(j + 1) * page]
        heads = [h for h in range(2) if 1 + h != j]
        for h in heads:
            k[at, h], v[at, h] = bad, bad
    assert torch.equal(run_attend(p, lists, 0.125).cpu(), clean)
    if new > 1:
        at = 199
        v[slots[at], 0, 5] = bad
        got = run_attend(p, lists, 0.125).cpu()
        assert torch.equal(got[:new - 1], clean[:new - 1])
        hit = got[new - 1, :4, 5].float()
        assert torch.isnan(hit).all() if bad != bad else (hit == bad).all()
        v[slots[at], 0, 5] = 0
    v[slots[3 * page + 1], 1, 7] = bad
    got = run_attend(p, lists, 0.125).cpu()
    hit = got[:, 4:, 7].float()
    assert torch.isnan(hit).all() if bad != bad else (hit == bad).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[:, 4:, 7] = False
    if new > 1:
        keep[new - 1, :4, 5] = False
    assert torch.isfinite(got[keep]).all()


def test_int8_scales_that_are_not_numbers():
    for page in (4, 16):
        p = ref.Paged(100, 8, 2, 64, page, [3], [120], True)
        lists = np.tile(np.array([0, 2, 5], np.int32), (3, 2, 1))
        clean = run_attend(p, lists, 0.125).cpu()
        slots = p.slots(0, 120)
        p.vs.view(-1, 2)[slots[page], :], p.ks.view(-1, 2)[slots[page], :] = float("nan"), float("inf")  # page 1
        assert torch.equal(run_attend(p, lists, 0.125).cpu(), clean)
        p.vs.view(-1, 2)[slots[2 * page + 1], 1] = float("nan")
        p.ks.view(-1, 2)[slots[5 * page], 0] = float("nan")
        got = run_attend(p, lists, 0.125).cpu()
        assert torch.isnan(got).all()


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_attention_scales(scale):
    p = ref.Paged(101, 8, 2, 64, 16, [3], [400])
    lists = sel.random_lists(p, 9, 102)
    check_attend(p, run_attend(p, lists, scale), lists, scale)


def test_lists_and_lengths_far_into_a_large_pool():
    """A pool of more than 4 GiB a tensor, the pages at its far end."""
    kv, hd, page = 8, 256, 1024
    n = 2 ** 32 // (page * kv * hd * 2) + 8
    k = torch.zeros((n, page, kv, hd), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    p = ref.Paged(103, 16, kv, hd, page, [1, 3], [1500, 2100], spare=0)
    far = p.pages
    k[n - far:], v[n - far:] = p.k.cuda(), p.v.cuda()
    cache = capi.PagedKV(k, v, torch.where(p.table >= 0, p.table + (n - far), -1).int().cuda())
    batch = capi.SeqBatch(p.starts.cuda(), p.seq_lens.cuda(), p.rows, 3, 2100)
    lists = np.array([[[0, 1, -1]] * kv, [[2, 0, -1]] * kv, [[1, 2, -1]] * kv, [[0, 2, 1]] * kv], np.int32)
    check_attend(p, run_attend(p, lists, 0.0625, cache, batch), lists, 0.0625)
    bounds = torch.full((n, kv, hd // 8, 2, 8), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((n, kv), 7.0, device="cuda")
    capi.kv_bounds(bounds, scales, batch, cache)
    check_bounds(p, (bounds[n - far:], scales[n - far:]))
    assert (bounds[:n - far] == 99).all()


# ---------------------------------------------------------------- how calls are made
@pytest.mark.parametrize("new,lens,page", [([1, 1, 1], [900, 30, 2500], 16), ([40, 1, 3], [700, 300, 64], 8), ([1], [2000], 1)])
def test_captured_and_replayed_with_other_lengths(new, lens, page):
    """The three calls captured on one stream, replayed with other lengths beside eager
    calls on another."""
    p = ref.Paged(104, 16, 2, 64, page, new, lens)
    cache, batch = p.device(capi, max_len=4000)
    n = 20
    q = p.q.cuda()
    bounds = torch.zeros((p.pages, 2, 8, 2, 8), dtype=torch.int8, device="cuda")
    scales = torch.zeros((p.pages, 2), device="cuda")
    start = [torch.from_numpy(a).cuda() for a in sel.random_bounds(105, p.pages, 2, 64)]
    lists = torch.zeros((p.rows, 2, n), dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        capi.kv_bounds(bounds, scales, batch, cache, stream=s)
        capi.select_pages(lists, q, bounds, scales, batch, cache, 1, 2, stream=s)
        capi.attention_selected_f16(out, q, lists, batch, cache, 0.125, stream=s)
    for step in range(4):
        now = [max(k, m - 17 * step) for k, m in zip(new, lens)]
        p.lens, p.seq_lens = now, torch.tensor(now, dtype=torch.int32)
        batch.tensors[1].copy_(p.seq_lens)
        bounds.copy_(start[0])
        scales.copy_(start[1])
        out.fill_(7.0), lists.fill_(-7)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        torch.cuda.synchronize()
        both, scale = start[0].cpu().numpy().copy(), start[1].cpu().numpy().copy()
        for pg, held in sel.touched(p, max_len=4000):
            both[pg], scale[pg] = sel.bounds(p, pg, held)
        assert np.array_equal(bounds.cpu().numpy(), both) and np.array_equal(scales.cpu().numpy(), scale)
        check_select(p, lists, both, scale, n, 1, 2, max_len=4000)
        check_attend(p, out, lists.cpu().numpy(), 0.125)
        again, other = torch.zeros_like(lists), torch.zeros_like(out)
        capi.select_pages(again, q, bounds, scales, batch, cache, 1, 2)
        capi.attention_selected_f16(other, q, again, batch, cache, 0.125)
        assert torch.equal(again, lists) and torch.equal(other, out)
    capi.release_workspace(s)


def test_two_streams_at_once():
    a = ref.Paged(106, 32, 8, 64, 1, [1, 1], [3000, 2000])
    b = ref.Paged(107, 32, 8, 64, 1, [1], [4000])
    sides = []
    for p, seed in ((a, 108), (b, 109)):
        cache, batch = p.device(capi)
        both, scale = sel.random_bounds(seed, p.pages, 8, 64)
        q = p.q.cuda()
        sides.append((p, cache, batch, both, scale, q, torch.from_numpy(both).cuda(), torch.from_numpy(scale).cuda(),
                      torch.zeros((p.rows, 8, 50), dtype=torch.int32, device="cuda"), torch.empty_like(q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for p, cache, batch, _, _, q, bounds, scales, lists, out, s in sides:
            capi.select_pages(lists, q, bounds, scales, batch, cache, 1, 2, stream=s)
            capi.attention_selected_f16(out, q, lists, batch, cache, 0.125, stream=s)
    torch.cuda.synchronize()
    for p, _, _, both, scale, _, _, _, lists, out, s in sides:
        check_select(p, lists, both, scale, 50, 1, 2)
        check_attend(p, out, lists.cpu().numpy(), 0.125)
        capi.release_workspace(s)


def test_results_repeat_bit_for_bit_and_out_may_be_q():
    p = ref.Paged(110, 32, 8, 128, 16, [1, 70, 1, 3], [4000, 900, 3, 2000])
    cache, batch = p.device(capi)
    lists = torch.from_numpy(sel.random_lists(p, 30, 111)).cuda()
    first = run_attend(p, lists, 0.09, cache, batch).clone()
    for _ in range(3):
        assert torch.equal(run_attend(p, lists, 0.09, cache, batch), first)
    q = p.q.cuda()
    capi.attention_selected_f16(q, q, lists, batch, cache, 0.09)
    assert torch.equal(q, first)


@pytest.mark.parametrize("n", [65, 300, 5000])
def test_many_sequences(n):
    new = [0 if i % 13 == 5 else 1 + i % 3 for i in range(n)]
    lens = [0 if i % 31 == 7 else 1 + (i * 97) % 150 for i in range(n)]
    p = ref.Paged(112, 2, 1, 16, 8, new, lens)
    both, scale = sel.random_bounds(113, p.pages, 1, 16)
    how = (6, 1, 1)
    got = run_select(p, both, scale, *how)
    check_select(p, got, both, scale, *how)
    check_bounds(p, run_bounds(p))
    lists = got.cpu().numpy()
    check_attend(p, run_attend(p, got, 0.25), lists, 0.25)


def test_contiguous_cache_as_one_sequence():
    """page_table None: page j of the sequence is page j."""
    p = ref.Paged(114, 8, 2, 64, 16, [3], [300], spare=0)
    p.table = torch.arange(p.pages, dtype=torch.int32)[None]
    both, scale = sel.random_bounds(115, p.pages, 2, 64)
    cache = capi.PagedKV(p.k.cuda(), p.v.cuda())
    batch = capi.SeqBatch(p.starts.cuda(), p.seq_lens.cuda(), 3, 3, 300)
    how = (5, 1, 1)
    got = run_select(p, both, scale, *how, cache=cache, batch=batch)
    check_select(p, got, both, scale, *how)
    check_attend(p, run_attend(p, got, 0.125, cache, batch), got.cpu().numpy(), 0.125)
    check_bounds(p, run_bounds(p, cache, batch))


def test_a_cache_without_pages():
    """Nothing to see: lists of -1, zeros."""
    k = torch.zeros((0, 16, 2, 64), dtype=torch.float16, device="cuda")
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = capi.PagedKV(k, k.clone(), torch.full((1, 4), -1, dtype=torch.int32, device="cuda"))
    batch = capi.SeqBatch(t(0, 2), t(30), 2, 2, 64)
    q = torch.randn((2, 8, 64), device="cuda").half()
    bounds = torch.zeros((0, 2, 8, 2, 8), dtype=torch.int8, device="cuda")
    scales = torch.zeros((0, 2), device="cuda")
    lists = torch.full((2, 2, 5), -7, dtype=torch.int32, device="cuda")
    capi.kv_bounds(bounds, scales, batch, cache)
    capi.select_pages(lists, q, bounds, scales, batch, cache)
    assert (lists == -1).all()
    out = torch.full_like(q, 7.0)
    capi.attention_selected_f16(out, q, torch.zeros_like(lists), batch, cache, 0.125)
    assert not out.any()
